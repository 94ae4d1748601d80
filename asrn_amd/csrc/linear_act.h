// The epilogue of a product: bias, activation, residual, and the activation's input kept for the backward.
#pragma once
#include "types.h"

namespace asrn {

struct Epilogue {
  const void* bias;               // (N) in the operands' type, or null
  const void* res; int64_t ldr;   // (M, N), or null
  void* pre; int64_t ldp;         // (M, N) in the operands' type, or null
  void* y; int64_t ldy;
  int act, res32, y32;            // res and y in fp32, else in the operands' type
  int vec;                        // whether neighbouring values may be read and written as vectors

  // v, the product's result at (m, n)
  template <typename T>
  __device__ __forceinline__ void one(int64_t m, int n, float v) const {
    if (bias) v += (float)static_cast<const T*>(bias)[n];
    if (pre) static_cast<T*>(pre)[m * ldp + n] = (T)v;
    v = activate(v, act);
    if (res) v += res32 ? static_cast<const float*>(res)[m * ldr + n] : (float)static_cast<const T*>(res)[m * ldr + n];
    if (y32) static_cast<float*>(y)[m * ldy + n] = v;
    else static_cast<T*>(y)[m * ldy + n] = (T)v;
  }
};

int64_t gemm_epilogue_workspace(int64_t M, int64_t N, int64_t K);
// x (M, K) W (N, K)^T in fp32 with the epilogue, as asrn_gemm forms the product (gemm.hip)
int gemm_epilogue(const float* x, int64_t ldx, const float* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e,
                  void* workspace, int64_t workspace_bytes, hipStream_t st);

}  // namespace asrn
