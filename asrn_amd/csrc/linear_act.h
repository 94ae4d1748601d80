// What the 16-bit products share, and the epilogue of a product: bias, activation, residual, and the activation's input kept for
// the backward.
#pragma once
#include "types.h"

namespace asrn {

typedef float fx16 __attribute__((ext_vector_type(16)));
typedef bf16_t bfx8 __attribute__((ext_vector_type(8)));
typedef fp16_t hx8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ fx16 mfma32(bfx8 a, bfx8 b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ fx16 mfma32(hx8 a, hx8 b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

constexpr unsigned kPast = 1u << 31;              // past the end of a buffer of this many bytes: reads 0

// 16 bytes a lane from memory to LDS, lane i's to l[i] (l: the same in every lane)
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t rsrc, uint4* l, unsigned at, unsigned off) {
#ifdef __HIP_DEVICE_COMPILE__                     // the host's pass does not know the 16-byte form
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)l, 16, at, off, 0, 0);
#endif
}

// For products of 16-bit operands: Phi(-|x|) = t p(t) exp(-x^2 / 2) with Abramowitz and Stegun's 7.1.26, erfc within 1.5e-7:
// one exponential and one reciprocal (erff costs about twice the instructions, and the epilogue counts beside the product).
// Phi is within 7.5e-8 before fp32's roundings and within 2.7e-7 with them (the polynomial's terms cancel near t = 1), GELU
// within 2.8e-7 |x| and its derivative within 2.8e-7 (bf16's half step at 1 is 3.9e-3). -> t p(t), *e = exp(-x^2 / 2)
__device__ __forceinline__ float normal_tail(float x, float* e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(x), 1.f));
  const float z = x * 0.84932180028801904f;                        // sqrt(log2(e) / 2)
  *e = __builtin_amdgcn_exp2f(-z * z);
  return t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f),
                          0.5f * -0.284496736f), 0.5f * 0.254829592f);
}
__device__ __forceinline__ float gelu16(float x) {
  float e;
  const float p = normal_tail(x, &e);
  return fmaf(-fabsf(fminf(x, 64.f)), p * e, fmaxf(x, 0.f));       // infinity stays itself
}
__device__ __forceinline__ float gelu16_grad(float x) {
  float e;
  const float p = normal_tail(x, &e), m = e * fmaf(-0.39894228040143268f, fabsf(x), p);
  return x < 0.f ? m : 1.f - m;
}

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
    v = sizeof(T) == 2 && act == kActGelu ? gelu16(v) : activate(v, act);
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
