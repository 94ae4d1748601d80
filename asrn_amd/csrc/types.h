// Element types of the operators that take fp32, bf16 and fp16 (type 0, 1, 2 at the C entries), and the activations they
// share. Values are widened exactly and rounded to nearest even.
#pragma once
#include "common.h"

namespace asrn {

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;

// f(the C++ type of `type`), for types that type_ok has passed
template <typename F>
inline int with_type(int32_t type, F&& f) {
  if (type == 1) return f(bf16_t{});
  if (type == 2) return f(fp16_t{});
  return f(float{});
}
inline bool type_ok(int32_t type) { return type >= 0 && type <= 2; }
// whether n threads in workgroups of `group` are a launch: fewer than 2^32
inline bool grid_ok(int64_t n, int group) { return (n + group - 1) / group * group < ((int64_t)1 << 32); }
inline int type_bytes(int32_t type) { return type == 0 ? 4 : 2; }

// V adjacent values, one access of V elements (V = 1: no alignment beyond the element's)
template <int V, typename T>
__device__ __forceinline__ void load_v(const T* p, float (&x)[V]) {
  typedef T TV __attribute__((ext_vector_type(V)));
  if constexpr (V == 1) {
    x[0] = (float)*p;
  } else {
    const TV v = *reinterpret_cast<const TV*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (float)v[i];
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_v(T* p, const float (&x)[V]) {
  typedef T TV __attribute__((ext_vector_type(V)));
  if constexpr (V == 1) {
    *p = (T)x[0];
  } else {
    TV v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)x[i];
    *reinterpret_cast<TV*>(p) = v;
  }
}

enum Activation { kActNone = 0, kActGelu = 1, kActSilu = 2 };

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
// 1 / (1 + exp(-x)): the exponential of a large -x is infinite and its reciprocal 0
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + exp_fast(-x)); }

// Phi(x) and phi(x) of the standard normal distribution for erf's GELU
__device__ __forceinline__ float normal_cdf(float x) { return 0.5f * (1.f + erff(x * 0.70710678118654752f)); }
__device__ __forceinline__ float normal_pdf(float x) { return 0.3989422804014327f * exp_fast(-0.5f * x * x); }

__device__ __forceinline__ float activate(float x, int act) {
  if (act == kActGelu) return x * normal_cdf(x);
  return act == kActSilu ? x * sigmoid(x) : x;
}
__device__ __forceinline__ float activate_grad(float x, int act) {
  if (act == kActGelu) return normal_cdf(x) + x * normal_pdf(x);
  if (act == kActSilu) {
    const float s = sigmoid(x);
    return s * (1.f + x * (1.f - s));
  }
  return 1.f;
}

}  // namespace asrn
