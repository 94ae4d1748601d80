// Matrices of texts by tokens read in place through both strides (slices, expanded rows), for the losses over them.
#pragma once
#include "common.h"

namespace asrn {

struct Strided {
  const void* p; int64_t sb, st;            // element (b, t) at b sb + t st; p null: absent
  __device__ __forceinline__ float at(int64_t b, int64_t t) const {
    return reinterpret_cast<const float*>(p)[b * sb + t * st];
  }
  // a mask of one byte a token; an absent one keeps every token
  __device__ __forceinline__ bool on(int64_t b, int64_t t) const {
    return !p || reinterpret_cast<const uint8_t*>(p)[b * sb + t * st] != 0;
  }
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

}  // namespace asrn
