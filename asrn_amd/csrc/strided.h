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
  // n <= 4 tokens from t (the rest as `other`). ROW: tokens adjacent, read as one vector from any element's address
  template <bool ROW>
  __device__ __forceinline__ void four(int64_t b, int64_t t, int n, float other, float* x) const {
    if (ROW && n == 4) {
      __builtin_memcpy(x, reinterpret_cast<const float*>(p) + b * sb + t, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = k < n ? at(b, t + k) : other;
    }
  }
  // the mask of n <= 4 tokens from t, a byte each (the rest 0)
  template <bool ROW>
  __device__ __forceinline__ uint32_t on4(int64_t b, int64_t t, int n) const {
    uint32_t w = 0;
    if (!p) {
      w = 0x01010101u;
    } else if (ROW && n == 4) {
      __builtin_memcpy(&w, reinterpret_cast<const uint8_t*>(p) + b * sb + t, 4);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n) w |= (uint32_t)reinterpret_cast<const uint8_t*>(p)[b * sb + (t + k) * st] << (8 * k);
    }
    return n == 4 ? w : n > 0 ? w & ((1u << (8 * n)) - 1u) : 0u;
  }
  bool row() const { return !p || st == 1; }
};

// sums of doubles over the wave, in a fixed order: DPP rotations within each row of 16 lanes (no LDS), the rows by lane
// reads
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t u = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double readlane_d(double v, int lane) {
  const uint64_t u = __double_as_longlong(v);
  return __longlong_as_double((long long)((uint64_t)(uint32_t)readlane_i((int)(uint32_t)(u >> 32), lane) << 32 |
                                          (uint32_t)readlane_i((int)(uint32_t)u, lane)));
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v += dpp_d<0x128>(v);
  v += dpp_d<0x124>(v);
  v += dpp_d<0x122>(v);
  v += dpp_d<0x121>(v);
  return ((readlane_d(v, 0) + readlane_d(v, 16)) + readlane_d(v, 32)) + readlane_d(v, 48);
}

// lanes (a power of two up to a wave) that share a text's pieces in the reductions over them
inline int lanes_for(int64_t pieces) {
  int g = 1;
  while (g < kWave && g < pieces) g *= 2;
  return g;
}
// the sum over each aligned group of g lanes, in every lane of it
__device__ __forceinline__ double group_sum_d(double v, int g) {
  for (int m = g >> 1; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

}  // namespace asrn
