// Activations kept in 8 bits for the backward pass: the LayerNorm and the GELU of a local block whose backward reads its
// input back from 8 bits, and what a product's weight gradient reads.
//
// The format: 32 neighbouring channels of a row share a scale 2^e, the smallest with max |x| <= 127 2^e (a byte, e + 127;
// -126 <= e <= 121), and each is the integer nearest to x 2^-e (ties to even). A power of two divides and multiplies exactly,
// so the one rounding is the integer's, at most 2^e / 2 = max |x| / 127, and what is read back has 7 bits and fits bf16
// exactly: bf16 products take it without another rounding. A group that holds an infinity, a NaN or a value past 127 2^121
// (the last 1% of fp32's range) reads back as NaN (byte 255): the step's gradients are then not finite.
//
//   k_norm8_fwd  LayerNorm in fp32 (two-pass variance), y in fp32 or bf16, (mean, rstd) per row, and x's 8 bits: one
//                pass over x. A wave takes a row as 4 channels a lane, two rows in flight.
//   k_norm8_bwd  its gradient with xhat = (x8 - mean) rstd; [+ the residual path's gradient], d gamma and d beta as
//                partial rows of a workgroup, summed in a fixed order.
//   k_norm8_read the LayerNorm's output again, as the columns of a causal window of k tokens (k = 1: as it was).
//   k_gelu8_fwd  gelu(u) [+ h], and u's 8 bits: 8 channels a lane.
//   k_gelu8_bwd  d u = gelu'(u8) d y;   k_gelu8_read gelu(u8);   k_pack8, k_unpack8 the format alone.
// All are bound by HBM (16384 x 768 bf16: LayerNorm 16 and 25 us, 5.5-5.7 TB/s, read back 10 and, as a window of 4, 24;
// 16384 x 1536 bf16: the GELU's gradient 21 us, 6.1 TB/s, read back 17, 20 with nothing of it in a cache) but the GELU's
// forward in bf16, by erff's instructions (27 us, 4.7 TB/s), and the LayerNorm's backward past 4,096 channels, whose 222
// registers leave 2 waves a SIMD (4096 x 8192: 100 us for 370 MB).
#include <math.h>

#include "common.h"

namespace asrn {

constexpr int kE8Threads = 256;
constexpr int kE8Waves = kE8Threads / kWave;
constexpr int kE8Group = 32;
constexpr int kE8MaxD = 8192;                 // the LayerNorm's widths
constexpr int kE8WaveD = 1024;                // up to this a wave takes a row, past it a workgroup

typedef __bf16 e8_b2 __attribute__((ext_vector_type(2)));
typedef float e8_f2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t e8_pack_bf16(float a, float b) {       // rounded to nearest even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((e8_f2){a, b}, e8_b2));
}
__device__ __forceinline__ uint32_t e8_abs(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// the scale's byte from the largest |x| of a group, as bits: 127 / 128 of the next power of two is 127 2^e; 0x7f7e0000 is
// 127 2^121, past which the integer 64 would stand for 2^128
__device__ __forceinline__ uint32_t e8_byte(uint32_t top) {
  const int e = (int)(top >> 23) - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return top > 0x7f7e0000u ? 255u : (uint32_t)(e < 1 ? 1 : e);
}
__device__ __forceinline__ float e8_inverse(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float e8_scale(uint32_t byte) { return byte == 255u ? NAN : __uint_as_float(byte << 23); }
__device__ __forceinline__ uint32_t e8_int(float x, float inv) {
  return (uint32_t)(inv == 0.f ? 0 : __float2int_rn(x * inv)) & 0xffu;
}
__device__ __forceinline__ uint32_t e8_quad(const float4& x, float inv) {
  return e8_int(x.x, inv) | (e8_int(x.y, inv) << 8) | (e8_int(x.z, inv) << 16) | (e8_int(x.w, inv) << 24);
}
__device__ __forceinline__ float4 e8_open(uint32_t q, float s) {
  return make_float4((float)(int8_t)q * s, (float)(int8_t)(q >> 8) * s, (float)(int8_t)(q >> 16) * s,
                     (float)(int8_t)(q >> 24) * s);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return o > v ? o : v;
}
// the largest over each aligned 4 lanes (quad permutes), and over each aligned 8 (mirrored halves of a row)
__device__ __forceinline__ uint32_t max_of4(uint32_t v) { return dpp_max<0x4E>(dpp_max<0xB1>(v)); }
__device__ __forceinline__ uint32_t max_of8(uint32_t v) { return dpp_max<0x141>(max_of4(v)); }

// ---- GELU ----------------------------------------------------------------------------------------------------------
// exact GELU, as torch forms it in fp32
__device__ __forceinline__ float e8_gelu(float x) { return x * 0.5f * (1.f + erff(x * 0.70710678118654752f)); }
// For the values read back: Phi(-|x|) = e p with e = exp(-x^2 / 2), from Abramowitz and Stegun's 7.1.26: erfc within 1.5e-7,
// so Phi within 8e-8 at every x before fp32's roundings. Of itself the vanishing tail is less exact the further out: 5e-5
// at |x| = 3, 5e-4 at 4, 1e-2 at 8, where it weighs nothing beside the 8 bits' own rounding. One exponential and one reciprocal
// serve the value and the derivative: with m = Phi(-|x|) - |x| phi(x), gelu = max(x, 0) - |x| Phi(-|x|) and gelu' = m
// below 0, 1 - m above (erff's two branches cost about twice the instructions, and these kernels run out of them first)
__device__ __forceinline__ float e8_tail(float x, float* e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(x), 1.f));
  const float z = x * 0.84932180028801904f;                        // sqrt(log2(e) / 2)
  *e = __builtin_amdgcn_exp2f(-z * z);
  return t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f),
                          0.5f * -0.284496736f), 0.5f * 0.254829592f);
}
__device__ __forceinline__ float e8_gelu_read(float x) {
  float e;
  const float p = e8_tail(x, &e);
  return fmaf(-fabsf(x), p * e, fmaxf(x, 0.f));                    // p is NaN where x is
}
__device__ __forceinline__ float e8_dgelu(float x) {
  float e;
  const float p = e8_tail(x, &e);
  const float m = e * fmaf(-0.39894228040143268f, fabsf(x), p);
  return x < 0.f ? m : 1.f - m;
}

// ---- elementwise kernels: 8 channels a lane, 4 lanes a group ---------------------------------------------------------
struct E8Args {
  const void* u; const float* h; void* out; int8_t* q; uint8_t* e; const void* dy;
  int64_t rows; int d; int groups;            // groups = ceil(d / 32)
  int64_t lanes;                              // rows * groups * 4
};

// the lane's row, first channel and number of channels (0: past the row)
struct E8Place { int64_t row; int c0, n; int64_t at, group; };
template <bool WHOLE>                         // d a multiple of 32: lanes run through the tensor
__device__ __forceinline__ E8Place e8_place(const E8Args& a, int64_t i) {
  E8Place p;
  if constexpr (WHOLE) {
    p.row = 0; p.c0 = 0; p.n = 8; p.at = 8 * i; p.group = i >> 2;
  } else {
    const uint32_t per = 4u * (uint32_t)a.groups;
    p.row = (uint32_t)i / per;                // lanes < 2^32
    p.c0 = 8 * (int)(i - p.row * per);
    p.n = a.d - p.c0 < 0 ? 0 : a.d - p.c0 > 8 ? 8 : a.d - p.c0;
    p.at = p.row * a.d + p.c0;
    p.group = p.row * a.groups + (p.c0 >> 5);
  }
  return p;
}
template <bool B16>
__device__ __forceinline__ void e8_load(const void* p, int64_t at, int n, float* x) {
  if (n == 8) {
    if constexpr (B16) {
      uint4 v;
      __builtin_memcpy(&v, reinterpret_cast<const uint16_t*>(p) + at, 16);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    } else {
      __builtin_memcpy(x, reinterpret_cast<const float*>(p) + at, 32);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k] = 0.f;
      if (k < n) x[k] = B16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[at + k] << 16)
                            : reinterpret_cast<const float*>(p)[at + k];
    }
  }
}
template <bool B16>
__device__ __forceinline__ void e8_store(void* p, int64_t at, int n, const float* x) {
  if (n == 8) {
    if constexpr (B16) {
      const uint4 v = make_uint4(e8_pack_bf16(x[0], x[1]), e8_pack_bf16(x[2], x[3]), e8_pack_bf16(x[4], x[5]),
                                 e8_pack_bf16(x[6], x[7]));
      __builtin_memcpy(reinterpret_cast<uint16_t*>(p) + at, &v, 16);
    } else {
      __builtin_memcpy(reinterpret_cast<float*>(p) + at, x, 32);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) {
        if constexpr (B16) reinterpret_cast<uint16_t*>(p)[at + k] = (uint16_t)e8_pack_bf16(x[k], 0.f);
        else reinterpret_cast<float*>(p)[at + k] = x[k];
      }
  }
}
// the group's scale over its 4 lanes, the lane's integers and, by the group's first lane, the scale's byte
__device__ __forceinline__ void e8_write(const E8Args& a, const E8Place& p, const float* x) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = e8_abs(x[k]) > top ? e8_abs(x[k]) : top;
  const uint32_t byte = e8_byte(max_of4(top));
  const float inv = e8_inverse(byte);
  const uint32_t w[2] = {e8_quad(make_float4(x[0], x[1], x[2], x[3]), inv), e8_quad(make_float4(x[4], x[5], x[6], x[7]), inv)};
  if (p.n == 8) {
    __builtin_memcpy(a.q + p.at, w, 8);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < p.n) a.q[p.at + k] = (int8_t)(w[k >> 2] >> (8 * (k & 3)));
  }
  if ((threadIdx.x & 3) == 0) a.e[p.group] = (uint8_t)byte;
}
__device__ __forceinline__ void e8_read(const E8Args& a, const E8Place& p, float* x) {
  const float s = e8_scale(a.e[p.group]);
  uint32_t w[2] = {0u, 0u};
  if (p.n == 8) {
    __builtin_memcpy(w, a.q + p.at, 8);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < p.n) w[k >> 2] |= (uint32_t)(uint8_t)a.q[p.at + k] << (8 * (k & 3));
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = (float)(int8_t)(w[k >> 2] >> (8 * (k & 3))) * s;
}

enum { kE8Gelu = 0, kE8Pack = 1 };
// u -> out = gelu(u) [+ h], and u's 8 bits (kE8Pack: the bits alone). Every lane of a group reaches the group's maximum:
// the four enter or leave together, and channels past a row's end count as 0.
template <bool B16, int OP, bool ADD, bool WHOLE>
__global__ __launch_bounds__(kE8Threads) void k_gelu8_fwd(E8Args a) {
  const int64_t i = (int64_t)blockIdx.x * kE8Threads + threadIdx.x;
  if (i >= a.lanes) return;                   // lanes come in fours, so groups leave whole
  const E8Place p = e8_place<WHOLE>(a, i);
  float x[8];
  e8_load<B16>(a.u, p.at, p.n, x);
  float h[8];
  if constexpr (ADD) e8_load<false>(a.h, p.at, p.n, h);
  e8_write(a, p, x);
  if constexpr (OP == kE8Gelu) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k] = e8_gelu(x[k]);
      if constexpr (ADD) {                    // rounded to u's type before the sum, as the separate operations round
        if constexpr (B16) x[k] = __uint_as_float(e8_pack_bf16(x[k], 0.f) << 16);
        x[k] += h[k];
      }
    }
    e8_store<B16 && !ADD>(a.out, p.at, p.n, x);
  }
}

enum { kE8Read = 0, kE8ReadGelu = 1, kE8Grad = 2 };
// kE8Read: out = u8; kE8ReadGelu: out = gelu(u8); kE8Grad: out = gelu'(u8) dy
template <bool O16, bool D16, int OP, bool WHOLE>
__global__ __launch_bounds__(kE8Threads) void k_gelu8_bwd(E8Args a) {
  const int64_t i = (int64_t)blockIdx.x * kE8Threads + threadIdx.x;
  if (i >= a.lanes) return;
  const E8Place p = e8_place<WHOLE>(a, i);
  float x[8], d[8];
  if constexpr (OP == kE8Grad) e8_load<D16>(a.dy, p.at, p.n, d);
  e8_read(a, p, x);
  if constexpr (OP == kE8Grad) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = e8_dgelu(x[k]) * d[k];
  }
  if constexpr (OP == kE8ReadGelu) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = e8_gelu_read(x[k]);
  }
  e8_store<O16>(a.out, p.at, p.n, x);
}

// ---- the LayerNorm ---------------------------------------------------------------------------------------------------
struct N8Args {
  const float* x; const float* gamma; const float* beta; int64_t rows; int d; float eps;
  void* y; float2* stats; uint32_t* q; uint8_t* e; int groups;      // q as words of 4 channels
  const void* dy; const float* dres; float* dx; float* partial;
  int64_t L; int k;
  int per;                                    // backward: rows of a workgroup
};
constexpr int kN8FwdRows = 2;                 // rows a wave has in flight
// Rows a backward's workgroup takes: enough workgroups for two a CU, as long as each has 8 rows at least (its partial row
// of parameter gradients costs as much as 2 rows), 32 at most (us with 32 always / so: 1505 x 260 11.0 / 7.7, 4096 x 2048
// 54.8 / 23.2, 4096 x 8192 258 / 107)
constexpr int kN8BwdLeast = 8, kN8BwdMost = 32, kN8BwdGroups = 512;
static int n8_bwd_rows(int64_t rows) {
  const int64_t per = (rows + kN8BwdGroups - 1) / kN8BwdGroups;
  return per <= kN8BwdLeast ? kN8BwdLeast : per >= kN8BwdMost ? kN8BwdMost : (int)((per + 7) / 8 * 8);
}

__device__ __forceinline__ float n8_dot(const float4& a, const float4& b) { return a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w; }
template <bool B16>
__device__ __forceinline__ float4 n8_load(const void* p, int64_t quad) {
  if constexpr (B16) {
    const uint2 u = reinterpret_cast<const uint2*>(p)[quad];
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
  } else {
    return reinterpret_cast<const float4*>(p)[quad];
  }
}
template <bool B16>
__device__ __forceinline__ void n8_store(void* p, int64_t quad, const float4& v) {
  if constexpr (B16) reinterpret_cast<uint2*>(p)[quad] = make_uint2(e8_pack_bf16(v.x, v.y), e8_pack_bf16(v.z, v.w));
  else reinterpret_cast<float4*>(p)[quad] = v;
}

// the 4 channels c of a row: y, the codes and, by a group's first lane, the scale's byte. All lanes of a wave call it, so
// that a group's 8 lanes meet; x is 0 past the row (the last group's scale is that of its own channels)
template <bool O16>
__device__ __forceinline__ void n8_row_out(const N8Args& a, int64_t r, int c, const float4& t, float mean, float rstd) {
  uint32_t top = e8_abs(t.x);
  top = e8_abs(t.y) > top ? e8_abs(t.y) : top;
  top = e8_abs(t.z) > top ? e8_abs(t.z) : top;
  top = e8_abs(t.w) > top ? e8_abs(t.w) : top;
  const uint32_t byte = e8_byte(max_of8(top));
  const int d4 = a.d >> 2;
  if (c < d4) {
    const float4 w = reinterpret_cast<const float4*>(a.gamma)[c], b = reinterpret_cast<const float4*>(a.beta)[c];
    n8_store<O16>(a.y, r * d4 + c, make_float4((t.x - mean) * rstd * w.x + b.x, (t.y - mean) * rstd * w.y + b.y,
                                               (t.z - mean) * rstd * w.z + b.z, (t.w - mean) * rstd * w.w + b.w));
    a.q[r * d4 + c] = e8_quad(t, e8_inverse(byte));
    if ((c & 7) == 0) a.e[r * a.groups + (c >> 3)] = (uint8_t)byte;
  }
}

template <int D4, bool O16>
__global__ __launch_bounds__(kE8Threads) void k_norm8_fwd(N8Args a) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6, d4 = a.d >> 2;
  const int64_t r0 = ((int64_t)blockIdx.x * kE8Waves + wave) * kN8FwdRows;
  const float inv_d = 1.f / (float)a.d;
  float4 x[kN8FwdRows][D4];
#pragma unroll
  for (int u = 0; u < kN8FwdRows; ++u)
#pragma unroll
    for (int k = 0; k < D4; ++k) {
      const int c = lane + kWave * k;
      x[u][k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r0 + u < a.rows && c < d4) x[u][k] = reinterpret_cast<const float4*>(a.x)[(r0 + u) * d4 + c];
    }
#pragma unroll
  for (int u = 0; u < kN8FwdRows; ++u) {
    const int64_t r = r0 + u;
    if (r >= a.rows) break;
    float s = 0.f, v = 0.f;
#pragma unroll
    for (int k = 0; k < D4; ++k) s += (x[u][k].x + x[u][k].y) + (x[u][k].z + x[u][k].w);
    const float mean = wave_sum_u(s) * inv_d;
#pragma unroll
    for (int k = 0; k < D4; ++k)
      if (lane + kWave * k < d4) {
        const float4 c = make_float4(x[u][k].x - mean, x[u][k].y - mean, x[u][k].z - mean, x[u][k].w - mean);
        v += n8_dot(c, c);
      }
    const float rstd = rsqrtf(wave_sum_u(v) * inv_d + a.eps);
#pragma unroll
    for (int k = 0; k < D4; ++k) n8_row_out<O16>(a, r, lane + kWave * k, x[u][k], mean, rstd);
    if (lane == 0) a.stats[r] = make_float2(mean, rstd);
  }
}

template <int D4, bool D16>
__global__ __launch_bounds__(kE8Threads) void k_norm8_bwd(N8Args a) {
  __shared__ float4 red[kE8Waves][2 * D4 * kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6, d4 = a.d >> 2;
  const float inv_d = 1.f / (float)a.d;
  const int64_t r0 = (int64_t)blockIdx.x * a.per + wave * (a.per / kE8Waves);
  float4 gw[D4], gb[D4], w[D4];
#pragma unroll
  for (int k = 0; k < D4; ++k) {
    const int c = lane + kWave * k;
    gw[k] = gb[k] = w[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < d4) w[k] = reinterpret_cast<const float4*>(a.gamma)[c];
  }
  constexpr int U = 2;                        // rows in flight
  for (int b = 0; b < a.per / kE8Waves; b += U) {
    uint32_t q[U][D4], e[U][D4];
    float4 dy[U][D4], dr[U][D4];
    float2 st[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + b + u;
      const bool ok = r < a.rows;
      st[u] = ok ? a.stats[r] : make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < D4; ++k) {
        const int c = lane + kWave * k;
        q[u][k] = e[u][k] = 0u;
        dy[u][k] = dr[u][k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ok && c < d4) {
          q[u][k] = a.q[r * d4 + c];
          e[u][k] = a.e[r * a.groups + (c >> 3)];
          dy[u][k] = n8_load<D16>(a.dy, r * d4 + c);
          if (a.dres) dr[u][k] = reinterpret_cast<const float4*>(a.dres)[r * d4 + c];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + b + u;
      if (r >= a.rows) break;
      const float mean = st[u].x, rstd = st[u].y;
      float4 xh[D4], g[D4];
      float m1 = 0.f, m2 = 0.f;
#pragma unroll
      for (int k = 0; k < D4; ++k) {
        xh[k] = g[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (lane + kWave * k < d4) {
          const float4 t = e8_open(q[u][k], e8_scale(e[u][k])), d = dy[u][k];
          xh[k] = make_float4((t.x - mean) * rstd, (t.y - mean) * rstd, (t.z - mean) * rstd, (t.w - mean) * rstd);
          g[k] = make_float4(d.x * w[k].x, d.y * w[k].y, d.z * w[k].z, d.w * w[k].w);
          m1 += (g[k].x + g[k].y) + (g[k].z + g[k].w);
          m2 += n8_dot(g[k], xh[k]);
          gw[k].x += d.x * xh[k].x; gw[k].y += d.y * xh[k].y; gw[k].z += d.z * xh[k].z; gw[k].w += d.w * xh[k].w;
          gb[k].x += d.x; gb[k].y += d.y; gb[k].z += d.z; gb[k].w += d.w;
        }
      }
      m1 = wave_sum_u(m1) * inv_d;
      m2 = wave_sum_u(m2) * inv_d;
#pragma unroll
      for (int k = 0; k < D4; ++k) {
        const int c = lane + kWave * k;
        if (c < d4) {
          const float4 o = dr[u][k];
          reinterpret_cast<float4*>(a.dx)[r * d4 + c] =
              make_float4(rstd * (g[k].x - m1 - xh[k].x * m2) + o.x, rstd * (g[k].y - m1 - xh[k].y * m2) + o.y,
                          rstd * (g[k].z - m1 - xh[k].z * m2) + o.z, rstd * (g[k].w - m1 - xh[k].w * m2) + o.w);
        }
      }
    }
  }
  // the workgroup's partial row [d gamma | d beta], the waves in order
#pragma unroll
  for (int k = 0; k < D4; ++k) {
    red[wave][lane + kWave * k] = gw[k];
    red[wave][D4 * kWave + lane + kWave * k] = gb[k];
  }
  __syncthreads();
  float4* out = reinterpret_cast<float4*>(a.partial) + (int64_t)blockIdx.x * 2 * d4;
  for (int c = threadIdx.x; c < 2 * d4; c += kE8Threads) {
    const int src = c < d4 ? c : D4 * kWave + (c - d4);
    float4 v = red[0][src];
#pragma unroll
    for (int i = 1; i < kE8Waves; ++i) {
      v.x += red[i][src].x; v.y += red[i][src].y; v.z += red[i][src].z; v.w += red[i][src].w;
    }
    out[c] = v;
  }
}

// Rows past 1,024 channels: a workgroup takes a row, 4 channels a thread and step, and the sums over the row go through
// LDS. The backward's threads keep their own channels' parameter gradients over the workgroup's rows, so nothing is joined
// at the end (4096 x 2048 bf16: forward 11.8 us, backward 23.2 us).
__device__ __forceinline__ float2 n8_block_sums(float a, float b, float2* red) {
  a = wave_sum_u(a);
  b = wave_sum_u(b);
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x >> 6] = make_float2(a, b);
  __syncthreads();
  float2 r = red[0];
#pragma unroll
  for (int w = 1; w < kE8Waves; ++w) {
    r.x += red[w].x;
    r.y += red[w].y;
  }
  return r;
}

template <int D4, bool O16>
__global__ __launch_bounds__(kE8Threads) void k_norm8_fwd_wide(N8Args a) {
  __shared__ float2 red[2][kE8Waves];
  const int tid = threadIdx.x, d4 = a.d >> 2;
  const int64_t r = blockIdx.x;
  const float inv_d = 1.f / (float)a.d;
  float4 x[D4];
  float s = 0.f, v = 0.f;
#pragma unroll
  for (int k = 0; k < D4; ++k) {
    const int c = tid + kE8Threads * k;
    x[k] = c < d4 ? reinterpret_cast<const float4*>(a.x)[r * d4 + c] : make_float4(0.f, 0.f, 0.f, 0.f);
    s += (x[k].x + x[k].y) + (x[k].z + x[k].w);
  }
  const float mean = n8_block_sums(s, 0.f, red[0]).x * inv_d;
#pragma unroll
  for (int k = 0; k < D4; ++k)
    if (tid + kE8Threads * k < d4) {
      const float4 c = make_float4(x[k].x - mean, x[k].y - mean, x[k].z - mean, x[k].w - mean);
      v += n8_dot(c, c);
    }
  const float rstd = rsqrtf(n8_block_sums(v, 0.f, red[1]).x * inv_d + a.eps);
#pragma unroll
  for (int k = 0; k < D4; ++k) n8_row_out<O16>(a, r, tid + kE8Threads * k, x[k], mean, rstd);
  if (tid == 0) a.stats[r] = make_float2(mean, rstd);
}

template <int D4, bool D16>
__global__ __launch_bounds__(kE8Threads) void k_norm8_bwd_wide(N8Args a) {
  __shared__ float2 red[2][kE8Waves];
  const int tid = threadIdx.x, d4 = a.d >> 2;
  const float inv_d = 1.f / (float)a.d;
  const int64_t r0 = (int64_t)blockIdx.x * a.per, r1 = r0 + a.per < a.rows ? r0 + a.per : a.rows;
  float4 gw[D4], gb[D4];
#pragma unroll
  for (int k = 0; k < D4; ++k) gw[k] = gb[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t r = r0; r < r1; ++r) {
    uint32_t q[D4], e[D4];
    float4 xh[D4], g[D4], dr[D4];
    const float2 st = a.stats[r];
#pragma unroll
    for (int k = 0; k < D4; ++k) {
      const int c = tid + kE8Threads * k;
      q[k] = e[k] = 0u;
      g[k] = dr[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < d4) {
        q[k] = a.q[r * d4 + c];
        e[k] = a.e[r * a.groups + (c >> 3)];
        g[k] = n8_load<D16>(a.dy, r * d4 + c);
        if (a.dres) dr[k] = reinterpret_cast<const float4*>(a.dres)[r * d4 + c];
      }
    }
    float m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int k = 0; k < D4; ++k) {
      const int c = tid + kE8Threads * k;
      xh[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < d4) {
        const float4 w = reinterpret_cast<const float4*>(a.gamma)[c], d = g[k], t = e8_open(q[k], e8_scale(e[k]));
        xh[k] = make_float4((t.x - st.x) * st.y, (t.y - st.x) * st.y, (t.z - st.x) * st.y, (t.w - st.x) * st.y);
        gw[k].x += d.x * xh[k].x; gw[k].y += d.y * xh[k].y; gw[k].z += d.z * xh[k].z; gw[k].w += d.w * xh[k].w;
        gb[k].x += d.x; gb[k].y += d.y; gb[k].z += d.z; gb[k].w += d.w;
        g[k] = make_float4(d.x * w.x, d.y * w.y, d.z * w.z, d.w * w.w);
        m1 += (g[k].x + g[k].y) + (g[k].z + g[k].w);
        m2 += n8_dot(g[k], xh[k]);
      }
    }
    // two buffers in turn: a wave may be a row ahead of the slowest, never two
    const float2 m = n8_block_sums(m1, m2, red[r & 1]);
    m1 = m.x * inv_d;
    m2 = m.y * inv_d;
#pragma unroll
    for (int k = 0; k < D4; ++k) {
      const int c = tid + kE8Threads * k;
      if (c < d4)
        reinterpret_cast<float4*>(a.dx)[r * d4 + c] =
            make_float4(st.y * (g[k].x - m1 - xh[k].x * m2) + dr[k].x, st.y * (g[k].y - m1 - xh[k].y * m2) + dr[k].y,
                        st.y * (g[k].z - m1 - xh[k].z * m2) + dr[k].z, st.y * (g[k].w - m1 - xh[k].w * m2) + dr[k].w);
    }
  }
  float4* out = reinterpret_cast<float4*>(a.partial) + (int64_t)blockIdx.x * 2 * d4;
#pragma unroll
  for (int k = 0; k < D4; ++k) {
    const int c = tid + kE8Threads * k;
    if (c < d4) {
      out[c] = gw[k];
      out[d4 + c] = gb[k];
    }
  }
}

// y again from x8 and the statistics, as columns of a causal window: out[b, t, c k + j] = y[b, t + j - (k - 1), c], 0
// before a text's start. For k = 1 and 4 a thread takes 4 channels of kN8Run tokens in a row and reads each token once,
// all in flight (16384 x 768 bf16 with a token a thread: 17 and 37 us); any other k a token at a time.
constexpr int kN8Run = 8;
template <bool O16, int K>
__global__ __launch_bounds__(kE8Threads) void k_norm8_run(N8Args a) {
  const int d4 = a.d >> 2;
  const int64_t runs = (a.L + kN8Run - 1) / kN8Run, texts = a.rows / a.L;
  const int64_t i = (int64_t)blockIdx.x * kE8Threads + threadIdx.x;
  if (i >= texts * runs * d4) return;
  const int64_t run = (uint32_t)i / (uint32_t)d4;       // lanes < 2^32
  const int c = (int)(i - run * d4);
  const int64_t b = (uint32_t)run / (uint32_t)runs, t0 = (run - b * runs) * kN8Run, r0 = b * a.L;
  const float4 w = reinterpret_cast<const float4*>(a.gamma)[c], z = reinterpret_cast<const float4*>(a.beta)[c];
  uint32_t q[kN8Run + K - 1], e[kN8Run + K - 1];
  float2 st[kN8Run + K - 1];
  float4 v[kN8Run + K - 1];
#pragma unroll
  for (int j = 0; j < kN8Run + K - 1; ++j) {            // tokens outside the text read its nearest, not used
    int64_t t = t0 + j - (K - 1);
    t = t < 0 ? 0 : t < a.L ? t : a.L - 1;
    q[j] = a.q[(r0 + t) * d4 + c];
    e[j] = a.e[(r0 + t) * a.groups + (c >> 3)];
    st[j] = a.stats[r0 + t];
  }
#pragma unroll
  for (int j = 0; j < kN8Run + K - 1; ++j) {
    const float4 x = e8_open(q[j], e8_scale(e[j]));
    v[j] = make_float4((x.x - st[j].x) * st[j].y * w.x + z.x, (x.y - st[j].x) * st[j].y * w.y + z.y,
                       (x.z - st[j].x) * st[j].y * w.z + z.z, (x.w - st[j].x) * st[j].y * w.w + z.w);
    if (t0 + j < K - 1) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int u = 0; u < kN8Run; ++u) {
    if (t0 + u >= a.L) break;
    const int64_t at = (r0 + t0 + u) * d4 + c;          // in groups of 4 channels
    if constexpr (K == 1) {
      n8_store<O16>(a.y, at, v[u]);
    } else {
      n8_store<O16>(a.y, 4 * at, make_float4(v[u].x, v[u + 1].x, v[u + 2].x, v[u + 3].x));
      n8_store<O16>(a.y, 4 * at + 1, make_float4(v[u].y, v[u + 1].y, v[u + 2].y, v[u + 3].y));
      n8_store<O16>(a.y, 4 * at + 2, make_float4(v[u].z, v[u + 1].z, v[u + 2].z, v[u + 3].z));
      n8_store<O16>(a.y, 4 * at + 3, make_float4(v[u].w, v[u + 1].w, v[u + 2].w, v[u + 3].w));
    }
  }
}

template <bool O16>
__global__ __launch_bounds__(kE8Threads) void k_norm8_read(N8Args a) {
  const int d4 = a.d >> 2;
  const int64_t i = (int64_t)blockIdx.x * kE8Threads + threadIdx.x;
  if (i >= a.rows * d4) return;
  const int64_t r = (uint32_t)i / (uint32_t)d4;         // lanes < 2^32
  const int c = (int)(i - r * d4);
  const int64_t t = (uint32_t)r % (uint32_t)a.L;       // rows, L < 2^31
  const float4 w = reinterpret_cast<const float4*>(a.gamma)[c], b = reinterpret_cast<const float4*>(a.beta)[c];
  for (int j = 0; j < a.k; ++j) {
    const int64_t back = a.k - 1 - j;
    const bool in = back <= t;
    const int64_t s = r - (in ? back : 0);
    const float2 st = a.stats[s];
    const float4 x = e8_open(a.q[s * d4 + c], e8_scale(a.e[s * a.groups + (c >> 3)]));
    const float v[4] = {(x.x - st.x) * st.y * w.x + b.x, (x.y - st.x) * st.y * w.y + b.y, (x.z - st.x) * st.y * w.z + b.z,
                        (x.w - st.x) * st.y * w.w + b.w};
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int64_t at = (r * a.d + 4 * c + h) * a.k + j;
      const float o = in ? v[h] : 0.f;
      if constexpr (O16) reinterpret_cast<uint16_t*>(a.y)[at] = (uint16_t)e8_pack_bf16(o, 0.f);
      else reinterpret_cast<float*>(a.y)[at] = o;
    }
  }
}

// a launch has fewer than 2^32 threads
constexpr int64_t kE8Lanes = (int64_t(1) << 32) - kE8Threads;

static int e8_groups(int64_t d) { return (int)((d + kE8Group - 1) / kE8Group); }

static int e8_setup(E8Args& a, int64_t rows, int64_t d, const char* what) {
  ASRN_REQUIRE(rows >= 0 && d >= 1 && d < (int64_t(1) << 28) && rows < (int64_t(1) << 40) &&
                   (rows == 0 || d < (int64_t(1) << 38) / rows),
               "%s: bad sizes rows=%lld d=%lld", what, (long long)rows, (long long)d);
  a.rows = rows; a.d = (int)d; a.groups = e8_groups(d); a.lanes = rows * a.groups * 4;
  ASRN_REQUIRE(a.lanes <= kE8Lanes, "%s: too many values (%lld x %lld)", what, (long long)rows, (long long)d);
  return 0;
}
static int n8_check(const N8Args& a, const char* what) {
  ASRN_REQUIRE(a.rows >= 0 && a.d > 0 && a.d % 4 == 0 && a.d <= kE8MaxD &&
                   a.rows <= (a.d <= kE8WaveD ? kE8Lanes / 32 : kE8Lanes / kE8Threads),
               "%s: bad sizes rows=%lld d=%d (a multiple of 4, <= %d)", what, (long long)a.rows, a.d, kE8MaxD);
  return 0;
}
static bool e8_aligned(const void* p, unsigned to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace asrn

using namespace asrn;

#define E8_WHOLE(CALL) if (a.d % kE8Group == 0) { CALL(true); } else { CALL(false); }
#define E8_GRID dim3((unsigned)((a.lanes + kE8Threads - 1) / kE8Threads)), dim3(kE8Threads), 0, st, a

extern "C" int asrn_pack8(const void* x, int32_t x_bf16, int64_t rows, int64_t d, int8_t* q, uint8_t* e, void* stream) {
  E8Args a{};
  if (e8_setup(a, rows, d, "asrn_pack8")) return 1;
  if (rows == 0) return 0;
  ASRN_REQUIRE(x && q && e, "asrn_pack8: null pointer");
  a.u = x; a.q = q; a.e = e;
  hipStream_t st = (hipStream_t)stream;
#define E8_P(W)                                                                           \
  if (x_bf16) hipLaunchKernelGGL((k_gelu8_fwd<true, kE8Pack, false, W>), E8_GRID);        \
  else hipLaunchKernelGGL((k_gelu8_fwd<false, kE8Pack, false, W>), E8_GRID)
  E8_WHOLE(E8_P)
#undef E8_P
  return check_launch("asrn_pack8");
}

extern "C" int asrn_unpack8(const int8_t* q, const uint8_t* e, int64_t rows, int64_t d, int32_t gelu, int32_t out_bf16,
                            void* out, void* stream) {
  E8Args a{};
  if (e8_setup(a, rows, d, "asrn_unpack8")) return 1;
  if (rows == 0) return 0;
  ASRN_REQUIRE(out && q && e, "asrn_unpack8: null pointer");
  a.q = const_cast<int8_t*>(q); a.e = const_cast<uint8_t*>(e); a.out = out;
  hipStream_t st = (hipStream_t)stream;
#define E8_U2(W, OP)                                                                      \
  if (out_bf16) hipLaunchKernelGGL((k_gelu8_bwd<true, false, OP, W>), E8_GRID);           \
  else hipLaunchKernelGGL((k_gelu8_bwd<false, false, OP, W>), E8_GRID)
#define E8_U(W) if (gelu) { E8_U2(W, kE8ReadGelu); } else { E8_U2(W, kE8Read); }
  E8_WHOLE(E8_U)
#undef E8_U
#undef E8_U2
  return check_launch("asrn_unpack8");
}

extern "C" int asrn_gelu8_fwd(const void* u, int32_t u_bf16, const float* h, int64_t rows, int64_t d, void* out, int8_t* q,
                              uint8_t* e, void* stream) {
  E8Args a{};
  if (e8_setup(a, rows, d, "asrn_gelu8_fwd")) return 1;
  if (rows == 0) return 0;
  ASRN_REQUIRE(u && out && q && e, "asrn_gelu8_fwd: null pointer");
  a.u = u; a.h = h; a.out = out; a.q = q; a.e = e;
  hipStream_t st = (hipStream_t)stream;
#define E8_F2(W, B)                                                                       \
  if (h) hipLaunchKernelGGL((k_gelu8_fwd<B, kE8Gelu, true, W>), E8_GRID);                 \
  else hipLaunchKernelGGL((k_gelu8_fwd<B, kE8Gelu, false, W>), E8_GRID)
#define E8_F(W) if (u_bf16) { E8_F2(W, true); } else { E8_F2(W, false); }
  E8_WHOLE(E8_F)
#undef E8_F
#undef E8_F2
  return check_launch("asrn_gelu8_fwd");
}

extern "C" int asrn_gelu8_bwd(const int8_t* q, const uint8_t* e, const void* dy, int32_t dy_bf16, int64_t rows, int64_t d,
                              int32_t du_bf16, void* du, void* stream) {
  E8Args a{};
  if (e8_setup(a, rows, d, "asrn_gelu8_bwd")) return 1;
  if (rows == 0) return 0;
  ASRN_REQUIRE(q && e && dy && du, "asrn_gelu8_bwd: null pointer");
  a.q = const_cast<int8_t*>(q); a.e = const_cast<uint8_t*>(e); a.dy = dy; a.out = du;
  hipStream_t st = (hipStream_t)stream;
#define E8_B2(W, O)                                                                       \
  if (dy_bf16) hipLaunchKernelGGL((k_gelu8_bwd<O, true, kE8Grad, W>), E8_GRID);           \
  else hipLaunchKernelGGL((k_gelu8_bwd<O, false, kE8Grad, W>), E8_GRID)
#define E8_B(W) if (du_bf16) { E8_B2(W, true); } else { E8_B2(W, false); }
  E8_WHOLE(E8_B)
#undef E8_B
#undef E8_B2
  return check_launch("asrn_gelu8_bwd");
}

#define N8_ONE(KERNEL, D4, B16)                                                           \
  if (B16) hipLaunchKernelGGL((KERNEL<D4, true>), grid, block, 0, st, a);                 \
  else hipLaunchKernelGGL((KERNEL<D4, false>), grid, block, 0, st, a)
#define N8_SWITCH(KERNEL, B16)                                                            \
  switch ((a.d + 4 * kWave - 1) / (4 * kWave)) {                                          \
    case 1: N8_ONE(KERNEL, 1, B16); break;                                                \
    case 2: N8_ONE(KERNEL, 2, B16); break;                                                \
    case 3: N8_ONE(KERNEL, 3, B16); break;                                                \
    case 4: N8_ONE(KERNEL, 4, B16); break;                                                \
    default:                                                                              \
      if (a.d <= 2048) { N8_ONE(KERNEL##_wide, 2, B16); }                                 \
      else if (a.d <= 4096) { N8_ONE(KERNEL##_wide, 4, B16); }                            \
      else { N8_ONE(KERNEL##_wide, 8, B16); }                                             \
  }

extern "C" int asrn_norm8_fwd(const float* x, const float* gamma, const float* beta, int64_t rows, int32_t d, float eps,
                              int32_t out_bf16, void* y, float* stats, int8_t* q, uint8_t* e, void* stream) {
  N8Args a{};
  a.x = x; a.gamma = gamma; a.beta = beta; a.rows = rows; a.d = d; a.eps = eps; a.y = y;
  a.stats = reinterpret_cast<float2*>(stats); a.q = reinterpret_cast<uint32_t*>(q); a.e = e; a.groups = e8_groups(d);
  if (n8_check(a, "asrn_norm8_fwd")) return 1;
  ASRN_REQUIRE(eps > 0.f, "asrn_norm8_fwd: eps must be positive");
  if (rows == 0) return 0;
  ASRN_REQUIRE(x && gamma && beta && y && stats && q && e, "asrn_norm8_fwd: null pointer");
  ASRN_REQUIRE(e8_aligned(x, 16) && e8_aligned(gamma, 16) && e8_aligned(beta, 16) && e8_aligned(y, out_bf16 ? 8 : 16) &&
                   e8_aligned(q, 4) && e8_aligned(stats, 8),
               "asrn_norm8_fwd: rows and parameters must be 16-byte aligned (8 for bf16)");
  const int64_t per = d <= kE8WaveD ? kE8Waves * kN8FwdRows : 1;
  const dim3 grid((unsigned)((rows + per - 1) / per)), block(kE8Threads);
  hipStream_t st = (hipStream_t)stream;
  N8_SWITCH(k_norm8_fwd, out_bf16)
  return check_launch("asrn_norm8_fwd");
}

static int64_t n8_bwd_groups(int64_t rows) { return rows > 0 ? (rows + n8_bwd_rows(rows) - 1) / n8_bwd_rows(rows) : 1; }

extern "C" int64_t asrn_norm8_bwd_workspace(int64_t rows, int32_t d) {
  if (rows < 0 || d <= 0 || d > kE8MaxD || rows >= (int64_t(1) << 31)) return -1;
  const int64_t groups = n8_bwd_groups(rows), part = (groups * 2 * d * 4 + 255) / 256 * 256;
  const int64_t sums = asrn_column_sums_workspace(groups, 2 * (int64_t)d);
  return sums < 0 ? -1 : part + sums;
}

extern "C" int asrn_norm8_bwd(const int8_t* q, const uint8_t* e, const float* gamma, const float* stats, int64_t rows,
                              int32_t d, const void* dy, int32_t dy_bf16, const float* dres, float* dx, float* dparams,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  N8Args a{};
  a.gamma = gamma; a.rows = rows; a.d = d; a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.q = reinterpret_cast<uint32_t*>(const_cast<int8_t*>(q)); a.e = const_cast<uint8_t*>(e); a.groups = e8_groups(d);
  a.dy = dy; a.dres = dres; a.dx = dx; a.partial = (float*)workspace; a.per = n8_bwd_rows(rows);
  if (n8_check(a, "asrn_norm8_bwd")) return 1;
  const int64_t need = asrn_norm8_bwd_workspace(rows, d);
  ASRN_REQUIRE(need >= 0 && workspace && workspace_bytes >= need && e8_aligned(workspace, 256),
               "asrn_norm8_bwd: needs a 256-byte aligned workspace of %lld bytes", (long long)need);
  ASRN_REQUIRE(dparams, "asrn_norm8_bwd: null pointer");
  if (rows == 0)
    return asrn_column_sums(nullptr, 0, 0, 2 * (int64_t)d, 2 * (int64_t)d, dparams, nullptr, 0, stream);
  ASRN_REQUIRE(q && e && gamma && stats && dy && dx, "asrn_norm8_bwd: null pointer");
  ASRN_REQUIRE(e8_aligned(gamma, 16) && e8_aligned(dy, dy_bf16 ? 8 : 16) && e8_aligned(dres, 16) && e8_aligned(dx, 16) &&
                   e8_aligned(q, 4) && e8_aligned(stats, 8),
               "asrn_norm8_bwd: rows and parameters must be 16-byte aligned (8 for bf16)");
  const int64_t groups = n8_bwd_groups(rows);
  const dim3 grid((unsigned)groups), block(kE8Threads);
  hipStream_t st = (hipStream_t)stream;
  N8_SWITCH(k_norm8_bwd, dy_bf16)
  if (check_launch("asrn_norm8_bwd")) return 1;
  // one launch for up to 1,024 partial rows; more are summed in two levels
  if (groups <= 1024) return group_sums(a.partial, (int)groups, 2 * d, dparams, st);
  const int64_t part = (groups * 2 * d * 4 + 255) / 256 * 256;
  return asrn_column_sums(a.partial, 0, groups, 2 * (int64_t)d, 2 * (int64_t)d, dparams, (char*)workspace + part, need - part,
                          stream);
}

extern "C" int asrn_norm8_read(const int8_t* q, const uint8_t* e, const float* gamma, const float* beta, const float* stats,
                               int64_t B, int64_t L, int32_t d, int32_t k, int32_t out_bf16, void* out, void* stream) {
  N8Args a{};
  a.gamma = gamma; a.beta = beta; a.rows = B * L; a.d = d; a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.q = reinterpret_cast<uint32_t*>(const_cast<int8_t*>(q)); a.e = const_cast<uint8_t*>(e); a.groups = e8_groups(d);
  a.y = out; a.L = L; a.k = k;
  ASRN_REQUIRE(B >= 0 && L >= 0 && B < (int64_t(1) << 31) && L < (int64_t(1) << 31) && k >= 1 && k <= 16,
               "asrn_norm8_read: bad sizes B=%lld L=%lld k=%d (1 to 16)", (long long)B, (long long)L, k);
  if (n8_check(a, "asrn_norm8_read")) return 1;
  if (a.rows == 0) return 0;
  ASRN_REQUIRE(q && e && gamma && beta && stats && out, "asrn_norm8_read: null pointer");
  ASRN_REQUIRE(e8_aligned(gamma, 16) && e8_aligned(beta, 16) && e8_aligned(out, out_bf16 ? 8 : 16) && e8_aligned(q, 4) &&
                   e8_aligned(stats, 8),
               "asrn_norm8_read: rows and parameters must be 16-byte aligned (8 for bf16)");
  const bool run = k == 1 || k == 4;
  const int64_t lanes = (run ? B * ((L + kN8Run - 1) / kN8Run) : a.rows) * (d / 4);
  const int64_t blocks = (lanes + kE8Threads - 1) / kE8Threads;
  ASRN_REQUIRE(lanes <= kE8Lanes, "asrn_norm8_read: too many values");
  hipStream_t st = (hipStream_t)stream;
  if (run) {
    const dim3 grid((unsigned)blocks), block(kE8Threads);
    if (k == 1 && out_bf16) hipLaunchKernelGGL((k_norm8_run<true, 1>), grid, block, 0, st, a);
    else if (k == 1) hipLaunchKernelGGL((k_norm8_run<false, 1>), grid, block, 0, st, a);
    else if (out_bf16) hipLaunchKernelGGL((k_norm8_run<true, 4>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_norm8_run<false, 4>), grid, block, 0, st, a);
    return check_launch("asrn_norm8_read");
  }
  if (out_bf16) hipLaunchKernelGGL(k_norm8_read<true>, dim3((unsigned)blocks), dim3(kE8Threads), 0, st, a);
  else hipLaunchKernelGGL(k_norm8_read<false>, dim3((unsigned)blocks), dim3(kE8Threads), 0, st, a);
  return check_launch("asrn_norm8_read");
}
