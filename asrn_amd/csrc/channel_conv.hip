// The causal convolution of each channel with its bias and activation: y[b, t, c] = act(bias[c] + sum_j w[c, j]
// z[b, t - (k - 1) + j, c]), zeros before a text's start; its backward and one token's step.
//
// A lane takes V neighbouring channels of one piece of a text and walks along it, the last k - 1 rows of z in registers:
// z is read once, y written once. The backward walks the same way: it forms the pre-activation again from z, with it the
// gradient before the activation, g[t], keeps the last k - 1 of those too, and writes dz[t - (k - 1)] = sum_j w[c, j]
// g[t - j] while it gathers dw and dbias of its piece; it reads k - 1 rows past the piece's end. One partial row a piece,
// added in order (group_sums): no atomics. Both are bound by memory: 8 x 2048 x 768 bf16 with k = 4 and SiLU takes 15 us (3.4
// TB/s) and 27 (2.8 TB/s, and 5 for the pieces' sums).
#include "types.h"

namespace asrn {

constexpr int kConvThreads = 256;

struct ChannelConv {
  const void* z;
  int64_t zb, zt;                 // strides of z's texts and tokens in elements; the channels lie next to each other
  const float* w;                 // (d, k)
  const float* bias;              // (d) or null
  const void* g;                  // the output's gradient, dense
  void* out;                      // y, or dz: dense
  float* part;                    // backward: (B pieces, (k + 1) d), dw[c, j] at j d + c, then dbias
  int64_t B, L;
  int d, k, act, piece, pieces, groups;   // a piece's tokens, pieces a text, groups of V channels
};

// The taps of a lane's V channels, w[j][v]: channel v's tap j, j < K. EXACT (k = K, V = 4): its 4 K floats are 16-byte vectors
// next to each other; else tap by tap, 0 past k.
template <int V, int K, bool EXACT>
__device__ __forceinline__ void load_taps(const float* w, int k, float (&t)[K][V]) {
  if constexpr (EXACT) {
    float f[V * K];
#pragma unroll
    for (int i = 0; i < V * K / 4; ++i) {
      const float4 q = reinterpret_cast<const float4*>(w)[i];
      f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < K; ++j) t[j][v] = f[v * K + j];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < K; ++j) t[j][v] = j < k ? w[v * k + j] : 0.f;
  }
}

// K: the taps that the registers hold, k <= K (EXACT: k = K). The taps past k are skipped by a uniform branch. The register of
// the tap j tokens back is w[k - 1 - j]: w is read reversed, so that its number does not depend on k.
template <typename T, int V, int K, bool EXACT>
__global__ __launch_bounds__(kConvThreads) void k_channel_conv(ChannelConv a) {
  constexpr int R = 8;
  const int64_t i = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
  const int64_t row = i / a.groups;
  const int64_t b = row / a.pieces;
  if (b >= a.B) return;
  const int c = (int)(i % a.groups) * V, k = EXACT ? K : a.k;
  const int64_t t0 = (row % a.pieces) * a.piece, t1 = t0 + a.piece < a.L ? t0 + a.piece : a.L;
  const T* z = static_cast<const T*>(a.z) + b * a.zb + c;
  T* y = static_cast<T*>(a.out) + b * a.L * a.d + c;
  float w[K][V], bias[V], x[K - 1 + R][V];          // w[j]: the tap j tokens back
  if constexpr (EXACT) {
    float t[K][V];
    load_taps<V, K, true>(a.w + (int64_t)c * K, K, t);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) w[j][v] = t[K - 1 - j][v];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][v] = j < k ? a.w[(int64_t)(c + v) * k + k - 1 - j] : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[c + v] : 0.f;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {                 // x[j]: token t0 - (K - 1) + j
    const int64_t t = t0 - (K - 1) + j;
    if (t >= 0 && K - 1 - j < k) load_v<V>(z + t * a.zt, x[j]);
    else
#pragma unroll
      for (int v = 0; v < V; ++v) x[j][v] = 0.f;
  }
  for (int64_t t = t0; t < t1; t += R) {
#pragma unroll
    for (int r = 0; r < R; ++r)                     // past the end: the last row again, its result not stored
      load_v<V>(z + (t + r < t1 ? t + r : t1 - 1) * a.zt, x[K - 1 + r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[V];
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = bias[v];
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (j < k)
#pragma unroll
          for (int v = 0; v < V; ++v) s[v] = fmaf(w[j][v], x[K - 1 + r - j][v], s[v]);
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = activate(s[v], a.act);
      if (t + r < t1) store_v<V>(y + (t + r) * a.d, s);
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) x[j][v] = x[R + j][v];
  }
}

template <typename T, int V, int K, bool EXACT>
__global__ __launch_bounds__(kConvThreads) void k_channel_conv_bwd(ChannelConv a) {
  constexpr int R = 4;
  const int64_t i = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
  const int64_t row = i / a.groups;
  const int64_t b = row / a.pieces;
  if (b >= a.B) return;
  const int c = (int)(i % a.groups) * V, k = EXACT ? K : a.k;
  const int64_t t0 = (row % a.pieces) * a.piece, t1 = t0 + a.piece < a.L ? t0 + a.piece : a.L;
  const int64_t end = t1 + k - 1 < a.L ? t1 + k - 1 : a.L;       // the tokens whose g this piece's dz needs
  const T* z = static_cast<const T*>(a.z) + b * a.zb + c;
  const T* gy = static_cast<const T*>(a.g) + b * a.L * a.d + c;
  T* dz = static_cast<T*>(a.out) + b * a.L * a.d + c;
  float u[K][V], w[K][V], bias[V], dw[K][V], db[V], x[K - 1 + R][V], g[K - 1 + R][V];
  load_taps<V, K, EXACT>(a.w + (int64_t)c * k, k, u);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = a.bias ? a.bias[c + v] : 0.f;
    db[v] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      w[j][v] = EXACT ? u[K - 1 - j][v] : j < k ? a.w[(int64_t)(c + v) * k + k - 1 - j] : 0.f;     // the tap j tokens back
      dw[j][v] = 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const int64_t t = t0 - (K - 1) + j;
    if (t >= 0 && K - 1 - j < k) load_v<V>(z + t * a.zt, x[j]);
    else
#pragma unroll
      for (int v = 0; v < V; ++v) x[j][v] = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) g[j][v] = 0.f;
  }
  // tokens t0 .. t1 + k - 2; from the text's end on g is 0
  for (int64_t t = t0; t < t1 + k - 1; t += R) {
    float e[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t s = t + r < end ? t + r : end - 1;
      load_v<V>(z + s * a.zt, x[K - 1 + r]);
      load_v<V>(gy + s * a.d, e[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[V];
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = bias[v];
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (j < k)
#pragma unroll
          for (int v = 0; v < V; ++v) s[v] = fmaf(w[j][v], x[K - 1 + r - j][v], s[v]);
      const bool here = t + r < end, mine = t + r < t1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float q = here ? e[r][v] * activate_grad(s[v], a.act) : 0.f, m = mine ? q : 0.f;
        g[K - 1 + r][v] = q;
        db[v] += m;
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (j < k) dw[j][v] = mine ? fmaf(m, x[K - 1 + r - j][v], dw[j][v]) : dw[j][v];
      }
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (j < k)
#pragma unroll
          for (int v = 0; v < V; ++v) s[v] = fmaf(u[j][v], g[K - 1 + r - j][v], s[v]);
      const int64_t o = t + r - (k - 1);
      if (o >= t0 && o < t1) store_v<V>(dz + o * a.d, s);
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[j][v] = x[R + j][v];
        g[j][v] = g[R + j][v];
      }
  }
  float* p = a.part + row * (int64_t)(k + 1) * a.d + c;
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (j < k) store_v<V>(p + (int64_t)(k - 1 - j) * a.d, dw[j]);
  store_v<V>(p + (int64_t)k * a.d, db);
}

// One token: a lane takes a channel, its window of k - 1 values shifts by one.
template <typename T>
__global__ __launch_bounds__(kConvThreads) void k_channel_conv_step(const T* z, int64_t zb, const T* window, T* next,
                                                                    const float* w, const float* bias, int64_t n, int d,
                                                                    int k, int act, T* y) {
  const int64_t i = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
  if (i >= n) return;
  const int c = (int)(i % d);
  const T x = z[i / d * zb + c];
  const T* v = window + i * (k - 1);
  T* o = next + i * (k - 1);
  float s = bias ? bias[c] : 0.f;
  const float* wc = w + (int64_t)c * k;
  for (int j = 0; j < k - 1; ++j) {
    const T q = v[j];
    s = fmaf(wc[j], (float)q, s);
    if (j > 0) o[j - 1] = q;                        // read before it is written, also in place
  }
  if (k > 1) o[k - 2] = x;
  y[i] = (T)activate(fmaf(wc[k - 1], (float)x, s), act);
}

// A piece's tokens: enough lanes for 3 waves a SIMD, 16 at least for the k - 1 rows that a piece reads again. 8 x 2048 x 768 bf16,
// k = 4, forward / backward in us: pieces of 8 16.9 / 31.6, 16 15.0 / 27.4, 32 18.2 / 31.2, 64 26.8 / 44.4.
static int piece_of(int64_t B, int64_t L, int groups) {
  const int64_t want = (int64_t)3 * 1024 * kWave;
  int64_t p = (B * L * groups + want - 1) / want;
  p = (p + 7) / 8 * 8;
  return (int)(p < 16 ? 16 : p > 128 ? 128 : p);
}

static int vector_of(int32_t type, int d, const ChannelConv& a, bool bwd) {
  const uintptr_t al = (uintptr_t)type_bytes(type) * 4 - 1;
  const bool four = d % 4 == 0 && a.zb % 4 == 0 && a.zt % 4 == 0 && !((uintptr_t)a.z & al) && !((uintptr_t)a.out & al) &&
                    !((uintptr_t)a.g & al);
  return four && a.k <= (bwd ? 4 : 8) ? 4 : 1;
}

template <int V>
static void plan(ChannelConv& a) {
  a.groups = a.d / V;
  a.piece = piece_of(a.B, a.L, a.groups);
  a.pieces = (int)((a.L + a.piece - 1) / a.piece);
}

static int check(const ChannelConv& a, int32_t type, const char* what) {
  ASRN_REQUIRE(type_ok(type), "%s: type %d", what, type);
  ASRN_REQUIRE(a.B >= 0 && a.L >= 0 && a.d >= 1 && a.d < (1 << 24) && a.k >= 1 && a.k <= 16 && a.act >= 0 && a.act <= 2,
               "%s: bad sizes B=%lld L=%lld d=%d k=%d act=%d", what, (long long)a.B, (long long)a.L, a.d, a.k, a.act);
  ASRN_REQUIRE(a.B < (1 << 24) && a.L < ((int64_t)1 << 36) && a.B * a.L * a.d < ((int64_t)1 << 38), "%s: too many values",
               what);
  return 0;
}

}  // namespace asrn

using namespace asrn;

extern "C" int asrn_channel_conv_fwd(const void* z, int32_t type, int64_t stride_b, int64_t stride_t, const float* w,
                                     const float* bias, int64_t B, int64_t L, int32_t d, int32_t k, int32_t act, void* y,
                                     void* stream) {
  ChannelConv a = {z, stride_b, stride_t, w, bias, nullptr, y, nullptr, B, L, d, k, act, 0, 0, 0};
  if (check(a, type, "asrn_channel_conv_fwd")) return 1;
  if (B == 0 || L == 0) return 0;
  ASRN_REQUIRE(z && w && y, "asrn_channel_conv_fwd: null pointer");
  const int V = vector_of(type, d, a, false);
  if (V == 4) plan<4>(a);
  else plan<1>(a);
  const int64_t n = a.B * a.pieces * a.groups;
  ASRN_REQUIRE(grid_ok(n, kConvThreads), "asrn_channel_conv_fwd: too many texts and channels");
  const dim3 grid((unsigned)((n + kConvThreads - 1) / kConvThreads)), thr(kConvThreads);
  hipStream_t st = (hipStream_t)stream;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    if (V == 4) {
      if (k == 4 && !((uintptr_t)w & 15)) hipLaunchKernelGGL((k_channel_conv<T, 4, 4, true>), grid, thr, 0, st, a);
      else if (k <= 4) hipLaunchKernelGGL((k_channel_conv<T, 4, 4, false>), grid, thr, 0, st, a);
      else hipLaunchKernelGGL((k_channel_conv<T, 4, 8, false>), grid, thr, 0, st, a);
    } else {
      if (k <= 4) hipLaunchKernelGGL((k_channel_conv<T, 1, 4, false>), grid, thr, 0, st, a);
      else if (k <= 8) hipLaunchKernelGGL((k_channel_conv<T, 1, 8, false>), grid, thr, 0, st, a);
      else hipLaunchKernelGGL((k_channel_conv<T, 1, 16, false>), grid, thr, 0, st, a);
    }
    return check_launch("asrn_channel_conv_fwd");
  });
}

// The pieces are the vector width's too, so the size is that of the width with more of them.
extern "C" int64_t asrn_channel_conv_bwd_workspace(int64_t B, int64_t L, int32_t d, int32_t k) {
  if (B < 0 || L < 0 || d < 1 || k < 1 || k > 16) return -1;
  if (B == 0 || L == 0) return 0;
  ChannelConv a = {};
  a.B = B;
  a.L = L;
  a.d = d;
  plan<1>(a);
  int64_t most = a.pieces;
  if (d % 4 == 0) {
    plan<4>(a);
    if (a.pieces > most) most = a.pieces;
  }
  return B * most * (int64_t)(k + 1) * d * 4;
}

extern "C" int asrn_channel_conv_bwd(const void* z, int32_t type, int64_t stride_b, int64_t stride_t, const float* w,
                                     const float* bias, const void* dy, int64_t B, int64_t L, int32_t d, int32_t k,
                                     int32_t act, void* dz, float* dparams, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  ChannelConv a = {z, stride_b, stride_t, w, bias, dy, dz, (float*)workspace, B, L, d, k, act, 0, 0, 0};
  if (check(a, type, "asrn_channel_conv_bwd")) return 1;
  if (B == 0 || L == 0) return 0;
  ASRN_REQUIRE(z && w && dy && dz && dparams, "asrn_channel_conv_bwd: null pointer");
  const int V = vector_of(type, d, a, true);
  if (V == 4) plan<4>(a);
  else plan<1>(a);
  const int64_t rows = a.B * a.pieces, cols = (int64_t)(k + 1) * d;
  ASRN_REQUIRE(workspace && !((uintptr_t)workspace & 15) && workspace_bytes >= rows * cols * 4,
               "asrn_channel_conv_bwd: needs a 16-byte aligned workspace of %lld bytes (got %lld)",
               (long long)(rows * cols * 4), (long long)workspace_bytes);
  ASRN_REQUIRE(rows < (1 << 30) && cols < (1 << 30), "asrn_channel_conv_bwd: too many pieces");
  const int64_t n = rows * a.groups;
  ASRN_REQUIRE(grid_ok(n, kConvThreads), "asrn_channel_conv_bwd: too many texts and channels");
  const dim3 grid((unsigned)((n + kConvThreads - 1) / kConvThreads)), thr(kConvThreads);
  hipStream_t st = (hipStream_t)stream;
  const int rc = with_type(type, [&](auto t) {
    using T = decltype(t);
    if (V == 4) {
      if (k == 4 && !((uintptr_t)w & 15)) hipLaunchKernelGGL((k_channel_conv_bwd<T, 4, 4, true>), grid, thr, 0, st, a);
      else hipLaunchKernelGGL((k_channel_conv_bwd<T, 4, 4, false>), grid, thr, 0, st, a);
    } else {
      if (k <= 4) hipLaunchKernelGGL((k_channel_conv_bwd<T, 1, 4, false>), grid, thr, 0, st, a);
      else if (k <= 8) hipLaunchKernelGGL((k_channel_conv_bwd<T, 1, 8, false>), grid, thr, 0, st, a);
      else hipLaunchKernelGGL((k_channel_conv_bwd<T, 1, 16, false>), grid, thr, 0, st, a);
    }
    return check_launch("asrn_channel_conv_bwd");
  });
  return rc ? rc : group_sums(a.part, (int)rows, (int)cols, dparams, st);
}

extern "C" int asrn_channel_conv_step(const void* z, int32_t type, int64_t stride_b, const void* window, void* next,
                                      const float* w, const float* bias, int64_t B, int32_t d, int32_t k, int32_t act,
                                      void* y, void* stream) {
  ChannelConv a = {z, stride_b, 0, w, bias, nullptr, y, nullptr, B, 1, d, k, act, 0, 0, 0};
  if (check(a, type, "asrn_channel_conv_step")) return 1;
  if (B == 0) return 0;
  ASRN_REQUIRE(z && w && y && (k == 1 || (window && next)), "asrn_channel_conv_step: null pointer");
  const int64_t n = B * d;
  ASRN_REQUIRE(grid_ok(n, kConvThreads), "asrn_channel_conv_step: too many texts and channels");
  const dim3 grid((unsigned)((n + kConvThreads - 1) / kConvThreads)), thr(kConvThreads);
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_channel_conv_step<T>), grid, thr, 0, (hipStream_t)stream, (const T*)z, stride_b, (const T*)window,
                       (T*)next, w, bias, n, d, k, act, (T*)y);
    return check_launch("asrn_channel_conv_step");
  });
}
