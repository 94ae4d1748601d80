// The selective state space scan. For texts b, tokens t, channels c and states n:
//   delta = softplus(dl + bias) (or dl + bias),   h_t = exp(delta_t A) h_{t-1} + delta_t u_t B_t,
//   y_t = (sum_n C_t h_t + D u_t) silu(z_t)
// with A (d, N), B and C shared by the channels, h in fp32. Its backward and one token's step.
//
// A wave takes 64 channels of one text. For the tokens' values lane l is channel l; for the states a lane holds 4
// neighbouring channels (quad q = l / 4) by a quarter of the states (l % 4): what the channels share (B, C) and what the
// states share (delta, delta u) comes from LDS as vectors, the sum over the states is one exchange within the quad that
// leaves channel l in lane l again, and the sums over the channels that the backward needs (dB, dC) begin inside a lane.
// A wave's LDS is its own: no barriers in the forward.
// Every channel and state has its own decay, so there is no matrix product in it: what bounds it is the vector units' issue.
// A wave's token of 16 states a channel takes about 130 instructions forward (16 of them exponentials, of two slots each: 146
// slots; at the least the exponent's product, x B, two multiply-adds and an exponential a value, 96) and 404 backward; 65 to
// 80% of the issue slots are used.
// Measured, 16 states, bf16: 2 texts of 32768 tokens x 768 channels forward 398 us (a trace has 164 for the chunks' ends, 15 for
// their starts and 240 for all chunks), 8 texts of 2048 traced forward 124 and backward 276 (the tokens' kernel 207); the bytes
// at a copy's rate take 80, 20 and 36.
// Texts too few to fill the card are cut into chunks: each chunk's end state from a zero state and its sum of delta
// first, then the chunks' start states one after the other (exp(A sum delta) carries a state over a chunk), then all chunks
// at once. The backward does the same from the end with the states' gradients. A chunk is a multiple of kCheck
// tokens, where the forward of a training step leaves its state: the backward forms the states in between again in
// registers. Partial sums are added in a fixed order; the chunks are a function of the sizes alone.
#include <type_traits>

#include "types.h"

namespace asrn {

constexpr int kCheck = 8;         // tokens between two kept states; also the tile of the backward
constexpr int kTile = 16;         // tokens that the forward stages at once
constexpr int kMaxWaves = 4;      // of a workgroup, 64 channels each
constexpr int kMinChunk = 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Selective {
  const void *u, *dl, *z, *Bm, *Cm, *gy;                       // z may be null
  int64_t ub, ut, dlb, dlt, zb, zt, Bb, Bt, Cb, Ct, gb, gt;    // strides of texts and tokens in elements
  const float *A, *D, *bias, *h0;                              // D, bias, h0 may be null
  void* y;
  float* hend;                    // (B, d, N) or null
  float* check;                   // (B, ceil(L / kCheck), own) or null
  float* carry;                   // (B, chunks - 1, own): end states from zero, then the chunks' start states
  float* total;                   // (B, chunks, d): sums of delta
  int64_t B, L, chunk, own;       // own: floats of a state as the lanes hold it
  int d, N, chunks, softplus;
  // backward
  const float* ghend;             // (B, d, N) or null
  void *du, *ddl, *dz;
  float* dh0;                     // (B, d, N) or null
  float* bc;                      // (blocks, B L, 2, N): dB and dC of a workgroup's channels
  float* part;                    // (B chunks, d N + 2 d): dA, dD, dbias
};

// softplus(x) = max(x, 0) + log1p(exp(-|x|)); log1p(e) = 2 atanh(e / (2 + e)), whose series ends at s^15 / 15 of s <= 1/3
__device__ __forceinline__ float softplus_of(float x, float e) {
  const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
  float p = fmaf(q, 1.f / 15, 1.f / 13);
  p = fmaf(q, p, 1.f / 11);
  p = fmaf(q, p, 1.f / 9);
  p = fmaf(q, p, 1.f / 7);
  p = fmaf(q, p, 1.f / 5);
  p = fmaf(q, p, 1.f / 3);
  p = fmaf(q * s, p, s);
  return fmaxf(x, 0.f) + 2.f * p;
}
__device__ __forceinline__ float softplus(float x) { return softplus_of(x, exp_fast(-fabsf(x))); }
// and its derivative, 1 / (1 + exp(-x))
__device__ __forceinline__ float softplus(float x, float* slope) {
  const float e = exp_fast(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + e);
  *slope = x < 0.f ? e * r : r;
  return softplus_of(x, e);
}

// DPP within a quad: lane ^ 1 and lane ^ 2
__device__ __forceinline__ float quad_xor1(float v) { return dpp<0xB1>(v); }
__device__ __forceinline__ float quad_xor2(float v) { return dpp<0x4E>(v); }

// v[i] of channel i of the quad's four, partial over the quad's lanes -> lane i's sum of v[i]
__device__ __forceinline__ float quad_scatter(const float (&v)[4], int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
  const float r0 = (b0 ? v[1] : v[0]) + quad_xor1(b0 ? v[0] : v[1]);
  const float r1 = (b0 ? v[3] : v[2]) + quad_xor1(b0 ? v[2] : v[3]);
  return (b1 ? r1 : r0) + quad_xor2(b1 ? r0 : r1);
}

// a's sums over the wave's four rows of 16 lanes in lanes 0 .. 15 (and 16 .. 31), b's in lanes 32 .. 47 (and 48 .. 63)
__device__ __forceinline__ float rows_sum(float a, float b) {
#ifdef __HIP_DEVICE_COMPILE__
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  const unsigned h = __float_as_uint(__uint_as_float(q[0]) + __uint_as_float(q[1]));
  const auto r = __builtin_amdgcn_permlane16_swap(h, h, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
#else
  return a + b;
#endif
}

// What one wave's lanes write to LDS is read by its other lanes: in order in the hardware, and for the compiler here.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// x is formed here: the compiler would put a sum that only the loop's next turn reads off to its end, its terms in registers
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+v"(x)); }

// x[0 .. NPL) of LDS, NPL in {2, 4, 6, 8}
template <int NPL>
__device__ __forceinline__ void lds_vec(const float* p, float (&x)[NPL]) {
  if constexpr (NPL % 4 != 0) {
#pragma unroll
    for (int i = 0; i < NPL / 2; ++i) {
      const float2 v = reinterpret_cast<const float2*>(p)[i];
      x[2 * i] = v.x; x[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPL / 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(p)[i];
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    }
  }
}

// A wave's place: its 64 channels' number, lane l's own channel c, the lane's quad's channels q .. q + 3 and its states
// n0 .. n0 + NPL - 1
struct Place {
  int lane, wave, group, c, q, n0;
  bool live;
};
template <int NPL>
__device__ __forceinline__ Place place_of(const Selective& s) {
  Place p;
  p.lane = lane_id();
  p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  p.group = (int)blockIdx.x * (int)(blockDim.x >> 6) + p.wave;
  p.c = p.group * 64 + p.lane;
  p.q = p.group * 64 + (p.lane & ~3);
  p.n0 = (p.lane & 3) * NPL;
  p.live = p.c < s.d;
  return p;
}

// A in units of the binary exponent, finite: times a delta of 0 (past a chunk's end) an infinite one would not be 0
__device__ __forceinline__ float rate_of(float A) {
  const float x = A * kLog2e;
  return fabsf(x) == INFINITY ? copysignf(3.4e38f, x) : x;
}

// the lane's 4 x NPL values of a (d, N) array, 0 outside it; RATE: of A
template <int NPL, bool RATE = false>
__device__ __forceinline__ void load_state(const float* x, const Selective& s, const Place& p, float (&h)[4][NPL]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const float v = x && p.q + i < s.d && p.n0 + j < s.N ? x[(int64_t)(p.q + i) * s.N + p.n0 + j] : 0.f;
      h[i][j] = RATE ? rate_of(v) : v;
    }
}
template <int NPL>
__device__ __forceinline__ void store_state(float* x, const Selective& s, const Place& p, const float (&h)[4][NPL]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (p.q + i < s.d && p.n0 + j < s.N) x[(int64_t)(p.q + i) * s.N + p.n0 + j] = h[i][j];
}

// The kernels' own states (kept ones, carries) lie as the lanes hold them: per 64 channels 4 NPL x 64 floats, in vectors of
// V of a lane, padded channels and states among them (0).
template <int NPL>
struct Own {
  static constexpr int V = NPL % 4 ? 2 : 4, G = 4 * NPL / V;
  typedef float FV __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ void load(const float* x, const Place& p, float (&h)[4][NPL]) {
    const FV* v = reinterpret_cast<const FV*>(x) + (int64_t)p.group * 64 * G;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const FV w = v[(unsigned)(g * 64 + p.lane)];
#pragma unroll
      for (int k = 0; k < V; ++k) h[g * V / NPL][g * V % NPL + k] = w[k];
    }
  }
  static __device__ __forceinline__ void store(float* x, const Place& p, const float (&h)[4][NPL]) {
    FV* v = reinterpret_cast<FV*>(x) + (int64_t)p.group * 64 * G;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      FV w;
#pragma unroll
      for (int k = 0; k < V; ++k) w[k] = h[g * V / NPL][g * V % NPL + k];
      v[(unsigned)(g * 64 + p.lane)] = w;
    }
  }
  // the channel and the state of the i-th float
  static __device__ __forceinline__ void where(int64_t i, int64_t& c, int& n) {
    const int k = (int)(i % V), lane = (int)(i / V % 64), g = (int)(i / (V * 64) % G);
    c = i / (V * 64 * G) * 64 + (lane & ~3) + g * V / NPL;
    n = (lane & 3) * NPL + g * V % NPL + k;
  }
};

// the tokens of a tile of TT that begins at t of a chunk that ends at t1
template <int TT>
__device__ __forceinline__ int tokens_of(int64_t t, int64_t t1) {
  const int n = __builtin_amdgcn_readfirstlane((int)(t1 - t));       // opaque: compared as 64 bits, each use would fill a mask
  return n < TT ? n : TT;
}

// B or C of TT tokens from t on, the states padded with zeros to NP = 4 NPL: a wave's registers, then its LDS. Tokens past
// the chunk's end repeat its last.
template <typename T, int NPL, int TT>
struct Shared {
  static constexpr int NP = 4 * NPL, E = (TT * NP + 63) / 64;
  float x[E];
  __device__ __forceinline__ void load(const T* X, int64_t st, int64_t t, int64_t t1, int N, int lane) {
    const T* p = X + t * st;
    const int last = tokens_of<TT>(t, t1) - 1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = lane + 64 * e, n = i % NP;
      const int r = i / NP < last ? i / NP : last;
      const float v = (float)p[(unsigned)(r * (int)st + (n < N ? n : 0))];
      x[e] = n < N ? v : 0.f;
    }
  }
  __device__ __forceinline__ void store(float* l, int lane) const {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (TT * NP % 64 == 0 || lane + 64 * e < TT * NP) l[lane + 64 * e] = x[e];
  }
};

// A text's rows of channels from one token on, lane l at its channel: the row as the scalar offset of a buffer access (an
// address a row would fill the scalar registers). Lanes without a channel lie past the buffer's end: they read 0, so that
// their states stay 0 and nothing of theirs enters a sum, and what they store is dropped.
constexpr unsigned kBufferBytes = 1u << 30;
template <typename T>
struct Rows {
  __amdgpu_buffer_rsrc_t rsrc;
  unsigned at, step;
  __device__ __forceinline__ Rows(const T* row, int64_t st, const Place& p, bool on = true)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(row), 0, kBufferBytes, 0x00027000)),
        at(p.live && on ? p.c * (unsigned)sizeof(T) : kBufferBytes),
        // opaque: its multiples are formed where they are used, not kept over the tiles
        step(__builtin_amdgcn_readfirstlane((unsigned)st * (unsigned)sizeof(T))) {}
  __device__ __forceinline__ T load(unsigned row) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, row, 0));
    else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(rsrc, at, row, 0));
  }
  // without a branch: one between a tile's tokens would let the compiler put their sums off to its end
  __device__ __forceinline__ void store(T v, unsigned row, bool in) const {
    const unsigned to = in ? at : kBufferBytes;
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), rsrc, to, row, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), rsrc, to, row, 0);
  }
};

// lane l's channel of TT tokens from t on, of a text's rows; past the chunk's end its last token again
template <typename T, int TT>
__device__ __forceinline__ void load_channel(const T* rows, int64_t st, int64_t t, int64_t t1, const Place& p, T (&x)[TT]) {
  const Rows<T> q(rows + t * st, st, p);
  const int last = tokens_of<TT>(t, t1) - 1;
  unsigned row = 0;
#pragma unroll
  for (int r = 0; r < TT; ++r) {
    x[r] = q.load(row);
    row += r < last ? q.step : 0u;
  }
}

__device__ __forceinline__ float decay(float delta, float A2) { return __builtin_amdgcn_exp2f(delta * A2); }

// delta of a lane's TT tokens
template <typename T, int TT>
__device__ __forceinline__ void step_sizes(const T (&dl)[TT], float bias, bool sp, float (&delta)[TT]) {
  if (sp) {
#pragma unroll
    for (int r = 0; r < TT; ++r) delta[r] = softplus((float)dl[r] + bias);
  } else {
#pragma unroll
    for (int r = 0; r < TT; ++r) delta[r] = (float)dl[r] + bias;
  }
}

// The forward over one chunk. LOCAL: its end state from zero and its sum of delta only.
template <typename T, int NPL, bool LOCAL>
__global__ __launch_bounds__(64 * kMaxWaves) void k_selective(Selective s) {
  constexpr int NP = 4 * NPL, TT = kTile;
  __shared__ float lds[kMaxWaves][TT * (128 + 2 * NP)];
  const Place p = place_of<NPL>(s);
  const int64_t b = blockIdx.z, chunk = blockIdx.y, t0 = chunk * s.chunk, t1 = t0 + s.chunk < s.L ? t0 + s.chunk : s.L;
  float* sd = lds[p.wave];
  float *su = sd + TT * 64, *sB = su + TT * 64, *sC = sB + TT * NP;
  const int64_t dN = (int64_t)s.d * s.N, checks = (s.L + kCheck - 1) / kCheck;
  const T *pu = static_cast<const T*>(s.u) + b * s.ub, *pd = static_cast<const T*>(s.dl) + b * s.dlb,
          *pz = static_cast<const T*>(s.z) + b * s.zb, *pB = static_cast<const T*>(s.Bm) + b * s.Bb,
          *pC = static_cast<const T*>(s.Cm) + b * s.Cb;
  T* py = static_cast<T*>(s.y) + b * s.L * s.d;
  const bool gate = s.z != nullptr;
  float A2[4][NPL], h[4][NPL];
  load_state<NPL, true>(s.A, s, p, A2);
  if (!LOCAL && chunk) Own<NPL>::load(s.carry + (b * (s.chunks - 1) + chunk - 1) * s.own, p, h);
  else load_state<NPL>(!LOCAL && s.h0 ? s.h0 + b * dN : nullptr, s, p, h);
  const float bias = s.bias && p.live ? s.bias[p.c] : 0.f, D = s.D && p.live ? s.D[p.c] : 0.f;
  float sum = 0.f;
  T u[TT], dl[TT], z[TT];
  Shared<T, NPL, TT> mb, mc;
  auto load = [&](int64_t t) {
    load_channel<T, TT>(pu, s.ut, t, t1, p, u);
    load_channel<T, TT>(pd, s.dlt, t, t1, p, dl);
    mb.load(pB, s.Bt, t, t1, s.N, p.lane);
    if (!LOCAL) {
      if (gate) load_channel<T, TT>(pz, s.zt, t, t1, p, z);
      mc.load(pC, s.Ct, t, t1, s.N, p.lane);
    }
  };
  load(t0);
  for (int64_t t = t0; t < t1; t += TT) {
    wave_lds_fence();
    float delta[TT], du[TT], g[TT];   // du, g: D u and the gate of this tile, while u and z are loaded for the next
    const int left = tokens_of<TT>(t, t1);
    step_sizes<T, TT>(dl, bias, s.softplus != 0, delta);
    if (left < TT)                    // past the chunk's end a delta of 0 leaves the state as it is
#pragma unroll
      for (int r = 0; r < TT; ++r)
        if (r >= left) {
          delta[r] = 0.f;
          u[r] = (T)0.f;
        }
#pragma unroll
    for (int r = 0; r < TT; ++r) {
      sd[r * 64 + p.lane] = delta[r];
      su[r * 64 + p.lane] = delta[r] * (float)u[r];
      if (LOCAL) {
        sum += delta[r];
      } else {
        du[r] = D * (float)u[r];
        g[r] = gate ? (float)z[r] * sigmoid((float)z[r]) : 1.f;
      }
    }
    mb.store(sB, p.lane);
    if (!LOCAL) mc.store(sC, p.lane);
    wave_lds_fence();
    if (t + TT < t1) load(t + TT);
    const Rows<T> out(py + t * s.d, s.d, p);
    auto step = [&](int r) {
      if (!LOCAL && s.check && (r % kCheck) == 0 && r < left) Own<NPL>::store(s.check + (b * checks + (t + r) / kCheck) * s.own, p, h);
      float dt[4], x[4], B[NPL], C[NPL], y[4];
      lds_vec<4>(sd + r * 64 + (p.lane & ~3), dt);
      lds_vec<4>(su + r * 64 + (p.lane & ~3), x);
      lds_vec<NPL>(sB + r * NP + p.n0, B);
      if (!LOCAL) lds_vec<NPL>(sC + r * NP + p.n0, C);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          h[i][j] = fmaf(decay(dt[i], A2[i][j]), h[i][j], x[i] * B[j]);
          if (!LOCAL) y[i] = fmaf(h[i][j], C[j], y[i]);
        }
      }
      if (!LOCAL) {
        const float v = (quad_scatter(y, p.lane) + du[r]) * g[r];
        out.store((T)v, r * out.step, r < left);
      }
    };
#pragma unroll
    for (int r = 0; r < TT; ++r) step(r);
  }
  if (LOCAL) {
    Own<NPL>::store(s.carry + (b * (s.chunks - 1) + chunk) * s.own, p, h);
    if (p.live) s.total[(b * s.chunks + chunk) * s.d + p.c] = sum;
  } else if (s.hend && chunk == s.chunks - 1) {
    store_state<NPL>(s.hend + b * dN, s, p, h);
  }
}

// BACK false: the chunks' start states, in place of their end states from zero: carry[j] = the state that chunk j + 1 starts
// from. BACK: carry[j] holds the gradient that chunk j + 1 passes to the state before it from a zero gradient at its end, and
// becomes that of the state that chunk j ends in.
template <int NPL, bool BACK>
__global__ __launch_bounds__(256) void k_selective_carry(Selective s) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= s.B * s.own) return;
  const int64_t b = i / s.own, e = i % s.own;
  int64_t c;
  int n;
  Own<NPL>::where(e, c, n);
  if (c >= s.d || n >= s.N) return;               // stay 0
  const float A2 = rate_of(s.A[c * s.N + n]), *x0 = BACK ? s.ghend : s.h0;
  float h = x0 ? x0[(b * s.d + c) * s.N + n] : 0.f;
  float* x = s.carry + b * (s.chunks - 1) * s.own + e;
  const float* w = s.total + b * s.chunks * s.d + c;
  constexpr int R = 16;               // loads under way at once
  const int m = s.chunks - 1;
  for (int k0 = 0; k0 < m; k0 += R) {
    float v[R], t[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = k0 + r < m ? k0 + r : m - 1;
      const int64_t j = BACK ? m - 1 - k : k;
      v[r] = x[j * s.own];
      t[r] = w[(BACK ? j + 1 : j) * s.d];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (k0 + r < m) {
        const int64_t j = BACK ? m - 1 - (k0 + r) : k0 + r;
        h = fmaf(decay(t[r], A2), h, v[r]);
        x[j * s.own] = h;
      }
  }
}

// What a chunk passes back to the state before it, from a zero gradient at its end, and its sum of delta.
template <typename T, int NPL>
__global__ __launch_bounds__(64 * kMaxWaves) void k_selective_local_bwd(Selective s) {
  constexpr int NP = 4 * NPL, TT = kTile;
  __shared__ float lds[kMaxWaves][TT * (128 + NP)];
  const Place p = place_of<NPL>(s);
  const int64_t b = blockIdx.z, chunk = blockIdx.y + 1, t0 = chunk * s.chunk, t1 = t0 + s.chunk < s.L ? t0 + s.chunk : s.L;
  float* sd = lds[p.wave];
  float *sg = sd + TT * 64, *sC = sg + TT * 64;
  const T *pd = static_cast<const T*>(s.dl) + b * s.dlb, *pz = static_cast<const T*>(s.z) + b * s.zb,
          *pC = static_cast<const T*>(s.Cm) + b * s.Cb, *pg = static_cast<const T*>(s.gy) + b * s.gb;
  const bool gate = s.z != nullptr;
  float A2[4][NPL], g[4][NPL];
  load_state<NPL, true>(s.A, s, p, A2);
  load_state<NPL>(nullptr, s, p, g);
  const float bias = s.bias && p.live ? s.bias[p.c] : 0.f;
  float sum = 0.f;
  T gy[TT], dl[TT], z[TT];
  Shared<T, NPL, TT> mc;
  auto load = [&](int64_t t) {
    load_channel<T, TT>(pg, s.gt, t, t1, p, gy);
    load_channel<T, TT>(pd, s.dlt, t, t1, p, dl);
    if (gate) load_channel<T, TT>(pz, s.zt, t, t1, p, z);
    mc.load(pC, s.Ct, t, t1, s.N, p.lane);
  };
  int64_t t = t0 + (t1 - t0 - 1) / TT * TT;
  load(t);
  for (; t >= t0; t -= TT) {
    wave_lds_fence();
    float delta[TT];
    step_sizes<T, TT>(dl, bias, s.softplus != 0, delta);
    const int left = tokens_of<TT>(t, t1);
    if (left < TT)                    // past the chunk's end: no gradient, and a delta of 0 passes it on as it is
#pragma unroll
      for (int r = 0; r < TT; ++r)
        if (r >= left) {
          delta[r] = 0.f;
          gy[r] = z[r] = (T)0.f;
        }
#pragma unroll
    for (int r = 0; r < TT; ++r) {
      sd[r * 64 + p.lane] = delta[r];
      sum += delta[r];
    }
    if (gate) {
#pragma unroll
      for (int r = 0; r < TT; ++r) sg[r * 64 + p.lane] = (float)gy[r] * ((float)z[r] * sigmoid((float)z[r]));
    } else {
#pragma unroll
      for (int r = 0; r < TT; ++r) sg[r * 64 + p.lane] = (float)gy[r];
    }
    mc.store(sC, p.lane);
    wave_lds_fence();
    if (t > t0) load(t - TT);
    auto step = [&](int r) {
      float dt[4], x[4], C[NPL];
      lds_vec<4>(sd + r * 64 + (p.lane & ~3), dt);
      lds_vec<4>(sg + r * 64 + (p.lane & ~3), x);
      lds_vec<NPL>(sC + r * NP + p.n0, C);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NPL; ++j) g[i][j] = fmaf(x[i], C[j], g[i][j]) * decay(dt[i], A2[i][j]);
    };
#pragma unroll
    for (int r = TT - 1; r >= 0; --r) step(r);
  }
  Own<NPL>::store(s.carry + (b * (s.chunks - 1) + chunk - 1) * s.own, p, g);
  if (p.live) s.total[(b * s.chunks + chunk) * s.d + p.c] = sum;
}

// The backward over one chunk, a tile of kCheck tokens at a time from its end. A tile's values go to LDS, the next one's loads
// are on their way meanwhile. Its states are formed again from the kept one, half a tile at a time (the registers hold no more),
// then with G_t, the gradient of h_t, from the half's last token to its first:
//   G_t += gy_t C_t;  dC_t += gy_t h_t;  dB_t += G_t delta_t u_t;  d(delta u) = sum G_t B_t;
//   w = G_t exp(delta_t A) h_{t-1};  dA += w delta_t;  d delta += sum w A;  G_{t-1} = G_t exp(delta_t A)
// dB and dC are summed over the lane's 4 channels, then over a row of 16 lanes; the rows' and waves' sums through LDS.
template <typename T, int NPL>
__global__ __launch_bounds__(64 * kMaxWaves, NPL > 4 ? 1 : 2) void k_selective_bwd(Selective s) {
  constexpr int NP = 4 * NPL, TT = kCheck, HALF = TT / 2;
  constexpr int NJ = (NPL + 3) / 4;               // values of dB (and of dC) that a lane leaves of its row's sums
  __shared__ float lds[kMaxWaves][TT * (384 + 2 * NP)];
  __shared__ float red[2][TT][2][kMaxWaves][NP];  // in turns, so that a tile has one barrier
  const Place p = place_of<NPL>(s);
  const int waves = blockDim.x >> 6;
  const int64_t b = blockIdx.z, chunk = blockIdx.y, t0 = chunk * s.chunk, t1 = t0 + s.chunk < s.L ? t0 + s.chunk : s.L;
  float* sd = lds[p.wave];
  float *su = sd + TT * 64, *sg = su + TT * 64, *sB = sg + TT * 64, *sC = sB + TT * NP;
  float *lu = sC + TT * NP + p.lane, *ls = lu + TT * 64, *lz = ls + TT * 64;       // a lane's own
  const int64_t dN = (int64_t)s.d * s.N, checks = (s.L + kCheck - 1) / kCheck;
  const T *pu = static_cast<const T*>(s.u) + b * s.ub, *pd = static_cast<const T*>(s.dl) + b * s.dlb,
          *pz = static_cast<const T*>(s.z) + b * s.zb, *pB = static_cast<const T*>(s.Bm) + b * s.Bb,
          *pC = static_cast<const T*>(s.Cm) + b * s.Cb, *pg = static_cast<const T*>(s.gy) + b * s.gb;
  const bool gate = s.z != nullptr;
  float A2[4][NPL], dA[4][NPL], G[4][NPL];
  load_state<NPL, true>(s.A, s, p, A2);
  load_state<NPL>(nullptr, s, p, dA);
  if (chunk + 1 < s.chunks) Own<NPL>::load(s.carry + (b * (s.chunks - 1) + chunk) * s.own, p, G);
  else load_state<NPL>(s.ghend ? s.ghend + b * dN : nullptr, s, p, G);
  const float bias = s.bias && p.live ? s.bias[p.c] : 0.f, D = s.D && p.live ? s.D[p.c] : 0.f;
  float dD = 0.f, dbias = 0.f;
  const int cq = (p.lane >> 2) & 3;
  int turn = 0;
  T u[TT], dl[TT], z[TT], gy[TT];
  Shared<T, NPL, TT> mb, mc;
  auto load = [&](int64_t t) {
    load_channel<T, TT>(pu, s.ut, t, t1, p, u);
    load_channel<T, TT>(pd, s.dlt, t, t1, p, dl);
    load_channel<T, TT>(pg, s.gt, t, t1, p, gy);
    if (gate) load_channel<T, TT>(pz, s.zt, t, t1, p, z);
    mb.load(pB, s.Bt, t, t1, s.N, p.lane);
    mc.load(pC, s.Ct, t, t1, s.N, p.lane);
  };
  int64_t t = t0 + (t1 - t0 - 1) / TT * TT;
  load(t);
  for (; t >= t0; t -= TT) {
    const int left = tokens_of<TT>(t, t1);
    const float* check = s.check + (b * checks + t / kCheck) * s.own;
    wave_lds_fence();
    {
      float delta[TT], sig[TT];
      if (s.softplus) {
#pragma unroll
        for (int r = 0; r < TT; ++r) delta[r] = softplus((float)dl[r] + bias, &sig[r]);
      } else {
#pragma unroll
        for (int r = 0; r < TT; ++r) {
          delta[r] = (float)dl[r] + bias;
          sig[r] = 1.f;
        }
      }
      if (left < TT)                  // past the text's end: a delta of 0 leaves the state as it is, and no gradient enters a sum
#pragma unroll
        for (int r = 0; r < TT; ++r)
          if (r >= left) {
            delta[r] = sig[r] = 0.f;
            u[r] = gy[r] = z[r] = (T)0.f;
          }
#pragma unroll
      for (int r = 0; r < TT; ++r) {
        sd[r * 64 + p.lane] = delta[r];
        su[r * 64 + p.lane] = delta[r] * (float)u[r];
        lu[r * 64] = (float)u[r];
        ls[r * 64] = sig[r];
      }
      if (gate) {
#pragma unroll
        for (int r = 0; r < TT; ++r) {
          const float zf = (float)z[r], q = sigmoid(zf), gq = (float)gy[r] * q;
          sg[r * 64 + p.lane] = gq * zf;
          lz[r * 64] = gq * (1.f + zf * (1.f - q));
        }
      } else {
#pragma unroll
        for (int r = 0; r < TT; ++r) sg[r * 64 + p.lane] = (float)gy[r];
      }
      mb.store(sB, p.lane);
      mc.store(sC, p.lane);
    }
    wave_lds_fence();
    if (t > t0) load(t - TT);
    const int64_t o = (b * s.L + t) * s.d;
    const Rows<T> odu(static_cast<T*>(s.du) + o, s.d, p), odl(static_cast<T*>(s.ddl) + o, s.d, p), odz(static_cast<T*>(s.dz) + o, s.d, p, gate);
#pragma unroll
    for (int half = 1; half >= 0; --half) {
      float h[HALF + 1][4][NPL];
      Own<NPL>::load(check, p, h[0]);
      // the state after token r, from `from`
      auto again = [&](int r, const float (&from)[4][NPL], float (&to)[4][NPL]) __attribute__((always_inline)) {
        float dt[4], x[4], B[NPL];
        lds_vec<4>(sd + r * 64 + (p.lane & ~3), dt);
        lds_vec<4>(su + r * 64 + (p.lane & ~3), x);
        lds_vec<NPL>(sB + r * NP + p.n0, B);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < NPL; ++j) to[i][j] = fmaf(decay(dt[i], A2[i][j]), from[i][j], x[i] * B[j]);
        __builtin_amdgcn_sched_barrier(0);          // a step's LDS reads stay in it: the states leave few registers
      };
      if (half) {
#pragma unroll
        for (int r = 0; r < HALF; ++r) again(r, h[0], h[0]);
      }
#pragma unroll
      for (int r = 0; r < HALF; ++r) again(half * HALF + r, h[r], h[r + 1]);
      wave_lds_fence();   // the values are read, and the decays formed, again: kept from above they would fill the registers
#pragma unroll
      for (int k = HALF - 1; k >= 0; --k) {
        const int r = half * HALF + k;
        float dt[4], x[4], g[4], B[NPL], C[NPL], y[4], dx[4], dd[4], dB[NPL], dC[NPL];
        lds_vec<4>(sd + r * 64 + (p.lane & ~3), dt);
        lds_vec<4>(su + r * 64 + (p.lane & ~3), x);
        lds_vec<4>(sg + r * 64 + (p.lane & ~3), g);
        lds_vec<NPL>(sB + r * NP + p.n0, B);
        lds_vec<NPL>(sC + r * NP + p.n0, C);
#pragma unroll
        for (int j = 0; j < NPL; ++j) dB[j] = dC[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = dx[i] = dd[i] = 0.f;
#pragma unroll
          for (int j = 0; j < NPL; ++j) {
            const float G1 = fmaf(g[i], C[j], G[i][j]);
            y[i] = fmaf(h[k + 1][i][j], C[j], y[i]);
            dC[j] = fmaf(g[i], h[k + 1][i][j], dC[j]);
            dB[j] = fmaf(G1, x[i], dB[j]);
            dx[i] = fmaf(G1, B[j], dx[i]);
            G[i][j] = G1 * decay(dt[i], A2[i][j]);
            const float w = G[i][j] * h[k][i][j];
            dd[i] = fmaf(w, A2[i][j], dd[i]);
            dA[i][j] = fmaf(w, dt[i], dA[i][j]);
            pin(dA[i][j]);
          }
        }
        const float ys = quad_scatter(y, p.lane), ds = quad_scatter(dx, p.lane), dds = quad_scatter(dd, p.lane);
        const float delta = sd[r * 64 + p.lane], gg = sg[r * 64 + p.lane], uf = lu[r * 64];
        const float ddl = fmaf(dds, kLn2, ds * uf) * ls[r * 64];
        // past the text's end the state stays and w = G h: times an infinite decay's rate its sum may overflow, and 0 of it be NaN
        dbias += r < left ? ddl : 0.f;
        dD = fmaf(gg, uf, dD);
        odu.store((T)fmaf(ds, delta, gg * D), r * odu.step, r < left);
        odl.store((T)ddl, r * odl.step, r < left);
        odz.store((T)(fmaf(D, uf, ys) * lz[r * 64]), r * odz.step, r < left);
#pragma unroll
        for (int j = 0; j < NPL; ++j) {             // over the row's quads
          dB[j] += dpp<0x128>(dB[j]);
          dC[j] += dpp<0x128>(dC[j]);
          dB[j] += dpp<0x124>(dB[j]);
          dC[j] += dpp<0x124>(dC[j]);
        }
#pragma unroll
        for (int q = 0; q < NJ; ++q) {              // quad cq of the row leaves values 4 q + cq
          float vb = dB[4 * q], vc = dC[4 * q];
#pragma unroll
          for (int j = 1; j < 4; ++j)
            if (4 * q + j < NPL) {
              vb = cq == j ? dB[4 * q + j] : vb;
              vc = cq == j ? dC[4 * q + j] : vc;
            }
          // over the rows: dB's sum stays in the lower 32 lanes, dC's in the upper
          const float v = rows_sum(vb, vc);
          if (4 * q + cq < NPL && (p.lane & 16) == 0) red[turn][r][p.lane >> 5][p.wave][p.n0 + 4 * q + cq] = v;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < TT * 2 * NP; e += blockDim.x) {
      const int r = e / (2 * NP), k = e / NP % 2, n = e % NP;
      float v = red[turn][r][k][0][n];
      for (int w = 1; w < waves; ++w) v += red[turn][r][k][w][n];
      if (r < left && n < s.N) s.bc[((blockIdx.x * s.B + b) * s.L + t + r) * 2 * s.N + k * s.N + n] = v;
    }
    turn ^= 1;                                    // the next tile's sums are written elsewhere, those after it past its barrier
  }
  float* part = s.part + (b * s.chunks + chunk) * (dN + 2 * s.d);
  store_state<NPL>(part, s, p, dA);
  if (p.live) {
    part[dN + p.c] = dD;
    part[dN + s.d + p.c] = dbias;
  }
  if (s.dh0 && chunk == 0) store_state<NPL>(s.dh0 + b * dN, s, p, G);
}

// dB and dC: the workgroups' sums in order, in the tensors' type
template <typename T>
__global__ __launch_bounds__(256) void k_selective_shared(const float* bc, int blocks, int64_t rows, int N, T* dB, T* dC) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = rows * 2 * N;
  if (i >= n) return;
  float v = 0.f;
  for (int k = 0; k < blocks; ++k) v += bc[k * n + i];
  const int64_t row = i / (2 * N);
  const int e = (int)(i % (2 * N));
  if (e < N) dB[row * N + e] = (T)v;
  else dC[row * N + e - N] = (T)v;
}

// One token: 4 lanes a channel, each every fourth state.
template <typename T>
__global__ __launch_bounds__(256) void k_selective_step(Selective s, const float* h, float* next) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, q = i >> 2, b = q / s.d;
  const int ng = (int)(i & 3), c = (int)(q % s.d);
  const bool live = b < s.B;                      // whole quads: the exchange below stays within one
  const int64_t bb = live ? b : 0;
  const float dl = (float)static_cast<const T*>(s.dl)[bb * s.dlb + c] + (s.bias ? s.bias[c] : 0.f);
  const float u = (float)static_cast<const T*>(s.u)[bb * s.ub + c], delta = s.softplus ? softplus(dl) : dl;
  const T *Bm = static_cast<const T*>(s.Bm) + bb * s.Bb, *Cm = static_cast<const T*>(s.Cm) + bb * s.Cb;
  const float* hr = h + (bb * s.d + c) * s.N;
  float* hw = next + (bb * s.d + c) * s.N;
  float y = 0.f;
  for (int n = ng; n < s.N; n += 4) {
    const float x = fmaf(decay(delta, rate_of(s.A[(int64_t)c * s.N + n])), hr[n], delta * u * (float)Bm[n]);
    if (live) hw[n] = x;
    y = fmaf(x, (float)Cm[n], y);
  }
  y += quad_xor1(y);
  y += quad_xor2(y);
  if (live && ng == 0) {
    if (s.D) y = fmaf(s.D[c], u, y);
    if (s.z) {
      const float z = (float)static_cast<const T*>(s.z)[b * s.zb + c];
      y *= z * sigmoid(z);
    }
    static_cast<T*>(s.y)[q] = (T)y;
  }
}

// Waves of 64 channels a workgroup: at most kMaxWaves, spread evenly
static void grid_of(int d, int& waves, int& blocks) {
  const int n = (d + 63) / 64;
  blocks = (n + kMaxWaves - 1) / kMaxWaves;
  waves = (n + blocks - 1) / blocks;
  blocks = (n + waves - 1) / waves;
}

// Tokens of a chunk. A CU takes the workgroups in rounds of as many as fill its 4 SIMDs with one wave each, and walks a chunk's
// tokens twice when there are several (the local pass takes 3/4 of the other's time); the chunks' states are joined one
// after the other, about 0.4 tokens' time each. One wave a SIMD leaves about 2/5 of its time unused, two 1/5, three 1/10. Of the
// chunks that make 1 to 8 rounds, the one of the least time: 8 texts of 2048 tokens x 768 channels in chunks of 112 (1.8
// rounds) 445 us forward and backward, of 64 (3 rounds) 402; 2 prompts of 32768 in 208 (3.7 rounds) 453, in 256 (3.0) 402.
static int64_t chunk_of(int64_t B, int64_t L, int d) {
  int waves, blocks;
  grid_of(d, waves, blocks);
  static const float used[] = {0.f, 0.6f, 0.8f, 0.9f};
  const int64_t slots = 256 * 4 / waves, whole = (L + kTile - 1) / kTile * kTile;
  int64_t best = 0;
  float least = 0.f;
  auto rate = [&](int64_t c) {
    const int64_t n = (L + c - 1) / c, rounds = (B * blocks * n + slots - 1) / slots;
    const float t = rounds * (c + 6.f) / used[rounds < 3 ? rounds : 3] * (n > 1 ? 1.75f : 1.f) + 0.4f * n;
    if (best == 0 || t < least) {
      least = t;
      best = c;
    }
  };
  rate(whole);
  for (int r = 1; r <= 8; ++r) {
    const int64_t n = r * slots / (B * blocks);
    if (n < 2) continue;
    const int64_t c = ((L + n - 1) / n + kTile - 1) / kTile * kTile;
    rate(c < kMinChunk ? kMinChunk : c);
  }
  return best;
}
static int chunks_of(int64_t B, int64_t L, int d) {
  const int64_t c = chunk_of(B, L, d);
  return c > 0 ? (int)((L + c - 1) / c) : 0;
}

static int check(const Selective& s, int32_t type, const char* what) {
  ASRN_REQUIRE(type_ok(type), "%s: type %d", what, type);
  ASRN_REQUIRE(s.B >= 0 && s.L >= 0 && s.d >= 1 && s.d < (1 << 22) && s.N >= 1 && s.N <= 32,
               "%s: bad sizes B=%lld L=%lld d=%d N=%d (1 <= N <= 32)", what, (long long)s.B, (long long)s.L, s.d, s.N);
  ASRN_REQUIRE(s.B < 65536 && s.L < ((int64_t)1 << 30) && s.B * s.L < ((int64_t)1 << 36), "%s: too many tokens", what);
  // a tile's tokens are addressed in 32 bits
  for (int64_t st : {s.ut, s.dlt, s.zt, s.Bt, s.Ct, s.gt})
    ASRN_REQUIRE(st >= 0 && st < (1 << 24), "%s: a token stride of %lld: below 2^24 is needed", what, (long long)st);
  return 0;
}

template <typename F>
static int with_states(int N, F&& f) {
  if (N <= 8) return f(std::integral_constant<int, 2>{});
  if (N <= 16) return f(std::integral_constant<int, 4>{});
  if (N <= 24) return f(std::integral_constant<int, 6>{});
  return f(std::integral_constant<int, 8>{});
}

// a state as the lanes of all workgroups hold it, the last ones' waves without channels among them
static int64_t own_floats(int d, int N) {
  int waves, blocks;
  grid_of(d, waves, blocks);
  return (int64_t)blocks * waves * 64 * (N <= 8 ? 8 : N <= 16 ? 16 : N <= 24 ? 24 : 32);
}
static int64_t carry_bytes(int64_t B, int chunks, int d, int N) {
  return chunks > 1 ? (B * ((chunks - 1) * own_floats(d, N) + (int64_t)chunks * d) * 4 + 255) / 256 * 256 : 0;
}

}  // namespace asrn

using namespace asrn;

extern "C" int64_t asrn_selective_checks(int64_t B, int64_t L, int32_t d, int32_t N) {
  return B < 0 || L < 0 || d < 1 || N < 1 || N > 32 ? -1 : B * ((L + kCheck - 1) / kCheck) * own_floats(d, N);
}

extern "C" int64_t asrn_selective_fwd_workspace(int64_t B, int64_t L, int32_t d, int32_t N) {
  if (B < 0 || L < 0 || d < 1 || N < 1) return -1;
  if (B == 0 || L == 0) return 0;
  return carry_bytes(B, chunks_of(B, L, d), d, N);
}

extern "C" int asrn_selective_fwd(const void* u, const void* delta, const void* B_, const void* C_, const void* z,
                                  int32_t type, const int64_t* strides, const float* A, const float* D, const float* bias,
                                  const float* h0, int64_t B, int64_t L, int32_t d, int32_t N, int32_t softplus, void* y,
                                  float* hend, float* checks, void* workspace, int64_t workspace_bytes, void* stream) {
  Selective s = {};
  s.u = u; s.dl = delta; s.Bm = B_; s.Cm = C_; s.z = z;
  s.A = A; s.D = D; s.bias = bias; s.h0 = h0; s.y = y; s.hend = hend; s.check = checks;
  s.B = B; s.L = L; s.d = d; s.N = N; s.softplus = softplus;
  if (strides) {
    s.ub = strides[0]; s.ut = strides[1]; s.dlb = strides[2]; s.dlt = strides[3]; s.Bb = strides[4]; s.Bt = strides[5];
    s.Cb = strides[6]; s.Ct = strides[7]; s.zb = strides[8]; s.zt = strides[9];
  }
  if (check(s, type, "asrn_selective_fwd")) return 1;
  if (B == 0 || L == 0) return 0;
  ASRN_REQUIRE(u && delta && B_ && C_ && A && y && strides, "asrn_selective_fwd: null pointer");
  s.chunk = chunk_of(B, L, d);
  s.chunks = chunks_of(B, L, d);
  s.own = own_floats(d, N);
  ASRN_REQUIRE(s.chunks < 65536, "asrn_selective_fwd: too many chunks");
  ASRN_REQUIRE(!checks || grid_ok(B * L * 2 * N, 256), "asrn_selective_fwd: too many tokens for a backward");
  const int64_t need = carry_bytes(B, s.chunks, d, N);
  if (need) {
    ASRN_REQUIRE(workspace && workspace_bytes >= need && !((uintptr_t)workspace & 15),
                 "asrn_selective_fwd: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
                 (long long)workspace_bytes);
    s.carry = (float*)workspace;
    s.total = s.carry + B * (s.chunks - 1) * s.own;
  }
  int waves, blocks;
  grid_of(d, waves, blocks);
  hipStream_t st = (hipStream_t)stream;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return with_states(N, [&](auto npl) {
      constexpr int NPL = decltype(npl)::value;
      if (s.chunks > 1) {
        hipLaunchKernelGGL((k_selective<T, NPL, true>), dim3(blocks, s.chunks - 1, B), dim3(64 * waves), 0, st, s);
        hipLaunchKernelGGL((k_selective_carry<NPL, false>), dim3((unsigned)((B * s.own + 255) / 256)), dim3(256), 0, st, s);
      }
      hipLaunchKernelGGL((k_selective<T, NPL, false>), dim3(blocks, s.chunks, B), dim3(64 * waves), 0, st, s);
      return check_launch("asrn_selective_fwd");
    });
  });
}

static int64_t bc_floats(int64_t B, int64_t L, int d, int N) {
  int waves, blocks;
  grid_of(d, waves, blocks);
  return (blocks * B * L * 2 * N + 63) / 64 * 64;
}

extern "C" int64_t asrn_selective_bwd_workspace(int64_t B, int64_t L, int32_t d, int32_t N) {
  if (B < 0 || L < 0 || d < 1 || N < 1) return -1;
  if (B == 0 || L == 0) return 0;
  const int chunks = chunks_of(B, L, d);
  return carry_bytes(B, chunks, d, N) + bc_floats(B, L, d, N) * 4 + B * chunks * ((int64_t)d * N + 2 * d) * 4;
}

extern "C" int asrn_selective_bwd(const void* u, const void* delta, const void* B_, const void* C_, const void* z,
                                  const void* dy, int32_t type, const int64_t* strides, const float* A, const float* D,
                                  const float* bias, const float* checks, const float* dhend, int64_t B, int64_t L, int32_t d,
                                  int32_t N, int32_t softplus, void* du, void* ddelta, void* dB, void* dC, void* dz,
                                  float* dparams, float* dh0, void* workspace, int64_t workspace_bytes, void* stream) {
  Selective s = {};
  s.u = u; s.dl = delta; s.Bm = B_; s.Cm = C_; s.z = z; s.gy = dy;
  s.A = A; s.D = D; s.bias = bias; s.check = const_cast<float*>(checks); s.ghend = dhend;
  s.du = du; s.ddl = ddelta; s.dz = dz; s.dh0 = dh0;
  s.B = B; s.L = L; s.d = d; s.N = N; s.softplus = softplus;
  if (strides) {
    s.ub = strides[0]; s.ut = strides[1]; s.dlb = strides[2]; s.dlt = strides[3]; s.Bb = strides[4]; s.Bt = strides[5];
    s.Cb = strides[6]; s.Ct = strides[7]; s.zb = strides[8]; s.zt = strides[9]; s.gb = strides[10]; s.gt = strides[11];
  }
  if (check(s, type, "asrn_selective_bwd")) return 1;
  if (B == 0 || L == 0) return 0;
  ASRN_REQUIRE(u && delta && B_ && C_ && A && dy && checks && strides && du && ddelta && dB && dC && dparams && (!z || dz),
               "asrn_selective_bwd: null pointer");
  s.chunk = chunk_of(B, L, d);
  s.chunks = chunks_of(B, L, d);
  s.own = own_floats(d, N);
  ASRN_REQUIRE(s.chunks < 65536, "asrn_selective_bwd: too many chunks");
  ASRN_REQUIRE(grid_ok(B * L * 2 * N, 256), "asrn_selective_bwd: too many tokens");
  const int64_t need = asrn_selective_bwd_workspace(B, L, d, N), groups = B * s.chunks, cols = (int64_t)d * N + 2 * d;
  ASRN_REQUIRE(workspace && workspace_bytes >= need && !((uintptr_t)workspace & 15),
               "asrn_selective_bwd: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
               (long long)workspace_bytes);
  ASRN_REQUIRE(groups < (1 << 30) && cols < (1 << 30), "asrn_selective_bwd: too many chunks");
  s.carry = (float*)workspace;
  s.total = s.carry + B * (s.chunks - 1) * s.own;
  s.bc = (float*)((char*)workspace + carry_bytes(B, s.chunks, d, N));
  s.part = s.bc + bc_floats(B, L, d, N);
  int waves, blocks;
  grid_of(d, waves, blocks);
  hipStream_t st = (hipStream_t)stream;
  const int rc = with_type(type, [&](auto t) {
    using T = decltype(t);
    return with_states(N, [&](auto npl) {
      constexpr int NPL = decltype(npl)::value;
      if (s.chunks > 1) {
        hipLaunchKernelGGL((k_selective_local_bwd<T, NPL>), dim3(blocks, s.chunks - 1, B), dim3(64 * waves), 0, st, s);
        hipLaunchKernelGGL((k_selective_carry<NPL, true>), dim3((unsigned)((B * s.own + 255) / 256)), dim3(256), 0, st, s);
      }
      hipLaunchKernelGGL((k_selective_bwd<T, NPL>), dim3(blocks, s.chunks, B), dim3(64 * waves), 0, st, s);
      hipLaunchKernelGGL((k_selective_shared<T>), dim3((unsigned)((B * L * 2 * N + 255) / 256)), dim3(256), 0, st, s.bc, blocks,
                         B * L, N, (T*)dB, (T*)dC);
      return check_launch("asrn_selective_bwd");
    });
  });
  return rc ? rc : group_sums(s.part, (int)groups, (int)cols, dparams, st);
}

extern "C" int asrn_selective_step(const void* u, const void* delta, const void* B_, const void* C_, const void* z,
                                   int32_t type, const int64_t* strides, const float* A, const float* D, const float* bias,
                                   const float* h, float* next, int64_t B, int32_t d, int32_t N, int32_t softplus, void* y,
                                   void* stream) {
  Selective s = {};
  s.u = u; s.dl = delta; s.Bm = B_; s.Cm = C_; s.z = z;
  s.A = A; s.D = D; s.bias = bias; s.y = y;
  s.B = B; s.L = 1; s.d = d; s.N = N; s.softplus = softplus;
  if (check(s, type, "asrn_selective_step")) return 1;
  if (B == 0) return 0;
  ASRN_REQUIRE(u && delta && B_ && C_ && A && y && h && next && strides, "asrn_selective_step: null pointer");
  ASRN_REQUIRE(grid_ok(B * d * 4, 256), "asrn_selective_step: too many channels");
  s.ub = strides[0]; s.dlb = strides[1]; s.Bb = strides[2]; s.Cb = strides[3]; s.zb = strides[4];
  return with_type(type, [&](auto t) {
    hipLaunchKernelGGL((k_selective_step<decltype(t)>), dim3((unsigned)((B * d * 4 + 255) / 256)), dim3(256), 0,
                       (hipStream_t)stream, s, h, next);
    return check_launch("asrn_selective_step");
  });
}
