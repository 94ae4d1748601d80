// Log-probabilities of given tokens under a vocabulary's logits, and the rows' entropy, for the preference and policy
// losses: with z_v = (x_v - m) / T, m the row's maximum and s = sum_v exp z_v,
//   log p_y = z_y - log s,   H = log s - (1 / s) sum_v z_v exp z_v,
//   d x_v = (1 / T) [ g (1{v = y} - p_v) - g_H p_v (log p_v + H) ],   p_v = exp(z_v) / s.
// x in fp32, bf16 or fp16 as the model wrote it (no fp32 copy), every sum in fp32, the gradient rounded once to x's type.
//
//   k_logp_fwd  a row is read once: each thread keeps a running maximum, sum and (for the entropy) weighted sum over its
//               vectors of 16 bytes, four of them in flight, and the threads' are joined at the end, so that a row of any
//               length needs no second pass and no registers for its values. (m, s) are kept per row for the backward.
//               Rows whose target is ignored (a prompt's, padding) are not read.
//   k_logp_bwd  a row read once and its gradient written once; rows that are ignored are only written (zeros). With few
//               rows each is split along the vocabulary over the grid.
// Both are bound by HBM: 8192 x 50304 bf16, 61% of the tokens ignored, 55 and 208 us, 5.9 and 5.5 TB/s. Vectors are
// loaded and stored from any element's address (rows of an odd vocabulary, slices): the wide accesses need no more
// alignment than the elements have.
#include <math.h>

#include "common.h"

namespace asrn {

enum { kLpF32 = 0, kLpBf16 = 1, kLpF16 = 2 };

struct LpArgs {
  const void* x; int64_t L, V, sb, st;          // row (b, t) starts at element b sb + t st
  const int64_t* target; int64_t ignore; float inv_t;
  float* logp; float* ent; float2* stats; int64_t rows;
  const float* g; const float* gh; void* dx;    // backward: dx dense (rows, V)
  int splits;
};

typedef _Float16 lp_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 lp_b2 __attribute__((ext_vector_type(2)));
typedef float lp_f2 __attribute__((ext_vector_type(2)));

template <int T> struct LpType;                                  // E: elements of a 16-byte vector
template <> struct LpType<kLpF32> {
  static constexpr int E = 4, S = 4;
  static __device__ __forceinline__ float one(const void* p) { return *reinterpret_cast<const float*>(p); }
  static __device__ __forceinline__ void store(void* p, float v) { *reinterpret_cast<float*>(p) = v; }
  static __device__ __forceinline__ void open(uint32_t w, float* v) { v[0] = __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t close(const float* v) { return __float_as_uint(v[0]); }
};
template <> struct LpType<kLpBf16> {
  static constexpr int E = 8, S = 2;
  static __device__ __forceinline__ float one(const void* p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
  }
  static __device__ __forceinline__ void store(void* p, float v) { *reinterpret_cast<__bf16*>(p) = (__bf16)v; }
  static __device__ __forceinline__ void open(uint32_t w, float* v) {
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t close(const float* v) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((lp_f2){v[0], v[1]}, lp_b2));
  }
};
template <> struct LpType<kLpF16> {
  static constexpr int E = 8, S = 2;
  static __device__ __forceinline__ float one(const void* p) { return (float)*reinterpret_cast<const _Float16*>(p); }
  static __device__ __forceinline__ void store(void* p, float v) { *reinterpret_cast<_Float16*>(p) = (_Float16)v; }
  static __device__ __forceinline__ void open(uint32_t w, float* v) {
    const lp_h2 h = __builtin_bit_cast(lp_h2, w);
    v[0] = (float)h.x;
    v[1] = (float)h.y;
  }
  static __device__ __forceinline__ uint32_t close(const float* v) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((lp_f2){v[0], v[1]}, lp_h2));
  }
};

__device__ __forceinline__ uint4 lp_load(const char* p) {
  uint4 q;
  __builtin_memcpy(&q, p, 16);
  return q;
}
// past the caches' reuse: the gradient is as large as the logits (2177 x 32003 fp32 backward 121 -> 98 us)
typedef uint32_t lp_u4 __attribute__((ext_vector_type(4)));
typedef lp_u4 lp_u4_any __attribute__((aligned(2)));
__device__ __forceinline__ void lp_store(char* p, const uint4& q) {
  __builtin_nontemporal_store((lp_u4){q.x, q.y, q.z, q.w}, reinterpret_cast<lp_u4_any*>(p));
}
template <int T>
__device__ __forceinline__ void lp_open(const uint4& q, float* v) {
  constexpr int W = LpType<T>::E / 4;
  LpType<T>::open(q.x, v);
  LpType<T>::open(q.y, v + W);
  LpType<T>::open(q.z, v + 2 * W);
  LpType<T>::open(q.w, v + 3 * W);
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// the sums of one thread (or of several, joined) over part of a row: s = sum exp2((x - m) c), w = sum of z2 exp2(z2)
// with z2 = (x - m) c; m = -inf stands for no finite value yet, and the base is 0 then. NaN values reach s.
template <bool ENT>
struct LpSum {
  float m, s, w;
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void rebase(float to, float c) {       // to >= m
    if (m != -INFINITY) {
      const float d = (m - to) * c, f = exp2f(d);
      if constexpr (ENT) w = f > 0.f ? f * (w + d * s) : 0.f;
      s = f > 0.f ? s * f : (s != s ? s : 0.f);
    }
    m = to;
  }
  __device__ __forceinline__ void add(float x, float b, float c) {
    const float z = (x - b) * c, e = __builtin_amdgcn_exp2f(z);
    s += e;
    if constexpr (ENT) w += e > 0.f ? e * z : 0.f;
  }
};

// the first element of a row (rows < 2^31)
__device__ __forceinline__ int64_t lp_offset(const LpArgs& a, int64_t row) {
  const uint32_t i = (uint32_t)row, b = i / (uint32_t)a.L;
  return b * a.sb + (i - b * (uint32_t)a.L) * a.st;
}

template <int T, int TPR, bool ENT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_logp_fwd(LpArgs a) {
  constexpr int ROWS = TPR < 256 ? 256 / TPR : 1, E = LpType<T>::E, U = 4;
  const int tid = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  __shared__ float red[3][TPR / kWave];
  if (row >= a.rows) return;                               // whole waves (TPR = 64), or no row of the grid (TPR > 64)
  const int64_t y = a.target[row];
  if (y == a.ignore) {
    if (tid == 0) {
      a.logp[row] = 0.f;
      if (ENT) a.ent[row] = 0.f;
      a.stats[row] = make_float2(0.f, 1.f);
    }
    return;
  }
  const char* r = reinterpret_cast<const char*>(a.x) + lp_offset(a, row) * LpType<T>::S;
  const float c = a.inv_t * kLog2e;
  const int64_t nvec = a.V / E;
  LpSum<ENT> t{-INFINITY, 0.f, 0.f};
  for (int64_t v0 = tid; v0 < nvec; v0 += U * TPR) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t v = v0 + u * TPR;
      q[u] = lp_load(r + 16 * (v < nvec ? v : v0));        // past the row: this thread's first vector again, not used
    }
    float mc = t.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[E];
      lp_open<T>(q[u], x);
#pragma unroll
      for (int k = 0; k < E; ++k) mc = fmaxf(mc, x[k]);
    }
    if (mc > t.m) t.rebase(mc, c);
    const float b = t.base();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v0 + u * TPR >= nvec) break;
      float x[E];
      lp_open<T>(q[u], x);
#pragma unroll
      for (int k = 0; k < E; ++k) t.add(x[k], b, c);
    }
  }
  const int64_t tail = nvec * E + tid;                     // V % E elements, one a thread
  if (tail < a.V) {
    const float x = LpType<T>::one(r + tail * LpType<T>::S);
    if (x > t.m) t.rebase(x, c);
    t.add(x, t.base(), c);
  }
  // join: the wave's sums on its maximum, then the waves' in order
  const float mw = wave_max_u(t.m);
  t.rebase(mw, c);
  t.s = wave_sum_u(t.s);
  if (ENT) t.w = wave_sum_u(t.w);
  if constexpr (TPR > kWave) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & (kWave - 1)) == 0) {
      red[0][wave] = t.m;
      red[1][wave] = t.s;
      red[2][wave] = t.w;
    }
    __syncthreads();
    if (tid != 0) return;
    float mm = -INFINITY, s = 0.f, w = 0.f;
    for (int i = 0; i < TPR / kWave; ++i) mm = fmaxf(mm, red[0][i]);
    for (int i = 0; i < TPR / kWave; ++i) {
      LpSum<ENT> o{red[0][i], red[1][i], red[2][i]};
      o.rebase(mm, c);
      s += o.s;
      w += o.w;
    }
    t.m = mm; t.s = s; t.w = w;
  } else if (tid != 0) {
    return;
  }
  const float b = t.base(), ls = logf(t.s);
  const bool in = y >= 0 && y < a.V;                       // a target outside the vocabulary: NaN
  a.logp[row] = in ? (LpType<T>::one(r + (in ? y : 0) * LpType<T>::S) - b) * a.inv_t - ls : NAN;
  if (ENT) a.ent[row] = ls - kLn2 * (t.w / t.s);
  a.stats[row] = make_float2(b, t.s);
}

template <int T, int TH, bool ENT>
__global__ __launch_bounds__(256) void k_logp_bwd(LpArgs a) {
  constexpr int E = LpType<T>::E, U = 4, S = LpType<T>::S, W = E / 4;
  const int tid = threadIdx.x % TH;
  const int64_t row = (int64_t)blockIdx.x * (256 / TH) + threadIdx.x / TH;
  if (row >= a.rows) return;
  const int64_t nvec = a.V / E, per = (nvec + a.splits - 1) / a.splits;
  const int64_t lo = blockIdx.y * per, hi = lo + per < nvec ? lo + per : nvec;
  char* o = reinterpret_cast<char*>(a.dx) + row * a.V * S;
  const int64_t y = a.target[row], tail = nvec * E + tid;    // V % E elements past the vectors, one a thread
  const bool last = (int)blockIdx.y == a.splits - 1;
  if (y == a.ignore) {
    for (int64_t v = lo + tid; v < hi; v += TH) lp_store(o + 16 * v, make_uint4(0u, 0u, 0u, 0u));
    if (last && tail < a.V) LpType<T>::store(o + tail * S, 0.f);
    return;
  }
  const char* r = reinterpret_cast<const char*>(a.x) + lp_offset(a, row) * S;
  const float2 st = a.stats[row];
  const float c = a.inv_t * kLog2e, b = st.x, inv_s = 1.f / st.y;
  const bool in = y >= 0 && y < a.V;
  const int64_t yvec = in ? y / E : -1;
  const float g = in ? (a.g ? a.g[row] : 0.f) * a.inv_t : NAN;
  float A = inv_s * g, B = 0.f;
  if constexpr (ENT) {                                     // p (log p + H) = (e / s) (z ln 2 - log s + H)
    const float h = a.gh[row] * a.inv_t;
    A += inv_s * h * (a.ent[row] - logf(st.y));
    B = inv_s * h * kLn2;
  }
  const auto grad = [&](float x) {
    const float z = (x - b) * c, e = __builtin_amdgcn_exp2f(z);
    if constexpr (ENT) return e > 0.f ? -e * (A + B * z) : e * -A;
    return e * -A;
  };
  for (int64_t v0 = lo + tid; v0 < hi; v0 += U * TH) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t v = v0 + u * TH;
      q[u] = lp_load(r + 16 * (v < hi ? v : v0));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t v = v0 + u * TH;
      if (v >= hi) break;
      float x[E];
      lp_open<T>(q[u], x);
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = grad(x[k]);
      if (v == yvec) {                                     // the target's own element
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] += k == (int)(y % E) ? g : 0.f;
      }
      lp_store(o + 16 * v, make_uint4(LpType<T>::close(x), LpType<T>::close(x + W), LpType<T>::close(x + 2 * W),
                                      LpType<T>::close(x + 3 * W)));
    }
  }
  if (last && tail < a.V)
    LpType<T>::store(o + tail * S, grad(LpType<T>::one(r + tail * S)) + (tail == y ? g : 0.f));
}

static int lp_check(const LpArgs& a, int32_t type, const char* what) {
  ASRN_REQUIRE(type >= kLpF32 && type <= kLpF16, "%s: type=%d (0 fp32, 1 bf16, 2 fp16)", what, type);
  ASRN_REQUIRE(a.rows >= 0 && a.L >= 1 && a.V >= 1 && a.rows < (int64_t(1) << 31) && a.V < (int64_t(1) << 40) &&
                   a.sb >= 0 && a.st >= 0 && a.rows % a.L == 0,
               "%s: bad sizes rows=%lld L=%lld V=%lld strides %lld, %lld", what, (long long)a.rows, (long long)a.L,
               (long long)a.V, (long long)a.sb, (long long)a.st);
  // a launch has fewer than 2^32 threads: 64 a row for short vocabularies, else 256 (1,024 for up to 1,024 rows)
  ASRN_REQUIRE(a.rows < (int64_t(1) << (a.V <= 2048 ? 26 : 24)), "%s: too many rows (%lld)", what, (long long)a.rows);
  ASRN_REQUIRE(a.inv_t > 0.f && a.inv_t < INFINITY, "%s: the temperature's inverse must be positive and finite", what);
  return 0;
}

// Vectors of a row up to which a wave takes it, four rows a workgroup (16384 x 256 fp32 backward: 18 us with 256 threads a
// row, 7 with a wave; 16384 x 8000 bf16, 1000 vectors, stays with 256). Rows up to which a workgroup has 1,024 threads in
// the forward and a row is split over several in the backward: four workgroups a CU (512 x 50304 bf16: forward 13 us)
constexpr int64_t kLpWave = 512, kLpGroups = 1024;

template <int T, bool ENT>
static void lp_fwd(const LpArgs& a, hipStream_t st) {
  const int64_t nvec = a.V / LpType<T>::E;
#define ASRN_LP(TPR, ROWS)                                                                             \
  hipLaunchKernelGGL((k_logp_fwd<T, TPR, ENT>), dim3((unsigned)((a.rows + ROWS - 1) / ROWS)), dim3(TPR * ROWS), 0, st, a)
  if (nvec <= kLpWave) ASRN_LP(64, 4);
  else if (nvec <= 2048 || a.rows > kLpGroups) ASRN_LP(256, 1);
  else ASRN_LP(1024, 1);
#undef ASRN_LP
}

}  // namespace asrn

using namespace asrn;

#define ASRN_LP_TYPE(CALL)                 \
  if (type == kLpF32) { CALL(kLpF32); }    \
  else if (type == kLpBf16) { CALL(kLpBf16); } \
  else { CALL(kLpF16); }

extern "C" int asrn_token_logp_fwd(const void* logits, int32_t type, int64_t rows, int64_t L, int64_t V,
                                   int64_t stride_b, int64_t stride_t, const int64_t* target, int64_t ignore_index,
                                   float inv_temperature, float* logp, float* entropy, float* stats, void* stream) {
  LpArgs a{};
  a.x = logits; a.L = L; a.V = V; a.sb = stride_b; a.st = stride_t; a.target = target; a.ignore = ignore_index;
  a.inv_t = inv_temperature; a.logp = logp; a.ent = entropy; a.stats = reinterpret_cast<float2*>(stats); a.rows = rows;
  if (lp_check(a, type, "asrn_token_logp_fwd")) return 1;
  if (rows == 0) return 0;
  ASRN_REQUIRE(logits && target && logp && stats, "asrn_token_logp_fwd: null pointer");
  hipStream_t st = (hipStream_t)stream;
#define ASRN_LP_F(T) if (entropy) lp_fwd<T, true>(a, st); else lp_fwd<T, false>(a, st)
  ASRN_LP_TYPE(ASRN_LP_F)
#undef ASRN_LP_F
  return check_launch("asrn_token_logp_fwd");
}

extern "C" int asrn_token_logp_bwd(const void* logits, int32_t type, int64_t rows, int64_t L, int64_t V,
                                   int64_t stride_b, int64_t stride_t, const int64_t* target, int64_t ignore_index,
                                   float inv_temperature, const float* stats, const float* entropy,
                                   const float* g_logp, const float* g_entropy, void* dlogits, void* stream) {
  LpArgs a{};
  a.x = logits; a.L = L; a.V = V; a.sb = stride_b; a.st = stride_t; a.target = target; a.ignore = ignore_index;
  a.inv_t = inv_temperature; a.ent = const_cast<float*>(entropy);
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats)); a.rows = rows;
  a.g = g_logp; a.gh = g_entropy; a.dx = dlogits;
  if (lp_check(a, type, "asrn_token_logp_bwd")) return 1;
  ASRN_REQUIRE(!g_entropy || entropy, "asrn_token_logp_bwd: the entropy's gradient needs the forward's entropy");
  if (rows == 0) return 0;
  ASRN_REQUIRE(logits && target && stats && dlogits && (g_logp || g_entropy), "asrn_token_logp_bwd: null pointer");
  // rows split along the vocabulary until the grid fills the chip, each part at least one round of its threads' loads
  const int64_t round = (type == kLpF32 ? 4 : 8) * 4 * 256;
  int64_t splits = (kLpGroups + rows - 1) / rows, most = (V + round - 1) / round;
  splits = splits < most ? splits : most;
  a.splits = (int)(splits < 1 ? 1 : splits > 65535 ? 65535 : splits);
  const bool corto = V / (type == kLpF32 ? 4 : 8) <= kLpWave;
  const dim3 grid((unsigned)(corto ? (rows + 3) / 4 : rows), (unsigned)a.splits), block(256);
  hipStream_t st = (hipStream_t)stream;
#define ASRN_LP_B2(T, TH)                                                               \
  if (g_entropy) hipLaunchKernelGGL((k_logp_bwd<T, TH, true>), grid, block, 0, st, a);  \
  else hipLaunchKernelGGL((k_logp_bwd<T, TH, false>), grid, block, 0, st, a)
#define ASRN_LP_B(T) if (corto) { ASRN_LP_B2(T, 64); } else { ASRN_LP_B2(T, 256); }
  ASRN_LP_TYPE(ASRN_LP_B)
#undef ASRN_LP_B
#undef ASRN_LP_B2
  return check_launch("asrn_token_logp_bwd");
}
