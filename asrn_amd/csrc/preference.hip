// The preference loss over pairs of texts, from the log-probabilities of their tokens. Rows 0 .. P - 1 of lp (2P, L) are
// the chosen texts, P .. 2P - 1 the rejected ones, m the tokens of the answers:
//   R_i = sum_t m_it (lp_it - ref_it)  [/ sum_t m_it],   h_i = beta (R_i - R_{P+i}) - margin,
//   sigmoid  -(1 - e) log sigma(h) - e log sigma(-h),   ipo  (h / beta - 1 / (2 beta))^2,   hinge  max(0, 1 - h),
// averaged over the pairs. d loss / d lp_it = m_it c_i with one coefficient a row, formed in the forward.
//
//   k_pref_rows  a row in pieces of 2,048 tokens, one workgroup each: the masked sum and the count of a piece. Long rows
//                and few rows alike spread over the chip; the sums are in double (a long text's log-probability is a
//                small difference of large sums), each piece's in a fixed order.
//   k_pref_loss  one workgroup, a pair a group of lanes, one lane a piece: the pieces added in a fixed order, the loss, the
//                rewards and the coefficients.
//   k_pref_few   the two in one launch for a few short texts.
//   k_pref_bwd   d lp = m g c, written once.
// Bound by launches for short batches (one pair of 60: 3.0 and 2.1 us); 24 pairs of 50,001 tokens take 5.4 + 6.3 + 5.2 us
// (the first reads 21.6 MB; 8.4 us with 4-byte loads). k_pref_loss is one workgroup at any size, each step's loads waiting
// for the ones before: 3 to 5 us up to 2,048 pieces, then 1.4 us a thousand, which past 16,000 texts of one piece is as long
// as k_pref_rows.
#include <math.h>

#include "common.h"
#include "strided.h"

namespace asrn {

constexpr int kPfThreads = 256;
constexpr int kPfUnroll = 2;
constexpr int kPfPiece = 4 * kPfUnroll * kPfThreads;       // tokens a workgroup sums, all loads in flight at once
constexpr int kPfLossThreads = 1024;

struct PfPart { double sum; double n; };

struct PfArgs {
  Strided lp, ref, mask;                    // ref.p null: none; ref_rows: one sum a row (ref.st unused), 2: in double
  int64_t P, L;
  int32_t ref_rows, kind, mean;
  double beta, smooth, margin;
  PfPart* part; uint32_t pieces; int lanes;
  float* loss; float* reward; float* coef;
  const float* g; float* dlp;
};

// adds n <= 4 tokens of a text from t. ROW: a text's tokens lie next to each other and are read 4 at a time
template <bool ROW>
__device__ __forceinline__ void pf_four(const PfArgs& a, int64_t row, int64_t t, int n, double& s, int& count) {
  const bool ref = a.ref.p && !a.ref_rows;
  float x[4], r[4];
  const uint32_t m = a.mask.on4<ROW>(row, t, n);
  a.lp.four<ROW>(row, t, n, 0.f, x);
  if (ref) a.ref.four<ROW>(row, t, n, 0.f, r);
#pragma unroll
  for (int k = 0; k < 4; ++k) {               // selected, not multiplied: what a mask hides may be infinite or NaN
    const bool on = m >> (8 * k) & 0xffu;
    s += on ? (double)x[k] - (ref ? (double)r[k] : 0.0) : 0.0;
    count += on;
  }
}

template <bool ROW>
__global__ __launch_bounds__(kPfThreads) void k_pref_rows(PfArgs a) {
  __shared__ PfPart red[kPfThreads / kWave];
  const int64_t row = blockIdx.x / a.pieces, t0 = (int64_t)(blockIdx.x % a.pieces) * kPfPiece;
  const int64_t t1 = t0 + kPfPiece < a.L ? t0 + kPfPiece : a.L;
  double s = 0.0;
  int n = 0;
#pragma unroll
  for (int u = 0; u < kPfUnroll; ++u) {
    const int64_t t = t0 + 4 * (threadIdx.x + u * kPfThreads);
    pf_four<ROW>(a, row, t, t1 - t >= 4 ? 4 : t1 > t ? (int)(t1 - t) : 0, s, n);
  }
  s = wave_sum_d(s);
  double c = wave_sum_d((double)n);
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = PfPart{s, c};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPfThreads / kWave; ++w) {
      s += red[w].sum;
      c += red[w].n;
    }
    a.part[blockIdx.x] = PfPart{s, c};
  }
}

// log(1 + exp(-|h|)) + max(-h, 0) = -log sigma(h)
__device__ __forceinline__ double neg_log_sigma(double h) { return log1p(exp(-fabs(h))) + (h < 0.0 ? -h : h != h ? h : 0.0); }

// pair i from its rows' sums (chosen, rejected): the rewards and coefficients; returns its loss
__device__ __forceinline__ double pf_pair(const PfArgs& a, int64_t i, const PfPart* q) {
  double R[2], div[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    double s = q[k].sum;
    const int64_t row = i + k * a.P;
    if (a.ref.p && a.ref_rows)
      s -= a.ref_rows == 2 ? reinterpret_cast<const double*>(a.ref.p)[row * a.ref.sb] : (double)a.ref.at(row, 0);
    div[k] = a.mean && q[k].n > 1.0 ? q[k].n : 1.0;           // an empty answer: a sum of nothing, divided by 1
    R[k] = s / div[k];
    a.reward[row] = (float)(a.beta * R[k]);
  }
  const double h = a.beta * (R[0] - R[1]) - a.margin;
  double v, dh;
  if (a.kind == 0) {
    v = (1.0 - a.smooth) * neg_log_sigma(h) + (a.smooth != 0.0 ? a.smooth * neg_log_sigma(-h) : 0.0);
    dh = a.smooth - 1.0 / (1.0 + exp(h));
  } else if (a.kind == 1) {
    const double w = (h - 0.5) / a.beta;
    v = w * w;
    dh = 2.0 * w / a.beta;
  } else {
    v = h < 1.0 ? 1.0 - h : h != h ? h : 0.0;
    dh = h < 1.0 ? -1.0 : h != h ? h : 0.0;
  }
  const double c = dh * a.beta / (double)a.P;
  a.coef[i] = (float)(c / div[0]);
  a.coef[i + a.P] = (float)(-c / div[1]);
  return v;
}
__device__ __forceinline__ void pf_finish(const PfArgs& a, double total) {
  __shared__ double red[kPfLossThreads / kWave];
  total = wave_sum_d(total);
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPfLossThreads / kWave; ++w) total += red[w];
    *a.loss = (float)(total / (double)a.P);
  }
}

__global__ __launch_bounds__(kPfLossThreads) void k_pref_loss(PfArgs a) {
  double total = 0.0;
  const int g = a.lanes, lane = threadIdx.x & (g - 1);
  // whole waves stay in the loop: a lane past the pairs sums the last pair again and writes nothing
  for (int64_t i0 = threadIdx.x / g; i0 - (threadIdx.x / g) < a.P; i0 += kPfLossThreads / g) {
    const int64_t i = i0 < a.P ? i0 : a.P - 1;
    PfPart q[2];
    for (int k = 0; k < 2; ++k) {
      double s = 0.0, n = 0.0;
      for (uint32_t p = lane; p < a.pieces; p += g) {
        const PfPart x = a.part[(i + k * a.P) * a.pieces + p];
        s += x.sum;
        n += x.n;
      }
      q[k] = PfPart{group_sum_d(s, g), group_sum_d(n, g)};
    }
    if (lane == 0 && i0 < a.P) total += pf_pair(a, i, q);
  }
  pf_finish(a, total);
}

// Few short texts in one launch: a wave a text, then a thread a pair (us in two launches / in one: 1 pair x 60 5.5 / 3.4, 8 x
// 512 5.5 / 4.7, 32 x 128, four texts a wave, 6.0 / 8.0)
constexpr int kPfFew = kPfLossThreads / kWave, kPfShort = 512;    // texts, tokens
template <bool ROW>
__global__ __launch_bounds__(kPfLossThreads) void k_pref_few(PfArgs a) {
  __shared__ PfPart part[kPfFew];
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = threadIdx.x / kWave;
  if (row < 2 * a.P) {
    double s = 0.0;
    int n = 0;
    for (int64_t t = 4 * lane; t < a.L; t += 4 * kWave) pf_four<ROW>(a, row, t, a.L - t < 4 ? (int)(a.L - t) : 4, s, n);
    s = wave_sum_d(s);
    const double c = wave_sum_d((double)n);
    if (lane == 0) part[row] = PfPart{s, c};
  }
  __syncthreads();
  double total = 0.0;
  if (threadIdx.x < a.P) {
    const PfPart q[2] = {part[threadIdx.x], part[threadIdx.x + a.P]};
    total = pf_pair(a, threadIdx.x, q);
  }
  pf_finish(a, total);
}

template <bool ROW>
__global__ __launch_bounds__(kPfThreads) void k_pref_bwd(PfArgs a) {
  const int64_t row = blockIdx.x / a.pieces, t0 = (int64_t)(blockIdx.x % a.pieces) * kPfPiece;
  const float c = a.coef[row] * *a.g;
  const int64_t t1 = t0 + kPfPiece < a.L ? t0 + kPfPiece : a.L;
  for (int64_t t = t0 + 4 * threadIdx.x; t < t1; t += 4 * kPfThreads) {
    const int n = t1 - t < 4 ? (int)(t1 - t) : 4;
    const uint32_t m = a.mask.on4<ROW>(row, t, n);
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = m >> (8 * k) & 0xffu ? c : 0.f;
    if (n == 4) {
      __builtin_memcpy(a.dlp + row * a.L + t, v, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n) a.dlp[row * a.L + t + k] = v[k];
    }
  }
}

}  // namespace asrn

using namespace asrn;

static int64_t pf_pieces(int64_t L) { return L > 0 ? (L + kPfPiece - 1) / kPfPiece : 1; }
static bool pf_sizes(int64_t P, int64_t L) {
  return P >= 1 && P < (int64_t(1) << 30) && L >= 0 && L < (int64_t(1) << 31) && 2 * P * pf_pieces(L) < (int64_t(1) << 24);   // a launch has fewer than 2^32 threads
}
static int pf_check(int64_t P, int64_t L, const char* what) {
  ASRN_REQUIRE(pf_sizes(P, L), "%s: bad sizes P=%lld L=%lld", what, (long long)P, (long long)L);
  return 0;
}

extern "C" int64_t asrn_preference_workspace(int64_t P, int64_t L) {
  if (!pf_sizes(P, L)) return -1;
  return 2 * P * pf_pieces(L) * (int64_t)sizeof(PfPart);
}

extern "C" int asrn_preference_fwd(const float* lp, const int64_t* lp_strides, const void* ref,
                                   const int64_t* ref_strides, int32_t ref_rows, const uint8_t* mask,
                                   const int64_t* mask_strides, int64_t P, int64_t L, int32_t kind, double beta,
                                   double smoothing, double margin, int32_t mean, float* loss, float* rewards,
                                   float* coef, void* workspace, int64_t workspace_bytes, void* stream) {
  if (pf_check(P, L, "asrn_preference_fwd")) return 1;
  ASRN_REQUIRE(kind >= 0 && kind <= 2, "asrn_preference_fwd: kind=%d (0 sigmoid, 1 ipo, 2 hinge)", kind);
  ASRN_REQUIRE(ref_rows >= 0 && ref_rows <= 2, "asrn_preference_fwd: ref_rows=%d (0 to 2)", ref_rows);
  ASRN_REQUIRE(beta > 0.0 && beta < INFINITY && smoothing >= 0.0 && smoothing <= 1.0 && margin == margin,
               "asrn_preference_fwd: beta=%g (positive) smoothing=%g (0 to 1) margin=%g", beta, smoothing, margin);
  ASRN_REQUIRE((lp || L == 0) && lp_strides && loss && rewards && coef && (!ref || ref_strides) && (!mask || mask_strides),
               "asrn_preference_fwd: null pointer");
  const int64_t need = asrn_preference_workspace(P, L);
  ASRN_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
               "asrn_preference_fwd: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  PfArgs a{};
  a.lp = Strided{lp, lp_strides[0], lp_strides[1]};
  if (ref) a.ref = Strided{ref, ref_strides[0], ref_rows ? 0 : ref_strides[1]};
  if (mask) a.mask = Strided{mask, mask_strides[0], mask_strides[1]};
  a.P = P; a.L = L; a.ref_rows = ref_rows; a.kind = kind; a.mean = mean;
  a.beta = beta; a.smooth = smoothing; a.margin = margin;
  a.part = (PfPart*)workspace; a.pieces = (uint32_t)pf_pieces(L); a.lanes = lanes_for(a.pieces);
  a.loss = loss; a.reward = rewards; a.coef = coef;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(a.pieces * 2 * P)), block(kPfThreads);
  const bool rows = a.lp.row() && a.mask.row() && (a.ref_rows || a.ref.row());
  if (2 * P <= kPfFew && L <= kPfShort) {
    if (rows) hipLaunchKernelGGL(k_pref_few<true>, dim3(1), dim3(kPfLossThreads), 0, st, a);
    else hipLaunchKernelGGL(k_pref_few<false>, dim3(1), dim3(kPfLossThreads), 0, st, a);
    return check_launch("asrn_preference_fwd");
  }
  if (rows) hipLaunchKernelGGL(k_pref_rows<true>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(k_pref_rows<false>, grid, block, 0, st, a);
  if (check_launch("asrn_preference_fwd")) return 1;
  hipLaunchKernelGGL(k_pref_loss, dim3(1), dim3(kPfLossThreads), 0, st, a);
  return check_launch("asrn_preference_fwd");
}

extern "C" int asrn_preference_bwd(const float* coef, const float* g, const uint8_t* mask, const int64_t* mask_strides,
                                   int64_t P, int64_t L, float* dlp, void* stream) {
  if (pf_check(P, L, "asrn_preference_bwd")) return 1;
  if (L == 0) return 0;
  ASRN_REQUIRE(coef && g && dlp && (!mask || mask_strides), "asrn_preference_bwd: null pointer");
  PfArgs a{};
  if (mask) a.mask = Strided{mask, mask_strides[0], mask_strides[1]};
  a.P = P; a.L = L; a.coef = const_cast<float*>(coef); a.g = g; a.dlp = dlp;
  a.pieces = (uint32_t)pf_pieces(L);
  const dim3 grid((unsigned)(a.pieces * 2 * P)), block(kPfThreads);
  if (a.mask.row()) hipLaunchKernelGGL(k_pref_bwd<true>, grid, block, 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(k_pref_bwd<false>, grid, block, 0, (hipStream_t)stream, a);
  return check_launch("asrn_preference_bwd");
}
