// The clipped policy loss with its KL and entropy terms, from the log-probabilities of sampled tokens. Per token, with
// d = lp - old, r = exp d, an advantage A (one a token or, with stride 0, one a text) and q = ref - lp:
//   l = -min(r A, clip(r, 1 - e_lo, 1 + e_hi) A)   [A < 0 and r > c: -c A, the second clip]
//       + beta (exp q - 1 - q) - w H,
//   d l / d lp = -r A where no clip holds, else 0, + beta (1 - exp q);   d l / d H = -w,
// averaged over the masked tokens, or over the texts' own means (texts without tokens left out).
// A token is clipped when d passes the border's logarithm: d in double is exact, so a value next to the border falls
// where the definition puts it. exp q - 1 - q cancels for small q and is taken from its series, which gives exp q - 1 and
// exp d as well. The exponentials are fp32's, products and sums double.
//
//   k_pol_tokens  pieces of 2,048 tokens of a text, one workgroup each: the per-token gradient (not yet divided), and
//                 the piece's count, loss, clipped tokens, KL to old (r - 1 - d) and to the reference, and entropy.
//   k_pol_loss    one workgroup: the pieces' sums in a fixed order, the loss, the statistics, each text's divisor.
//   k_pol_few     the two in one launch for a few short texts.
//   k_pol_bwd     the gradients over their divisor times the loss's own gradient.
// 160 texts of 20,001 tokens with every term: 22 + 6.8 + 9.4 us. The first takes 102 registers, so 4 waves a SIMD and 1,024
// workgroups at a time, and its 1,600 two rounds, 3.7 TB/s in all. k_pol_loss is one workgroup at any size: 4.6 us up to
// 2,048 pieces, then 0.7 us a thousand. Short batches are bound by launches (4 texts of 50: 5.8 and 3.3 us).
#include <math.h>

#include "common.h"
#include "strided.h"

namespace asrn {

constexpr int kPoThreads = 256;
constexpr int kPoPiece = 2048;
constexpr int kPoLossThreads = 1024;

struct PoPart { double n, loss, clip, kl_old, kl_ref, ent; };
constexpr int kPoSums = 6;

struct PoArgs {
  Strided lp, adv, old, ref, ent, mask;
  int64_t B, L;
  double lo, hi, log_lo, log_hi, cap, log_cap, beta, w_ent;     // cap 0: no second clip
  int32_t by_text;
  float* raw;                     // (B, L) gradient of each token's loss
  PoPart* part; uint32_t pieces; int lanes;
  float* loss; float* stats; float* weight;                     // weight (B): what a text's tokens are divided by
  const float* g; float* dlp; float* dent;
};

// exp d over double's range to a few steps of fp32: expf of d rounded, and the rounding's own factor; past fp32's range the
// square of the half's (two steps) or, from 160 on, the eighth power of the eighth's (eight steps; the double exp's
// registers would cost half the waves)
__device__ __forceinline__ double po_exp(double d) {
  const float f = (float)d;
  double e = expf(f > 160.f ? 0.125f * f : f > 80.f ? 0.5f * f : f);
  const double rest = d - (double)f;
  if (f > 80.f) e *= e;
  if (f > 160.f) {
    e *= e;
    e *= e;
  }
  return e * (fabs(rest) < 1.0 ? 1.0 + rest : 1.0);             // infinite d: expf's answer; NaN: NaN
}
// exp d - 1 (first) and exp d - 1 - d (second), each to a few steps of fp32 at every d: up to |d| = 1 from the second
// one's series, where the difference would cancel (the first term left out is 2^-32 of the sum), past it from exp d
struct PoExp { double e1, kl; };
__device__ __forceinline__ PoExp po_terms(double d) {
  const float f = (float)d;
  if (fabsf(f) <= 1.f) {
    float p = 1.f / 479001600.f;
    p = fmaf(p, f, 1.f / 39916800.f);
    p = fmaf(p, f, 1.f / 3628800.f);
    p = fmaf(p, f, 1.f / 362880.f);
    p = fmaf(p, f, 1.f / 40320.f);
    p = fmaf(p, f, 1.f / 5040.f);
    p = fmaf(p, f, 1.f / 720.f);
    p = fmaf(p, f, 1.f / 120.f);
    p = fmaf(p, f, 1.f / 24.f);
    p = fmaf(p, f, 1.f / 6.f);
    p = fmaf(p, f, 0.5f);
    const double kl = d * d * (double)p;
    return PoExp{d + kl, kl};
  }
  const double e1 = po_exp(d) - 1.0;
  return PoExp{e1, e1 - d};
}

// n <= 4 tokens of a text from t: their gradients, and what they add to a lane's sums. ROW: every text's tokens lie next to
// each other and are read 4 at a time (3.2 M tokens: 33 -> 23 us)
struct PoLane { double s[kPoSums] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0}; int kept = 0, clipped = 0; };
template <bool ROW>
__device__ __forceinline__ void po_four(const PoArgs& a, int64_t row, int64_t t, int n, PoLane& z) {
  float lp[4], old[4], adv[4], ref[4], ent[4], raw[4];
  const uint32_t m = a.mask.on4<ROW>(row, t, n);
  a.lp.four<ROW>(row, t, n, 0.f, lp);
  if (a.adv.st == 0) adv[0] = adv[1] = adv[2] = adv[3] = a.adv.at(row, 0);
  else a.adv.four<ROW>(row, t, n, 0.f, adv);
  if (a.old.p) a.old.four<ROW>(row, t, n, 0.f, old);
  if (a.ref.p) a.ref.four<ROW>(row, t, n, 0.f, ref);
  if (a.ent.p) a.ent.four<ROW>(row, t, n, 0.f, ent);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    double dl = 0.0;
    if (u < n && (m >> (8 * u) & 0xffu)) {    // what a mask hides may be infinite or NaN: nothing of it is used
      const double A = adv[u], d = a.old.p ? (double)lp[u] - (double)old[u] : (double)(lp[u] - lp[u]);
      const PoExp x = po_terms(d);
      // an advantage of 0 takes nothing from any finite d, also where exp d passes double's range
      const double rA = fma(A == 0.0 && fabs(d) < INFINITY ? 0.0 : x.e1, A, A);
      const bool cap = a.cap > 0.0 && A < 0.0 && d > a.log_cap;
      const bool out = cap || (A > 0.0 && d > a.log_hi) || (A < 0.0 && d < a.log_lo);
      double l = -(out ? (cap ? a.cap : A > 0.0 ? a.hi : a.lo) * A : rA);
      dl = out ? 0.0 : -rA;
      ++z.kept;
      z.clipped += out;
      z.s[3] += x.kl;
      if (a.ref.p) {
        const PoExp q = po_terms((double)ref[u] - (double)lp[u]);
        if (a.beta != 0.0) {
          l = fma(a.beta, q.kl, l);
          dl = fma(-a.beta, q.e1, dl);
        }
        z.s[4] += q.kl;
      }
      if (a.ent.p) {
        l = fma(-a.w_ent, (double)ent[u], l);
        z.s[5] += (double)ent[u];
      }
      z.s[1] += l;
    }
    raw[u] = (float)dl;
  }
  if (a.raw) {
    if (n == 4) {
      __builtin_memcpy(a.raw + row * a.L + t, raw, 16);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < n) a.raw[row * a.L + t + u] = raw[u];
    }
  }
}

template <bool ROW>
__global__ __launch_bounds__(kPoThreads) void k_pol_tokens(PoArgs a) {
  __shared__ double red[kPoThreads / kWave][kPoSums];
  const int64_t row = blockIdx.x / a.pieces, t0 = (int64_t)(blockIdx.x % a.pieces) * kPoPiece;
  const int64_t t1 = t0 + kPoPiece < a.L ? t0 + kPoPiece : a.L;
  PoLane z;
  for (int64_t t = t0 + 4 * threadIdx.x; t < t1; t += 4 * kPoThreads) po_four<ROW>(a, row, t, t1 - t < 4 ? (int)(t1 - t) : 4, z);
  z.s[0] = z.kept;
  z.s[2] = z.clipped;
#pragma unroll
  for (int k = 0; k < kPoSums; ++k) {
    const double v = wave_sum_d(z.s[k]);
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave][k] = v;
  }
  __syncthreads();
  if (threadIdx.x < kPoSums) {
    double v = 0.0;
    for (int w = 0; w < kPoThreads / kWave; ++w) v += red[w][threadIdx.x];
    reinterpret_cast<double*>(a.part + blockIdx.x)[threadIdx.x] = v;
  }
}

// The end of the loss over a workgroup of TH threads: s is a lane's share of the sums, then of the texts' means and of
// the texts with tokens; weight[b] holds a text's own count (at least 1) and becomes its divisor.
template <int TH>
__device__ __forceinline__ void po_finish(const PoArgs& a, double* s) {
  __shared__ double red[TH / kWave][kPoSums + 2];
  __shared__ double sums[kPoSums + 2];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int k = 0; k < kPoSums + 2; ++k) {
    s[k] = wave_sum_d(s[k]);
    if (lane == 0) red[wave][k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x < kPoSums + 2) {            // a sum a thread, the waves in order
    double v = 0.0;
    for (int w = 0; w < TH / kWave; ++w) v += red[w][threadIdx.x];
    sums[threadIdx.x] = v;
  }
  __syncthreads();
  const double n = sums[0], nt = sums[kPoSums + 1];
  if (threadIdx.x == 0) *a.loss = (float)(a.by_text ? sums[kPoSums] / nt : sums[1] / n);   // no token at all: 0 / 0
  if (threadIdx.x < 4) a.stats[threadIdx.x] = (float)(sums[2 + threadIdx.x] / n);
  for (int64_t b = threadIdx.x; b < a.B; b += TH)
    a.weight[b] = (float)(a.by_text ? (double)a.weight[b] * nt : n);
}

// Few short texts in one launch: a wave a text, and the workgroup the loss (us in two launches / in one: 4 x 50 8.7 / 6.2,
// 8 x 512 8.3 / 7.9, 16 x 256, two texts a wave, 8.3 / 8.7)
constexpr int kPoFew = 8, kPoShort = 512, kPoFewThreads = kPoFew * kWave;
template <bool ROW>
__global__ __launch_bounds__(kPoFewThreads) void k_pol_few(PoArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  double s[kPoSums + 2] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
  const int64_t b = threadIdx.x / kWave;
  if (b < a.B) {
    PoLane z;
    for (int64_t t = 4 * lane; t < a.L; t += 4 * kWave) po_four<ROW>(a, b, t, a.L - t < 4 ? (int)(a.L - t) : 4, z);
    z.s[0] = z.kept;
    z.s[2] = z.clipped;
#pragma unroll
    for (int k = 0; k < kPoSums; ++k) s[k] = z.s[k];
    const double n = wave_sum_d(z.s[0]), loss = wave_sum_d(z.s[1]);
    if (lane == 0) {
      a.weight[b] = (float)(n > 0.0 ? n : 1.0);
      s[kPoSums] += n > 0.0 ? loss / n : 0.0;
      s[kPoSums + 1] += n > 0.0 ? 1.0 : 0.0;
    }
  }
  po_finish<kPoFewThreads>(a, s);
}

__global__ __launch_bounds__(kPoLossThreads) void k_pol_loss(PoArgs a) {
  double s[kPoSums + 2] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};     // ..., the texts' means, texts with tokens
  const int g = a.lanes, part = threadIdx.x & (g - 1);
  // whole waves stay in the loop: a lane past the texts sums the last one again and keeps nothing
#pragma unroll 1
  for (int64_t b0 = threadIdx.x / g; b0 - (threadIdx.x / g) < a.B; b0 += kPoLossThreads / g) {
    const int64_t b = b0 < a.B ? b0 : a.B - 1;
    double n = 0.0, loss = 0.0;               // the text's own, over its lanes; the totals stay a lane's until the end
#pragma unroll 1
    for (uint32_t p = part; p < a.pieces; p += g) {
      const double* q = reinterpret_cast<const double*>(a.part + b * a.pieces + p);
      double r[kPoSums];
#pragma unroll
      for (int k = 0; k < kPoSums; ++k) r[k] = q[k];
      n += r[0];
      loss += r[1];
#pragma unroll
      for (int k = 0; k < kPoSums; ++k) s[k] += b0 < a.B ? r[k] : 0.0;
    }
    n = group_sum_d(n, g);
    loss = group_sum_d(loss, g);
    if (part != 0 || b0 >= a.B) continue;
    a.weight[b] = (float)(n > 0.0 ? n : 1.0);
    s[kPoSums] += n > 0.0 ? loss / n : 0.0;
    s[kPoSums + 1] += n > 0.0 ? 1.0 : 0.0;
  }
  po_finish<kPoLossThreads>(a, s);
}

template <bool ROW>
__global__ __launch_bounds__(kPoThreads) void k_pol_bwd(PoArgs a) {
  const int64_t row = blockIdx.x / a.pieces, t0 = (int64_t)(blockIdx.x % a.pieces) * kPoPiece;
  const int64_t t1 = t0 + kPoPiece < a.L ? t0 + kPoPiece : a.L;
  const float c = *a.g / a.weight[row], ce = (float)-a.w_ent * c;
  for (int64_t t = t0 + 4 * threadIdx.x; t < t1; t += 4 * kPoThreads) {
    const int64_t i = row * a.L + t;
    const int n = t1 - t < 4 ? (int)(t1 - t) : 4;
    const uint32_t m = a.mask.on4<ROW>(row, t, n);
    float raw[4] = {0.f, 0.f, 0.f, 0.f}, ent[4];
    if (a.dlp) Strided{a.raw, 0, 1}.four<true>(0, i, n, 0.f, raw);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool on = m >> (8 * u) & 0xffu;
      raw[u] = on ? raw[u] * c : 0.f;
      ent[u] = on ? ce : 0.f;
    }
    if (n == 4) {
      if (a.dlp) __builtin_memcpy(a.dlp + i, raw, 16);
      if (a.dent) __builtin_memcpy(a.dent + i, ent, 16);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u < n && a.dlp) a.dlp[i + u] = raw[u];
        if (u < n && a.dent) a.dent[i + u] = ent[u];
      }
    }
  }
}

}  // namespace asrn

using namespace asrn;

static int64_t po_pieces(int64_t L) { return L > 0 ? (L + kPoPiece - 1) / kPoPiece : 1; }
static bool po_sizes(int64_t B, int64_t L) {
  return B >= 1 && B < (int64_t(1) << 31) && L >= 0 && L < (int64_t(1) << 31) && B * po_pieces(L) < (int64_t(1) << 24);   // a launch has fewer than 2^32 threads
}
static int po_check(int64_t B, int64_t L, const char* what) {
  ASRN_REQUIRE(po_sizes(B, L), "%s: bad sizes B=%lld L=%lld", what, (long long)B, (long long)L);
  return 0;
}
static Strided po_view(const void* p, const int64_t* s) { return p ? Strided{p, s[0], s[1]} : Strided{nullptr, 0, 0}; }

extern "C" int64_t asrn_policy_workspace(int64_t B, int64_t L) {
  if (!po_sizes(B, L)) return -1;
  return B * po_pieces(L) * (int64_t)sizeof(PoPart);
}

extern "C" int asrn_policy_fwd(const float* lp, const float* advantage, const float* old_lp, const float* ref_lp,
                               const float* entropy, const uint8_t* mask, const int64_t* strides, int64_t B, int64_t L,
                               double clip_low, double clip_high, double cap, double beta, double entropy_weight,
                               int32_t by_text, float* raw, float* loss, float* stats, float* weight, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (po_check(B, L, "asrn_policy_fwd")) return 1;
  ASRN_REQUIRE(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0 && clip_high < INFINITY,
               "asrn_policy_fwd: clip_low=%g (0 to 1) clip_high=%g (from 0 on)", clip_low, clip_high);
  ASRN_REQUIRE(cap == 0.0 || (cap > 1.0 && cap < INFINITY), "asrn_policy_fwd: cap=%g (0, or above 1)", cap);
  ASRN_REQUIRE(beta >= 0.0 && beta < INFINITY && entropy_weight == entropy_weight && fabs(entropy_weight) < INFINITY,
               "asrn_policy_fwd: beta=%g (from 0 on) entropy_weight=%g", beta, entropy_weight);
  ASRN_REQUIRE(((lp && advantage) || L == 0) && strides && loss && stats && weight, "asrn_policy_fwd: null pointer");
  const int64_t need = asrn_policy_workspace(B, L);
  ASRN_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
               "asrn_policy_fwd: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  PoArgs a{};
  a.lp = po_view(lp, strides); a.adv = po_view(advantage, strides + 2); a.old = po_view(old_lp, strides + 4);
  a.ref = po_view(ref_lp, strides + 6); a.ent = po_view(entropy, strides + 8); a.mask = po_view(mask, strides + 10);
  a.B = B; a.L = L;
  a.lo = 1.0 - clip_low; a.hi = 1.0 + clip_high;
  a.log_lo = log1p(-clip_low); a.log_hi = log1p(clip_high);
  a.cap = cap; a.log_cap = cap > 0.0 ? log(cap) : 0.0;
  a.beta = beta; a.w_ent = entropy_weight; a.by_text = by_text;
  a.raw = raw; a.part = (PoPart*)workspace; a.pieces = (uint32_t)po_pieces(L); a.lanes = lanes_for(a.pieces);
  a.loss = loss; a.stats = stats; a.weight = weight;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(a.pieces * B)), block(kPoThreads);
  const bool rows = a.lp.row() && (a.adv.row() || a.adv.st == 0) && a.old.row() && a.ref.row() && a.ent.row() && a.mask.row();
  if (B <= kPoFew && L <= kPoShort) {
    if (rows) hipLaunchKernelGGL(k_pol_few<true>, dim3(1), dim3(kPoFewThreads), 0, st, a);
    else hipLaunchKernelGGL(k_pol_few<false>, dim3(1), dim3(kPoFewThreads), 0, st, a);
    return check_launch("asrn_policy_fwd");
  }
  if (rows)
    hipLaunchKernelGGL(k_pol_tokens<true>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(k_pol_tokens<false>, grid, block, 0, st, a);
  if (check_launch("asrn_policy_fwd")) return 1;
  hipLaunchKernelGGL(k_pol_loss, dim3(1), dim3(kPoLossThreads), 0, st, a);
  return check_launch("asrn_policy_fwd");
}

extern "C" int asrn_policy_bwd(const float* raw, const float* weight, const float* g, const uint8_t* mask,
                               const int64_t* mask_strides, int64_t B, int64_t L, double entropy_weight, float* dlp,
                               float* dentropy, void* stream) {
  if (po_check(B, L, "asrn_policy_bwd")) return 1;
  if (L == 0 || (!dlp && !dentropy)) return 0;
  ASRN_REQUIRE((raw || !dlp) && weight && g && (!mask || mask_strides), "asrn_policy_bwd: null pointer");
  PoArgs a{};
  a.mask = po_view(mask, mask_strides);
  a.B = B; a.L = L; a.w_ent = entropy_weight; a.raw = const_cast<float*>(raw); a.weight = const_cast<float*>(weight);
  a.g = g; a.dlp = dlp; a.dent = dentropy;
  a.pieces = (uint32_t)po_pieces(L);
  const dim3 grid((unsigned)(a.pieces * B)), block(kPoThreads);
  if (a.mask.row()) hipLaunchKernelGGL(k_pol_bwd<true>, grid, block, 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(k_pol_bwd<false>, grid, block, 0, (hipStream_t)stream, a);
  return check_launch("asrn_policy_bwd");
}
