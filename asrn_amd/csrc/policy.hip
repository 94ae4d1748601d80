// The clipped policy loss with its KL and entropy terms, from the log-probabilities of sampled tokens. Per token, with
// d = lp - old, r = exp d, an advantage A (one a token or, with stride 0, one a text) and q = ref - lp:
//   l = -min(r A, clip(r, 1 - e_lo, 1 + e_hi) A)   [A < 0 and r > c: -c A, the second clip]
//       + beta (exp q - 1 - q) - w H,
//   d l / d lp = -r A where no clip holds, else 0, + beta (1 - exp q);   d l / d H = -w,
// averaged over the masked tokens, or over the texts' own means (texts without tokens left out).
// A token is clipped when d passes the border's logarithm: d in double is exact, so a value next to the border falls
// where the definition puts it. exp q - 1 - q cancels for small q and is taken from its series there. The exponentials
// are fp32's (in double they alone took 55 of 75 us at 3.2 M tokens), products and sums double.
//
//   k_pol_tokens  pieces of 2,048 tokens of a text, one workgroup each: the per-token gradient (not yet divided), and
//                 the piece's count, loss, clipped tokens, KL to old (r - 1 - d) and to the reference, and entropy.
//   k_pol_loss    one workgroup: the pieces' sums in a fixed order, the loss, the statistics, each text's divisor.
//   k_pol_bwd     the gradients over their divisor times the loss's own gradient.
#include <math.h>

#include "common.h"
#include "strided.h"

namespace asrn {

constexpr int kPoThreads = 256;
constexpr int kPoUnroll = 4;
constexpr int kPoPiece = 2048;
constexpr int kPoLossThreads = 512;

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

// exp d within two steps of fp32: expf of d rounded, and the rounding's own factor; past fp32's range in double
__device__ __forceinline__ double po_exp(double d) {
  const float f = (float)d;
  if (f > 80.f) return exp(d);
  const double e = expf(f), rest = d - (double)f;
  return fabs(rest) < 1.0 ? e * (1.0 + rest) : e;        // -infinity and below fp32's range: expf's 0; NaN: NaN
}
// exp d - 1 - d to a few steps of fp32 at every d: its series up to |d| = 1/2, where the difference would cancel (the
// first term left out, d^10 / 10!, is 2^-29 of the sum there), the difference past it
__device__ __forceinline__ double po_kl(double d) {
  const float f = (float)d;
  if (fabsf(f) <= 0.5f) {
    float p = 1.f / 362880.f;
    p = fmaf(p, f, 1.f / 40320.f);
    p = fmaf(p, f, 1.f / 5040.f);
    p = fmaf(p, f, 1.f / 720.f);
    p = fmaf(p, f, 1.f / 120.f);
    p = fmaf(p, f, 1.f / 24.f);
    p = fmaf(p, f, 1.f / 6.f);
    p = fmaf(p, f, 0.5f);
    return d * d * (double)p;
  }
  return (double)expm1f(f) - d;
}

__global__ __launch_bounds__(kPoThreads) void k_pol_tokens(PoArgs a) {
  __shared__ double red[kPoThreads / kWave][kPoSums];
  const int64_t row = blockIdx.x / a.pieces, t0 = (int64_t)(blockIdx.x % a.pieces) * kPoPiece;
  const int64_t t1 = t0 + kPoPiece < a.L ? t0 + kPoPiece : a.L;
  double s[kPoSums] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
  for (int64_t tb = t0 + threadIdx.x; tb < t1; tb += kPoUnroll * kPoThreads) {
    float lp[kPoUnroll], old[kPoUnroll], adv[kPoUnroll], ref[kPoUnroll], ent[kPoUnroll];
    bool m[kPoUnroll];
#pragma unroll
    for (int u = 0; u < kPoUnroll; ++u) {
      const int64_t t = tb + u * kPoThreads, tc = t < t1 ? t : tb;
      m[u] = a.mask.on(row, tc);
      lp[u] = a.lp.at(row, tc);
      adv[u] = a.adv.at(row, tc);
      old[u] = a.old.p ? a.old.at(row, tc) : lp[u];
      ref[u] = a.ref.p ? a.ref.at(row, tc) : 0.f;
      ent[u] = a.ent.p ? a.ent.at(row, tc) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kPoUnroll; ++u) {
      const int64_t t = tb + u * kPoThreads;
      if (t >= t1) break;
      double dl = 0.0;
      if (m[u]) {                             // what a mask hides may be infinite or NaN: nothing of it is used
        const double A = adv[u], d = (double)lp[u] - (double)old[u], r = po_exp(d);
        const bool cap = a.cap > 0.0 && A < 0.0 && d > a.log_cap;
        const bool out = (A > 0.0 && d > a.log_hi) || (A < 0.0 && d < a.log_lo);
        double l = cap ? -a.cap * A : out ? -(A > 0.0 ? a.hi : a.lo) * A : -r * A;
        dl = cap || out ? 0.0 : -r * A;
        s[0] += 1.0;
        s[2] += cap || out;
        s[3] += po_kl(d);
        if (a.ref.p) {
          const double q = (double)ref[u] - (double)lp[u], kl = po_kl(q);
          if (a.beta != 0.0) {
            l += a.beta * kl;
            dl -= a.beta * (double)expm1f((float)q);
          }
          s[4] += kl;
        }
        if (a.ent.p) {
          l -= a.w_ent * (double)ent[u];
          s[5] += (double)ent[u];
        }
        s[1] += l;
      }
      if (a.raw) a.raw[row * a.L + t] = (float)dl;
    }
  }
#pragma unroll
  for (int k = 0; k < kPoSums; ++k) {
    s[k] = wave_sum_d(s[k]);
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave][k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x < kPoSums) {
    double v = 0.0;
    for (int w = 0; w < kPoThreads / kWave; ++w) v += red[w][threadIdx.x];
    reinterpret_cast<double*>(a.part + blockIdx.x)[threadIdx.x] = v;
  }
}

__global__ __launch_bounds__(kPoLossThreads) void k_pol_loss(PoArgs a) {
  __shared__ double red[kPoLossThreads / kWave][kPoSums + 2];
  __shared__ double total, texts;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  double s[kPoSums + 2] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};     // ..., the texts' means, texts with tokens
  const int g = a.lanes, part = threadIdx.x & (g - 1);
  // whole waves stay in the loop: a lane past the texts sums the last one again and keeps nothing
  for (int64_t b0 = threadIdx.x / g; b0 - (threadIdx.x / g) < a.B; b0 += kPoLossThreads / g) {
    const int64_t b = b0 < a.B ? b0 : a.B - 1;
    double r[kPoSums] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
    for (uint32_t p = part; p < a.pieces; p += g) {
      const double* q = reinterpret_cast<const double*>(a.part + b * a.pieces + p);
#pragma unroll
      for (int k = 0; k < kPoSums; ++k) r[k] += q[k];
    }
#pragma unroll
    for (int k = 0; k < kPoSums; ++k) r[k] = group_sum_d(r[k], g);
    if (part != 0 || b0 >= a.B) continue;
    const double n = r[0];
    a.weight[b] = (float)(n > 0.0 ? n : 1.0);
#pragma unroll
    for (int k = 0; k < kPoSums; ++k) s[k] += r[k];
    s[kPoSums] += n > 0.0 ? r[1] / n : 0.0;
    s[kPoSums + 1] += n > 0.0 ? 1.0 : 0.0;
  }
#pragma unroll
  for (int k = 0; k < kPoSums + 2; ++k) {
    s[k] = wave_sum_d(s[k]);
    if (lane == 0) red[wave][k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < kPoSums + 2; ++k) {
      s[k] = 0.0;
      for (int w = 0; w < kPoLossThreads / kWave; ++w) s[k] += red[w][k];
    }
    const double n = s[0], nt = s[kPoSums + 1];
    *a.loss = (float)(a.by_text ? s[kPoSums] / nt : s[1] / n);   // no token at all: 0 / 0
    a.stats[0] = (float)(s[2] / n);
    a.stats[1] = (float)(s[3] / n);
    a.stats[2] = (float)(s[4] / n);
    a.stats[3] = (float)(s[5] / n);
    total = n;
    texts = nt;
  }
  __syncthreads();
  const double n = total, nt = texts;
  for (int64_t b = threadIdx.x; b < a.B; b += kPoLossThreads)
    a.weight[b] = (float)(a.by_text ? (double)a.weight[b] * nt : n);
}

__global__ __launch_bounds__(kPoThreads) void k_pol_bwd(PoArgs a) {
  const int64_t row = blockIdx.x / a.pieces, t0 = (int64_t)(blockIdx.x % a.pieces) * kPoPiece;
  const int64_t t1 = t0 + kPoPiece < a.L ? t0 + kPoPiece : a.L;
  const float c = *a.g / a.weight[row], ce = (float)-a.w_ent * c;
  for (int64_t t = t0 + threadIdx.x; t < t1; t += kPoThreads) {
    const int64_t i = row * a.L + t;
    const bool m = a.mask.on(row, t);
    if (a.dlp) a.dlp[i] = m ? a.raw[i] * c : 0.f;
    if (a.dent) a.dent[i] = m ? ce : 0.f;
  }
}

}  // namespace asrn

using namespace asrn;

static int64_t po_pieces(int64_t L) { return L > 0 ? (L + kPoPiece - 1) / kPoPiece : 1; }
static bool po_sizes(int64_t B, int64_t L) {
  return B >= 1 && B < (int64_t(1) << 31) && L >= 0 && L < (int64_t(1) << 31) && B * po_pieces(L) < (int64_t(1) << 31);
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
  hipLaunchKernelGGL(k_pol_tokens, dim3((unsigned)(a.pieces * B)), dim3(kPoThreads), 0, st, a);
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
  hipLaunchKernelGGL(k_pol_bwd, dim3((unsigned)(a.pieces * B)), dim3(kPoThreads), 0, (hipStream_t)stream, a);
  return check_launch("asrn_policy_bwd");
}
