// The weight gradient of a 16-bit product: dW (N, K) = g^T x, g (M, N) and x (M, K) with their rows along the sum.
//
// A workgroup forms a BM x BN tile over a slab of rows in steps of 64. Both operands go from memory straight to LDS as they lie,
// rows of BM and BN values, in units of 8 whose column is exchanged by the row's number (4 units a row number: a half
// wave's reads meet every bank once), and are transposed on their way into registers (ds_read_b64_tr_b16: of 16 lanes that name 4 rows by
// 16 values, lane i gets the 4 rows' i-th). A step's loads are issued before the products of the one before, one barrier a step. The matrix
// instruction's rows are x's columns, in an order that leaves a lane with 16 neighbouring values of one row of dW.
// The rows are cut into slabs where the tiles are too few for the card; the slabs' sums are added in order, in fp32, and
// rounded once. 1536 x 768 over 16384 rows: 56 us (0.7 PFLOP/s: the matrix instructions and, in 128 x 128 tiles, L2) and 7 for the
// sums. Steps of 32 rows in four buffers, three of them on their way, took 8% longer: the loads are not what a step waits for.
#include "linear_act.h"

namespace asrn {

constexpr int kStepRows = 64;

struct WeightGrad {
  const void* g; int64_t ldg; const void* x; int64_t ldx;
  int64_t M, slab;                // rows of a slab, a multiple of kStepRows
  int N, K, tn, tk, slabs;
  float* part;                    // (slabs, N, K), or null: one slab, stored to out
  void* out;
  int out32;
};

// One operand's LDS tile of 64 rows by R values
template <typename T, int R, int THR>
struct Slice {
  static constexpr int U = kStepRows * R / 8 / THR;
  static_assert(kStepRows * R / 8 % THR == 0 && R % 128 == 0, "whole units, keys inside a row");
  const T* base;
  int64_t step;
  unsigned at[U];
  // columns past the matrix repeat its last unit: their results are not stored
  __device__ __forceinline__ void start(const void* X, int64_t ld, int64_t m, int c0, int cols, int tid) {
    base = static_cast<const T*>(X) + m * ld;
    step = kStepRows * ld;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int q = tid + THR * i, r = q / (R / 8), c = c0 + 8 * (q % (R / 8) ^ (r & 3) * 4);
      at[i] = (unsigned)(r * (int)ld + (c < cols ? c : cols - 8)) * (unsigned)sizeof(T);
    }
  }
  // the next 64 rows; left: the rows that there are, past them 0
  __device__ __forceinline__ void load(uint4* l, int tid, int wave, int64_t left) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, kPast, 0x00027000);
    if (left >= kStepRows) {
#pragma unroll
      for (int i = 0; i < U; ++i) to_lds(rsrc, l + wave * 64 + THR * i, at[i], 0);
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i)
        l[tid + THR * i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
            rsrc, (tid + THR * i) / (R / 8) < left ? at[i] : kPast, 0, 0));
    }
    base += step;
  }
};

typedef short short4v __attribute__((ext_vector_type(4)));
// lane i of 16 gets the i-th of the 16 values of each of 4 rows; p: lane i's quarter i % 4 of row i / 4
__device__ __forceinline__ short4v read_transposed(const char* p) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
#else
  return short4v{};
#endif
}

template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_weight_grad(WeightGrad a) {
  constexpr int THR = 64 * WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
  constexpr int GU = kStepRows * BM / 8, XU = kStepRows * BN / 8;
  typedef T TX8 __attribute__((ext_vector_type(8)));
  __shared__ uint4 lds0[GU + XU];
  __shared__ uint4 lds1[GU + XU];
  // XCD i takes a contiguous range, tiles of a slab next to each other: they share its rows in the XCD's L2
  const int tiles = a.tn * a.tk, total = tiles * a.slabs, per = (total + kXcdCount - 1) / kXcdCount;
  const int t = (int)(blockIdx.x % kXcdCount) * per + (int)(blockIdx.x / kXcdCount);
  if (t >= total || (int)(blockIdx.x / kXcdCount) >= per) return;
  const int z = t / tiles, n0 = t % tiles / a.tk * BM, k0 = t % tiles % a.tk * BN;
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, lc = lane >> 5;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int64_t m0 = z * a.slab, m1 = m0 + a.slab < a.M ? m0 + a.slab : a.M;
  Slice<T, BM, THR> sg;
  Slice<T, BN, THR> sx;
  sg.start(a.g, a.ldg, m0, n0, a.N, tid);
  sx.start(a.x, a.ldx, m0, k0, a.K, tid);
  // byte offsets of a lane's quarters: row 8 lc + (lane / 4) % 4 of 16; 32 columns are 8 quarters, g's in order, x's exchanged
  const int key = lane >> 2 & 3, quarter = lane >> 2 & 4 | (lane & 3), xq = (quarter & 1) * 4 + (quarter >> 1);
  int og[MI], ox[NI];
#pragma unroll
  for (int i = 0; i < MI; ++i) og[i] = (8 * lc + key) * BM * 2 + (((wm / 32 + i) ^ key) * 8 + quarter) * 8;
#pragma unroll
  for (int j = 0; j < NI; ++j) ox[j] = GU * 16 + (8 * lc + key) * BN * 2 + (((wn / 32 + j) ^ key) * 8 + xq) * 8;
  fx16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  auto load = [&](uint4* l, int64_t left) __attribute__((always_inline)) {
    sg.load(l, tid, wave, left);
    sx.load(l + GU, tid, wave, left);
  };
  struct Both { short4v lo, hi; };
  auto step = [&](uint4* l, uint4* next, int64_t left) __attribute__((always_inline)) {      // left: rows after this step's
    __builtin_amdgcn_s_waitcnt(0x0f70);           // vmcnt(0): this wave's part of the step has arrived
    __syncthreads();                              // everybody's has, and the other buffer's readers are done
    if (left > 0) load(next, left);
    const char* p = reinterpret_cast<const char*>(l);
#pragma unroll
    for (int kk = 0; kk < kStepRows / 16; ++kk) {
      TX8 fg[MI], fx[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const char* q = p + og[i] + kk * 16 * BM * 2;
        fg[i] = __builtin_bit_cast(TX8, Both{read_transposed(q), read_transposed(q + 4 * BM * 2)});
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const char* q = p + ox[j] + kk * 16 * BN * 2;
        fx[j] = __builtin_bit_cast(TX8, Both{read_transposed(q), read_transposed(q + 4 * BN * 2)});
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mfma32(fx[j], fg[i], acc[i][j]);
    }
  };
  load(lds0, m1 - m0);
  for (int64_t m = m0; m < m1; m += 2 * kStepRows) {
    step(lds0, lds1, m1 - m - kStepRows);
    if (m + kStepRows < m1) step(lds1, lds0, m1 - m - 2 * kStepRows);
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int n = n0 + wm + 32 * i + lr;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int k = k0 + wn + 32 * j + 16 * lc;
      if (n >= a.N) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {               // 8 divides K
        if (k + 8 * h >= a.K) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[i][j][8 * h + e];
        const int64_t o = (int64_t)n * a.K + k + 8 * h;
        if (a.part || a.out32) {
          float* y = a.part ? a.part + (int64_t)z * a.N * a.K + o : static_cast<float*>(a.out) + o;
          reinterpret_cast<float4*>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          store_v<8>(static_cast<T*>(a.out) + o, v);
        }
      }
    }
  }
}

// The slabs' sums in order, 4 values a thread
template <typename T>
__global__ __launch_bounds__(256) void k_weight_sum(const float* part, int slabs, int64_t n, T* out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  int z = 0;
  for (; z + 4 <= slabs; z += 4) {
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(part + (z + k) * n + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) { s[0] += v[k].x; s[1] += v[k].y; s[2] += v[k].z; s[3] += v[k].w; }
  }
  for (; z < slabs; ++z) {
    const float4 v = *reinterpret_cast<const float4*>(part + z * n + i);
    s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
  }
  store_v<4>(out + i, s);
}

struct WeightPlan {
  int tile, slabs;
  int64_t slab;
};

// Tile and slabs by an estimate of the time (us): a step takes longer the more workgroups share L2 (128 x 128: 0.66 alone, 0.86 with
// one a CU, 1.06 with two; 256 x 256: 1.32 and 1.7), and slabs write and read their sums. 128 x 128 / 256 x 256 at their best
// slabs, measured: 1536 x 768 over 16384 rows 57 (7 slabs) / 65 (12), over 4097 27 (3) / 37 (7); 512 x 2048 over 65536 153 (8) /
// 145 (16); 2048 x 2048 over 512 10.8 (1) / 17.9 (1); 4096 x 4096 over 4096 149 / 112 (1). asrn_gemm's kernels, through registers: 76,
// 39, 176, 49 and 146.
static WeightPlan weight_plan(int64_t M, int64_t N, int64_t K, int tile, int slabs) {
  WeightPlan best = {};
  float least = 0.f;
  const int64_t steps = (M + kStepRows - 1) / kStepRows;
  for (int b : {128, 256}) {
    if (tile && tile != b) continue;
    const int64_t tiles = ((N + b - 1) / b) * ((K + b - 1) / b), card = b == 128 ? 512 : 256;
    for (int64_t s = slabs ? slabs : 1; s <= (slabs ? slabs : 128); ++s) {
      const int64_t per = (steps + s - 1) / s, n = (steps + per - 1) / per, groups = tiles * n;
      if (s > 1 && !slabs && (groups > card || s > steps)) break;
      const float alone = b == 128 ? 0.66f : 1.32f, shared = b == 128 ? 0.2f : 0.38f;
      const int64_t whole = groups / card, rest = groups % card;
      const float us = 4.f + per * (whole * (alone + shared * card / 256) + (rest ? alone + shared * rest / 256 : 0.f)) +
                       (n > 1 ? 3.f + n * N * K * 8 / 5.0e6f : 0.f);
      if (!best.tile || us < least) {
        least = us;
        best = {b, (int)n, per * kStepRows};
      }
    }
  }
  return best;
}

static int64_t weight_bytes(const WeightPlan& p, int64_t N, int64_t K) { return p.slabs > 1 ? p.slabs * N * K * 4 : 0; }

}  // namespace asrn

using namespace asrn;

static bool weight_sizes(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && N >= 0 && K >= 0 && M < ((int64_t)1 << 36) && N < (1 << 21) && K < (1 << 21) && N % 8 == 0 && K % 8 == 0;
}

extern "C" int64_t asrn_weight_grad_workspace(int64_t M, int64_t N, int64_t K, int32_t tile, int32_t slabs) {
  if (slabs < 0 || !weight_sizes(M, N, K) || (tile != 0 && tile != 128 && tile != 256)) return -1;
  return M == 0 || N == 0 || K == 0 ? 0 : weight_bytes(weight_plan(M, N, K, tile, slabs), N, K);
}

extern "C" int asrn_weight_grad(const void* g, int64_t ldg, const void* x, int64_t ldx, int32_t type, int64_t M, int64_t N,
                                int64_t K, void* out, int32_t out_fp32, int32_t tile, int32_t slabs, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  const char* what = "asrn_weight_grad";
  ASRN_REQUIRE(type == 1 || type == 2, "%s: type %d: 16-bit operands are needed", what, type);
  ASRN_REQUIRE(weight_sizes(M, N, K), "%s: bad sizes M=%lld N=%lld K=%lld (multiples of 8 below 2^21)", what, (long long)M,
               (long long)N, (long long)K);
  ASRN_REQUIRE((tile == 0 || tile == 128 || tile == 256) && slabs >= 0, "%s: unknown tile %d or slabs %d", what, tile, slabs);
  if (M == 0 || N == 0 || K == 0) return 0;
  ASRN_REQUIRE(g && x && out, "%s: null pointer", what);
  ASRN_REQUIRE(ldg >= N && ldx >= K && ldg % 8 == 0 && ldx % 8 == 0 && ldg < (1 << 21) && ldx < (1 << 21),
               "%s: leading dimensions must be multiples of 8 that hold a row, below 2^21 (ldg=%lld ldx=%lld)", what,
               (long long)ldg, (long long)ldx);
  ASRN_REQUIRE(!(((uintptr_t)g | (uintptr_t)x | (uintptr_t)out) & 15), "%s: misaligned operand", what);
  const WeightPlan p = weight_plan(M, N, K, tile, slabs);
  const int64_t need = weight_bytes(p, N, K);
  ASRN_REQUIRE(need == 0 || (workspace && !((uintptr_t)workspace & 15) && workspace_bytes >= need),
               "%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", what, (long long)need, (long long)workspace_bytes);
  WeightGrad a = {g, ldg, x, ldx, M, p.slab, (int)N, (int)K, (int)((N + p.tile - 1) / p.tile), (int)((K + p.tile - 1) / p.tile),
                  p.slabs, need ? (float*)workspace : nullptr, out, out_fp32};
  const int64_t total = (int64_t)a.tn * a.tk * a.slabs;
  ASRN_REQUIRE(total < (1 << 30) && N * K < ((int64_t)1 << 34), "%s: too many tiles", what);
  const unsigned grid = (unsigned)((total + kXcdCount - 1) / kXcdCount * kXcdCount);
  hipStream_t st = (hipStream_t)stream;
  auto run = [&](auto t) {
    using T = decltype(t);
    if (p.tile == 256) hipLaunchKernelGGL((k_weight_grad<T, 256, 256, 2, 4>), dim3(grid), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((k_weight_grad<T, 128, 128, 2, 2>), dim3(grid), dim3(256), 0, st, a);
    if (a.part) {
      const dim3 blocks((unsigned)((N * K / 4 + 255) / 256));
      if (out_fp32) hipLaunchKernelGGL(k_weight_sum<float>, blocks, dim3(256), 0, st, a.part, a.slabs, N * K, (float*)out);
      else hipLaunchKernelGGL(k_weight_sum<T>, blocks, dim3(256), 0, st, a.part, a.slabs, N * K, (T*)out);
    }
    return check_launch(what);
  };
  return type == 1 ? run(bf16_t{}) : run(fp16_t{});
}
