// A product with its epilogue: y = [res +] act(x W^T + bias), x (M, K), W (N, K), and the gradient before the activation.
//
// 16-bit operands run on the matrix cores: a workgroup forms a BM x BN tile in steps of 64 k. The operands come in 16-byte
// units of 8 k and lie in LDS as units whose column is exchanged by the row's number, so that 8 lanes that read neighbouring
// rows use all banks. Rows of whole units on 16-byte boundaries go from memory straight to LDS (k_linear_direct), others
// through registers one step ahead (k_linear). The matrix instruction's rows are W's, in an order
// that leaves a lane with 16 neighbouring columns of one row of y: the epilogue reads and writes whole vectors from the
// accumulators, with no pass through LDS. Sums are fp32; the activation's input (kept in the operands' type for the backward)
// and y are rounded once each.
// Few rows (k_linear_rows, one token of a few texts) read W once: see there. fp32 operands run on asrn_gemm's kernel, with
// this epilogue.
#include "linear_act.h"

namespace asrn {

struct Linear {
  const void* x; int64_t ldx; const void* w; int64_t ldw;
  int M, N, K;
  Epilogue e;
  int tm, tn;
};

// 16 neighbouring results of row m from column n on, all in the matrix, every operand read and written in vectors of 4 or more
template <typename T>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t m, int n, float (&v)[16]) {
  constexpr int V = 16;
  if (e.bias) {
    float b[4];
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      load_v<4>(static_cast<const T*>(e.bias) + n + k, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k + i] += b[i];
    }
  }
  if (e.pre) {                    // past the caches: the backward reads it much later (16384 x 768 x 1536 with GELU 69 -> 67 us)
    typedef T TV __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int k = 0; k < V; k += 8) {
      TV q;
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = (T)v[k + i];
      __builtin_nontemporal_store(q, reinterpret_cast<TV*>(static_cast<T*>(e.pre) + m * e.ldp + n + k));
    }
  }
  if (e.act == kActGelu) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = gelu16(v[k]);
  } else if (e.act == kActSilu) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = activate(v[k], kActSilu);
  }
  if (e.res) {
    float b[4];
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      if (e.res32) load_v<4>(static_cast<const float*>(e.res) + m * e.ldr + n + k, b);
      else load_v<4>(static_cast<const T*>(e.res) + m * e.ldr + n + k, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k + i] += b[i];
    }
  }
  if (e.y32) {
    float* y = static_cast<float*>(e.y) + m * e.ldy + n;
#pragma unroll
    for (int k = 0; k < V; k += 4) *reinterpret_cast<float4*>(y + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
  } else {
    store_v<V>(static_cast<T*>(e.y) + m * e.ldy + n, v);
  }
}

// A wave's results: lane (lr, lc) holds, of 32 x 32 block (i, j), row 32 i + lr and columns 32 j + 16 lc + 0 .. 15. Where they
// are not whole vectors in the matrix, one after the other, through LDS (16 floats a thread, whose buffers are done with).
template <typename T, int MI, int NI, int THR>
__device__ __forceinline__ void finish_all(const Linear& g, fx16 (&acc)[MI][NI], int m0, int n0, float* lds) {
  const int lane = lane_id(), lr = lane & 31, lc = lane >> 5;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + 32 * i + lr;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n = n0 + 32 * j + 16 * lc;
      if (m >= g.M || n >= g.N) continue;
      if (g.e.vec && n + 16 <= g.N) {
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[i][j][e];
        finish<T>(g.e, m, n, v);
      } else {
        float* mine = lds + threadIdx.x;
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[e * THR] = acc[i][j][e];
        const int left = g.N - n < 16 ? g.N - n : 16;
#pragma unroll 1
        for (int e = 0; e < left; ++e) g.e.template one<T>(m, n + e, mine[e * THR]);
      }
    }
  }
}

// An operand's share of a step: R rows by 64 k, units of 8 k; a thread loads U units, 8 neighbouring threads a row's 128 bytes.
// The units are read wherever they lie, those of the last step element by element.
template <typename T, int R, int THR>
struct Units {
  static constexpr int U = R * 8 / THR;
  static_assert(R * 8 % THR == 0 && THR % 8 == 0, "whole units");
  const T* base;
  unsigned at[U], c;              // byte offsets of the rows; the thread's column of units
  uint4 v[U];
  // rows past the matrix repeat its last one: their results are not stored
  __device__ __forceinline__ void start(const void* X, int64_t ld, int r0, int rows, int tid) {
    base = static_cast<const T*>(X) + r0 * ld;
    c = tid % 8;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = (tid + THR * i) / 8;
      at[i] = (unsigned)((r0 + r < rows ? r : rows - 1 - r0) * ld + 8 * c) * (unsigned)sizeof(T);
    }
  }
  // k past K reads as 0
  __device__ __forceinline__ void load(int k0, int K) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const T* p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + at[i]) + k0;
      if (k0 + 64 <= K) {                         // uniform
        __builtin_memcpy(&v[i], p, 16);
      } else {
        unsigned q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = k0 + 8 * (int)c + j < K ? __builtin_bit_cast(unsigned short, p[j]) : 0u;
        v[i] = make_uint4(q[0] | q[1] << 16, q[2] | q[3] << 16, q[4] | q[5] << 16, q[6] | q[7] << 16);
      }
    }
  }
  template <typename KEY>
  __device__ __forceinline__ void store(uint4* lds, int tid, KEY key) const {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = (tid + THR * i) / 8;
      lds[r * 8 + (c ^ key(r))] = v[i];
    }
  }
};

// the units' exchange: 8 rows that a quarter of a wave reads at once have 8 keys. x's rows are read in order, W's in the
// order of w_row: lanes 0-3 and 4-7 read rows 4 q + r and 16 + 4 q + r
__device__ __forceinline__ int x_key(int r) { return r & 7; }
__device__ __forceinline__ int w_key(int r) { return (r & 3) | (r >> 2 & 4); }
__device__ __forceinline__ int w_row(int i) { return (i >> 2 & 1) * 16 + (i >> 3) * 4 + (i & 3); }

// Operands on any boundary, of any width
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_linear(Linear g) {
  constexpr int THR = 64 * WM * WN, BK = 64, MI = BM / WM / 32, NI = BN / WN / 32;
  typedef T TX8 __attribute__((ext_vector_type(8)));
  __shared__ uint4 lds[2][(BM + BN) * 8];
  // XCD i takes a contiguous range of tiles, n fastest: tiles that share rows of x share its L2
  const int total = g.tm * g.tn, per = (total + kXcdCount - 1) / kXcdCount;
  const int tile = (int)(blockIdx.x % kXcdCount) * per + (int)(blockIdx.x / kXcdCount);
  if (tile >= total || (int)(blockIdx.x / kXcdCount) >= per) return;
  const int m0 = tile / g.tn * BM, n0 = tile % g.tn * BN;
  const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, lr = lane & 31, lc = lane >> 5;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN), wr = w_row(lr);
  Units<T, BM, THR> ux;
  Units<T, BN, THR> uw;
  ux.start(g.x, g.ldx, m0, g.M, tid);
  uw.start(g.w, g.ldw, n0, g.N, tid);
  fx16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  ux.load(0, g.K);
  uw.load(0, g.K);
  int buf = 0;
  for (int k = 0; k < g.K; k += BK, buf ^= 1) {
    uint4 *lx = lds[buf], *lw = lx + BM * 8;
    ux.store(lx, tid, x_key);                     // read two steps ago: the last barrier lies between
    uw.store(lw, tid, w_key);
    __syncthreads();
    if (k + BK < g.K) {
      ux.load(k + BK, g.K);                       // in flight under this step's products
      uw.load(k + BK, g.K);
    }
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      TX8 fx[MI], fw[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = wm + 32 * i + lr;
        fx[i] = __builtin_bit_cast(TX8, lx[r * 8 + ((2 * kk + lc) ^ x_key(r))]);
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int r = wn + 32 * j + wr;
        fw[j] = __builtin_bit_cast(TX8, lw[r * 8 + ((2 * kk + lc) ^ w_key(r))]);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mfma32(fw[j], fx[i], acc[i][j]);
    }
  }
  finish_all<T, MI, NI, THR>(g, acc, m0 + wm, n0 + wn, reinterpret_cast<float*>(lds));
}

// Tiles in order: 4 rows of them at a time, column after column, so that the tiles which an XCD forms at once are as many
// down as across and read as little as they can (8192 x 2048 x 4096 in tiles of 256 x 256: row by row 130 us, so 124)
__device__ __forceinline__ void place_tile(int t, int tm, int tn, int& m, int& n) {
  constexpr int G = 4;
  const int group = t / (G * tn), first = group * G, rows = tm - first < G ? tm - first : G, r = t - group * G * tn;
  m = first + r % rows;
  n = r / rows;
}

// The same with the operands straight from memory to LDS, without registers in between (whole steps; a last part of one goes
// through them). Two buffers that the compiler can tell apart: a step's loads are issued before the products of the one
// before and waited for after them, with one barrier a step.
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_linear_direct(Linear g) {
  constexpr int THR = 64 * WM * WN, BK = 64, MI = BM / WM / 32, NI = BN / WN / 32, UX = BM * 8 / THR, UW = BN * 8 / THR;
  static_assert(BM * 8 % THR == 0 && BN * 8 % THR == 0, "whole units");
  typedef T TX8 __attribute__((ext_vector_type(8)));
  __shared__ uint4 lds0[(BM + BN) * 8];
  __shared__ uint4 lds1[(BM + BN) * 8];
  const int total = g.tm * g.tn, per = (total + kXcdCount - 1) / kXcdCount;
  const int tile = (int)(blockIdx.x % kXcdCount) * per + (int)(blockIdx.x / kXcdCount);
  if (tile >= total || (int)(blockIdx.x / kXcdCount) >= per) return;
  int m0, n0;
  place_tile(tile, g.tm, g.tn, m0, n0);
  m0 *= BM;
  n0 *= BN;
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, lc = lane >> 5;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN), wr = w_row(lr);
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<T*>(static_cast<const T*>(g.x) + (int64_t)m0 * g.ldx), 0, kPast, 0x00027000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<T*>(static_cast<const T*>(g.w) + (int64_t)n0 * g.ldw), 0, kPast, 0x00027000);
  unsigned ax[UX], aw[UW];        // byte offsets of the unit that lies where the thread's share of LDS does
#pragma unroll
  for (int i = 0; i < UX; ++i) {
    const int r = (tid + THR * i) / 8;
    ax[i] = (unsigned)((m0 + r < g.M ? r : g.M - 1 - m0) * g.ldx + 8 * (tid % 8 ^ x_key(r))) * 2u;
  }
#pragma unroll
  for (int i = 0; i < UW; ++i) {
    const int r = (tid + THR * i) / 8;
    aw[i] = (unsigned)((n0 + r < g.N ? r : g.N - 1 - n0) * g.ldw + 8 * (tid % 8 ^ w_key(r))) * 2u;
  }
  auto load = [&](uint4* l, int k) __attribute__((always_inline)) {
    const unsigned off = (unsigned)k * 2u;
    if (k + BK <= g.K) {
#pragma unroll
      for (int i = 0; i < UX; ++i)
        to_lds(rx, l + wave * 64 + THR * i, ax[i], off);
#pragma unroll
      for (int i = 0; i < UW; ++i)
        to_lds(rw, l + BM * 8 + wave * 64 + THR * i, aw[i], off);
    } else {                                      // the last part of a step: k past K is 0
#pragma unroll
      for (int i = 0; i < UX; ++i) {
        const int r = (tid + THR * i) / 8;
        l[tid + THR * i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
            rx, k + 8 * (tid % 8 ^ x_key(r)) < g.K ? ax[i] : kPast, off, 0));
      }
#pragma unroll
      for (int i = 0; i < UW; ++i) {
        const int r = (tid + THR * i) / 8;
        l[BM * 8 + tid + THR * i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
            rw, k + 8 * (tid % 8 ^ w_key(r)) < g.K ? aw[i] : kPast, off, 0));
      }
    }
  };
  fx16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  auto step = [&](uint4* l, uint4* next, int k) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);           // vmcnt(0): this wave's part of the step has arrived
    __syncthreads();                              // everybody's has, and the other buffer's readers are done
    if (k + BK < g.K) load(next, k + BK);
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      TX8 fx[MI], fw[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = wm + 32 * i + lr;
        fx[i] = __builtin_bit_cast(TX8, l[r * 8 + ((2 * kk + lc) ^ x_key(r))]);
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int r = wn + 32 * j + wr;
        fw[j] = __builtin_bit_cast(TX8, l[BM * 8 + r * 8 + ((2 * kk + lc) ^ w_key(r))]);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mfma32(fw[j], fx[i], acc[i][j]);
    }
  };
  load(lds0, 0);
  for (int k = 0; k < g.K; k += 2 * BK) {
    step(lds0, lds1, k);
    if (k + BK < g.K) step(lds1, lds0, k + BK);
  }
  finish_all<T, MI, NI, THR>(g, acc, m0 + wm, n0 + wn, reinterpret_cast<float*>(lds0));
}

// The sums over a wave's lanes of V values each (V = 16, 32 or 64), one a lane: at every distance a lane gives half of its
// values away and adds the other half's; lane l ends with value sum_of_lane(l). The halves and the rows of 16 change places
// by one instruction a pair; distances 8 to 1 by DPP (half a row mirrored stands for distance 4: its bit differs too).
template <int V>
__device__ __forceinline__ int sum_of_lane(int lane) {
  const int b5 = lane >> 5 & 1, b4 = lane >> 4 & 1, low = (lane >> 3 & 1) * 8 + (lane >> 2 & 1) * 4 + (lane & 3);
  if (V == 64) return b5 * 32 + b4 * 16 + low;
  if (V == 32) return b4 ? -1 : b5 * 16 + low;
  return b5 || b4 ? -1 : low;
}
template <int CTRL>
__device__ __forceinline__ float give(float keep, float away) { return keep + dpp<CTRL>(away); }
template <int V>
__device__ __forceinline__ float lane_sums(float* v, int lane) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (V == 64) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 32]), false, false);
      v[i] = __uint_as_float(q[0]) + __uint_as_float(q[1]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 16]), false, false);
      v[i] = __uint_as_float(q[0]) + __uint_as_float(q[1]);
    }
  } else if constexpr (V == 32) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 16]), false, false);
      v[i] = __uint_as_float(q[0]) + __uint_as_float(q[1]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += __shfl_xor(v[i], 16, 64);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] += __shfl_xor(v[i], 32, 64);
      v[i] += __shfl_xor(v[i], 16, 64);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = give<0x128>(lane & 8 ? v[i + 8] : v[i], lane & 8 ? v[i] : v[i + 8]);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = give<0x141>(lane & 4 ? v[i + 4] : v[i], lane & 4 ? v[i] : v[i + 4]);
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = give<0x4E>(lane & 2 ? v[i + 2] : v[i], lane & 2 ? v[i] : v[i + 2]);
  return give<0xB1>(lane & 1 ? v[1] : v[0], lane & 1 ? v[0] : v[1]);
#else
  return 0.f;
#endif
}

// Few rows (M <= 16): W is read once and each of its values meets every row, so the weights' bytes bound it. A wave takes 4
// rows of W (columns of y) and all rows of x; its lanes run along k in units of 4, each with 4 x MR sums, which then
// meet by a transposing exchange. x comes from the caches. 16 rows, 768 x 1536 fp32: 6.7 us, where 4.7 MB of weights from the
// caches and a launch are the rest of a call's 7.2.
template <typename T, int MR, bool VEC>
__global__ __launch_bounds__(256) void k_linear_rows(Linear g) {
  constexpr int NR = 4, UN = sizeof(T) == 4 ? 4 : 8;
  __shared__ float red[4][64];
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  // the workgroup's 4 waves share 4 columns and cut k
  const int n0 = blockIdx.x * NR, m0 = blockIdx.y * MR;
  float acc[NR][MR];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[n][m] = 0.f;
  const T *x = static_cast<const T*>(g.x), *w = static_cast<const T*>(g.w);
  for (int k = (wave * 64 + lane) * UN; k < g.K; k += 256 * UN) {
    float a[NR][UN];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const T* p = w + (int64_t)(n0 + n < g.N ? n0 + n : g.N - 1) * g.ldw + k;
      if constexpr (VEC) {
        load_v<UN>(p, a[n]);
      } else {
#pragma unroll
        for (int j = 0; j < UN; ++j) a[n][j] = k + j < g.K ? (float)p[j] : 0.f;
      }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const T* p = x + (int64_t)(m0 + m < g.M ? m0 + m : g.M - 1) * g.ldx + k;
      float b[UN];
      if constexpr (VEC) {
        load_v<UN>(p, b);
      } else {
#pragma unroll
        for (int j = 0; j < UN; ++j) b[j] = k + j < g.K ? (float)p[j] : 0.f;
      }
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < UN; ++j) acc[n][m] = fmaf(a[n][j], b[j], acc[n][m]);
    }
  }
  const float mine = lane_sums<NR * MR>(&acc[0][0], lane);
  red[wave][lane] = mine;
  __syncthreads();
  const int mine_is = sum_of_lane<NR * MR>(lane);
  if (wave == 0 && mine_is >= 0) {
    const int n = n0 + mine_is / MR, m = m0 + mine_is % MR;
    if (n < g.N && m < g.M) {
      const float v = ((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane];
      g.e.template one<T>(m, n, v);
    }
  }
}

// The gradient before the activation, gp = gy act'(pre), and its column sums (the bias gradient) from the unrounded values: CW
// lanes of V columns by 256 / CW rows a workgroup, a slab of rows each, 4 rows of a lane under way at once.
template <typename T, typename G, int V, int CW>
__global__ __launch_bounds__(256) void k_act_grad(const G* gy, int64_t ldg, const T* pre, int64_t ldp, int act, int64_t M, int N,
                                                  int64_t slab, T* gp, float* part) {
  constexpr int RL = 256 / CW, R = 4;
  __shared__ float red[RL][CW * V];
  const int cl = threadIdx.x % CW, rl = threadIdx.x / CW;
  const int c = (blockIdx.x * CW + cl) * V;
  const int64_t r0 = blockIdx.y * slab, r1 = r0 + slab < M ? r0 + slab : M;
  float s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = 0.f;
  if (c < N) {
    for (int64_t r = r0 + rl; r < r1; r += R * RL) {
      float g[R][V], p[R][V];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int64_t q = r + k * RL < r1 ? r + k * RL : r1 - 1;       // past the slab: its last row, neither stored nor added
        load_v<V>(gy + q * ldg + c, g[k]);
        if (act != kActNone) load_v<V>(pre + q * ldp + c, p[k]);
      }
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (r + k * RL >= r1) break;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (act == kActGelu) g[k][v] *= sizeof(T) == 2 ? gelu16_grad(p[k][v]) : activate_grad(p[k][v], kActGelu);
          else if (act == kActSilu) g[k][v] *= activate_grad(p[k][v], kActSilu);
          s[v] += g[k][v];
        }
        if (gp) store_v<V>(gp + (r + k * RL) * N + c, g[k]);
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int v = 0; v < V; ++v) red[rl][cl * V + v] = s[v];
  __syncthreads();
  for (int i = threadIdx.x; i < CW * V; i += 256) {
    const int64_t n = (int64_t)blockIdx.x * CW * V + i;
    float v = red[0][i];
#pragma unroll
    for (int k = 1; k < RL; ++k) v += red[k][i];
    if (n < N) part[blockIdx.y * (int64_t)N + n] = v;
  }
}

template <typename T, bool VEC>
static int launch_rows(const Linear& g, hipStream_t st) {
  const unsigned gx = (unsigned)((g.N + 3) / 4);
  ASRN_REQUIRE(grid_ok((int64_t)gx * 256, 256), "asrn_linear_act_fwd: too many columns");
  if (g.M <= 4)
    hipLaunchKernelGGL((k_linear_rows<T, 4, VEC>), dim3(gx, (g.M + 3) / 4), dim3(256), 0, st, g);
  else if (g.M <= 8)
    hipLaunchKernelGGL((k_linear_rows<T, 8, VEC>), dim3(gx, (g.M + 7) / 8), dim3(256), 0, st, g);
  else
    hipLaunchKernelGGL((k_linear_rows<T, 16, VEC>), dim3(gx, (g.M + 15) / 16), dim3(256), 0, st, g);
  return check_launch("asrn_linear_act_fwd");
}

template <typename T, int BM, int BN, int WM, int WN>
static int launch_tiles(Linear g, bool vec, hipStream_t st) {
  g.tm = (g.M + BM - 1) / BM;
  g.tn = (g.N + BN - 1) / BN;
  const int64_t tiles = (int64_t)g.tm * g.tn;
  ASRN_REQUIRE(grid_ok((tiles + kXcdCount) * (64 * WM * WN), 64 * WM * WN), "asrn_linear_act_fwd: too many tiles");
  const unsigned grid = (unsigned)((tiles + kXcdCount - 1) / kXcdCount * kXcdCount);
  if (vec) hipLaunchKernelGGL((k_linear_direct<T, BM, BN, WM, WN>), dim3(grid), dim3(64 * WM * WN), 0, st, g);
  else hipLaunchKernelGGL((k_linear<T, BM, BN, WM, WN>), dim3(grid), dim3(64 * WM * WN), 0, st, g);
  return check_launch("asrn_linear_act_fwd");
}

constexpr int kFewRows = 16;

// The tile by an estimate of the time: a start of 3 us and 4 a 768 of k (the steps wait for their loads), and for each tile that a
// CU takes its products at 2.5 PFLOP/s times what the tile needs over that. Measured (us; 64 x 64, 128 x 128, 256 x 192,
// 256 x 256, without an epilogue): 1024 x 768 x 768 8.2 / 12.2 / 18.5 / 23.4, 2048 x 768 x 1536 (M, K, N) 11.5 / 16.1 / 24.3 /
// 31.3, 4096 x 1024 x 1024 16.1 / 17.9 / 28.3 / 36.0, 16384 x 768 x 1536 64 / 53 / 47 / 54, 4096 x 4096 x 4096 203 / 136 / 166 /
// 116, 8192 x 2048 x 4096 211 / 146 / 149 / 124 (the library's product alone: 46 at the fourth, 108 and 106 at the last two).
static int tile_of(int64_t M, int64_t N, int64_t K) {
  struct Tile { int bm, bn; float over; };
  static const Tile all[] = {{64, 64, 2.5f}, {128, 128, 2.3f}, {256, 192, 1.9f}, {256, 256, 1.75f}};
  int best = 0;
  float least = 0.f;
  for (const Tile& t : all) {
    const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
    const float us = 3.f + 4.f * K / 768.f + (float)((tiles + 255) / 256) * t.over * (2.f * t.bm * t.bn * K / (2.5e9f / 256));
    if (best == 0 || us < least) {
      least = us;
      best = t.bm << 8 | (t.bn & 255);
    }
  }
  return best;
}

}  // namespace asrn

using namespace asrn;

static bool aligned(const void* p, int64_t ld, int bytes, int values) {
  return ((uintptr_t)p % (uintptr_t)(bytes * values)) == 0 && ld % values == 0;
}

extern "C" int64_t asrn_linear_act_workspace(int64_t M, int64_t N, int64_t K, int32_t type) {
  if (M < 0 || N < 0 || K < 1 || !type_ok(type)) return -1;
  return type == 0 && M > kFewRows && N > 0 ? gemm_epilogue_workspace(M, N, K) : 0;
}

extern "C" int asrn_linear_act_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t type, const void* bias,
                                   int64_t M, int64_t N, int64_t K, int32_t act, const void* res, int64_t ldr, int32_t res_fp32,
                                   void* pre, int64_t ldp, void* y, int64_t ldy, int32_t y_fp32, int32_t tile, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const char* what = "asrn_linear_act_fwd";
  ASRN_REQUIRE(type_ok(type), "%s: type %d", what, type);
  ASRN_REQUIRE(M >= 0 && N >= 0 && K >= 1 && M < (1 << 30) && N < (1 << 30) && K < (1 << 30) && act >= 0 && act <= 2,
               "%s: bad sizes M=%lld N=%lld K=%lld act=%d", what, (long long)M, (long long)N, (long long)K, act);
  if (M == 0 || N == 0) return 0;
  ASRN_REQUIRE(x && w && y, "%s: null pointer", what);
  ASRN_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!res || ldr >= N) && (!pre || ldp >= N) && ldx < (1 << 21) && ldw < (1 << 21),
               "%s: leading dimensions must hold a row and x's and W's be below 2^21 (ldx=%lld ldw=%lld ldy=%lld)", what,
               (long long)ldx, (long long)ldw, (long long)ldy);
  ASRN_REQUIRE(tile == 0 || tile == (256 << 8) || tile == (256 << 8 | 192) || tile == (128 << 8 | 128) || tile == (64 << 8 | 64),
               "%s: unknown tile %d", what, tile);
  const int b = type_bytes(type), by = y_fp32 ? 4 : b, br = res_fp32 ? 4 : b;
  Linear g = {x, ldx, w, ldw, (int)M, (int)N, (int)K, {}, 0, 0};
  g.e = {bias, res, ldr, pre, ldp, y, ldy, act, res_fp32, y_fp32, 0};
  // vectors of the epilogue: 16 results of the operands' type, 4 of fp32 and of what it reads
  g.e.vec = (!bias || aligned(bias, 4, b, 4)) && (!res || aligned(res, ldr, br, 4)) && (!pre || aligned(pre, ldp, b, 16)) &&
            aligned(y, ldy, by, y_fp32 ? 4 : 16);
  hipStream_t st = (hipStream_t)stream;
  if (M <= kFewRows)
    return with_type(type, [&](auto t) {
      using T = decltype(t);
      constexpr int un = sizeof(T) == 4 ? 4 : 8;
      const bool vec = K % un == 0 && aligned(x, ldx, b, un) && aligned(w, ldw, b, un);
      return vec ? launch_rows<T, true>(g, st) : launch_rows<T, false>(g, st);
    });
  if (type == 0) return gemm_epilogue((const float*)x, ldx, (const float*)w, ldw, M, N, K, g.e, workspace, workspace_bytes, st);
  const bool vec = K % 8 == 0 && aligned(x, ldx, 2, 8) && aligned(w, ldw, 2, 8);
  const int how = tile ? tile : tile_of(M, N, K);
  auto run = [&](auto t) {
    using T = decltype(t);
    switch (how) {
      case 256 << 8: return launch_tiles<T, 256, 256, 2, 4>(g, vec, st);
      case 256 << 8 | 192: return launch_tiles<T, 256, 192, 4, 2>(g, vec, st);
      case 128 << 8 | 128: return launch_tiles<T, 128, 128, 2, 2>(g, vec, st);
      default: return launch_tiles<T, 64, 64, 2, 2>(g, vec, st);
    }
  };
  return type == 1 ? run(bf16_t{}) : run(fp16_t{});
}

// column lanes of a workgroup, 64 or fewer where those leave fewer of them idle (768 columns by 8: 3 times 32)
static int lanes_of(int64_t N, int V) {
  const int64_t groups = (N + V - 1) / V;
  int best = 64;
  for (int cw : {32, 16})
    if ((groups + cw - 1) / cw * cw < (groups + best - 1) / best * best) best = cw;
  return best;
}
// rows of a slab: enough slabs to fill the card, 4 rows a lane at least
static int64_t slab_of(int64_t M, int64_t N, int V) {
  const int cw = lanes_of(N, V);
  const int64_t cols = (N + (int64_t)cw * V - 1) / ((int64_t)cw * V), least = 4 * (256 / cw);
  int64_t n = 2048 / cols;
  if (n < 1) n = 1;
  const int64_t s = (M + n - 1) / n;
  return s < least ? least : (s + least - 1) / least * least;
}

extern "C" int64_t asrn_act_grad_workspace(int64_t M, int64_t N) {
  if (M < 0 || N < 0) return -1;
  if (M == 0 || N == 0) return 0;
  int64_t s = slab_of(M, N, 1);                   // the width is chosen by the addresses: the smallest slab of the three
  for (int V : {4, 8})
    if (slab_of(M, N, V) < s) s = slab_of(M, N, V);
  return (M + s - 1) / s * N * 4;
}

extern "C" int asrn_act_grad(const void* gy, int64_t ldg, int32_t gy_fp32, const void* pre, int64_t ldp, int32_t type, int64_t M,
                             int64_t N, int32_t act, void* gp, float* colsum, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  const char* what = "asrn_act_grad";
  ASRN_REQUIRE(type_ok(type), "%s: type %d", what, type);
  ASRN_REQUIRE(M >= 0 && N >= 0 && M < ((int64_t)1 << 40) && N < (1 << 30) && act >= 0 && act <= 2,
               "%s: bad sizes M=%lld N=%lld act=%d", what, (long long)M, (long long)N, act);
  if (M == 0 || N == 0) return 0;
  ASRN_REQUIRE(gy && (gp || colsum) && (act == 0 || pre), "%s: null pointer", what);
  ASRN_REQUIRE(ldg >= N && (!pre || ldp >= N), "%s: leading dimensions must hold a row", what);
  const int b = type_bytes(type), bg = gy_fp32 ? 4 : b;
  const int W = type == 0 ? 4 : 8;
  const bool vec = N % W == 0 && aligned(gy, ldg, bg, W) && (!act || aligned(pre, ldp, b, W)) && (!gp || aligned(gp, N, b, W));
  const int V = vec ? W : 1;
  const int64_t slab = slab_of(M, N, V), slabs = (M + slab - 1) / slab;
  ASRN_REQUIRE(slabs < 65536, "%s: too many rows", what);
  float* part = nullptr;
  if (colsum) {
    ASRN_REQUIRE(workspace && !((uintptr_t)workspace & 15) && workspace_bytes >= slabs * N * 4,
                 "%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", what, (long long)(slabs * N * 4),
                 (long long)workspace_bytes);
    part = (float*)workspace;
  }
  const int cw = lanes_of(N, V);
  const dim3 grid((unsigned)((N + (int64_t)cw * V - 1) / ((int64_t)cw * V)), (unsigned)slabs);
  ASRN_REQUIRE(grid_ok((int64_t)grid.x * 256, 256), "%s: too many columns", what);
  hipStream_t st = (hipStream_t)stream;
  const int rc = with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr int WT = sizeof(T) == 4 ? 4 : 8;
    auto go = [&](auto g) {
      using G = decltype(g);
#define ASRN_ACT_GRAD(V, CW)                                                                                              \
  hipLaunchKernelGGL((k_act_grad<T, G, V, CW>), grid, dim3(256), 0, st, (const G*)gy, ldg, (const T*)pre, ldp, act, M, (int)N, \
                     slab, (T*)gp, part)
      if (vec) {
        if (cw == 64) ASRN_ACT_GRAD(WT, 64);
        else if (cw == 32) ASRN_ACT_GRAD(WT, 32);
        else ASRN_ACT_GRAD(WT, 16);
      } else {
        if (cw == 64) ASRN_ACT_GRAD(1, 64);
        else if (cw == 32) ASRN_ACT_GRAD(1, 32);
        else ASRN_ACT_GRAD(1, 16);
      }
#undef ASRN_ACT_GRAD
      return check_launch("asrn_act_grad");
    };
    return gy_fp32 ? go(float{}) : go(T{});
  });
  return rc || !colsum ? rc : group_sums(part, (int)slabs, (int)N, colsum, st);
}
