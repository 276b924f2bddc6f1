// int8 matrix product with scales: out[m][n] = round(xs[m] * ws[n] * sum_k x[m][k] w[n][k] + bias[n] + residual[m][n]),
// x [M][K] and w [N][K] int8 rows, int32 sums (exact: K <= 131071 keeps 128 * 128 * K below 2^31), the epilogue in fp32,
// one rounding to the output's type.
//
// dot_kernel: up to DOT_M rows of x.  The work is the stream of w: a wave reads 8 rows x 128 bytes per
// load (8 lanes a row, whole cache lines), takes v_dot4_i32_i8 against the rows of x, and the waves of a workgroup
// share the K axis.  16 rows x 64 bytes, the MFMA's own operand order, reads at 0.7 of that rate.
//
// tile_kernel: BM x BN outputs per workgroup.  Both operands go to LDS 128 bytes of K at a time by
// direct loads (8 rows x 128 bytes per wave and load), in two buffers: the loads of step s + 1 are in flight while the
// MFMAs of step s run.  16-byte chunk c of row r sits at slot c ^ (r & 7), so that the MFMA operand reads (one chunk
// of 16 or 32 rows) touch every bank once per phase.  w is the MFMA's first operand: a lane then holds four
// consecutive n of one m.  Rows past M or N read the last row, chunks past K the row's last chunk; what they add is
// masked (K, on x) or not stored (M, N).
//
// With few tiles the K axis is split over workgroups: int32 partials, summed by linear_join_kernel.
#pragma once
#include "common.h"
#include "rows.hip"

#include <algorithm>
#include <type_traits>

namespace tri {

constexpr int LIN_KS = 128;          // bytes of K per step
constexpr int LIN_MAX_K = 131071;
constexpr int64_t LIN_MAX_LD = 1 << 22;

struct LinearArgs {
  const int8_t* x;
  const int8_t* w;
  int64_t ldx, ldw;
  const float* xs;
  const float* ws;
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* out;
  int64_t ldo;
  int32_t* part;       // split sums [splits][m][n]
  int dtype;
  int m, n, k;
  int tiles_m, tiles_n, splits, per;  // per: 128-byte steps of a split
};

__device__ __forceinline__ float lin_load(const void* p, int64_t i, int dtype) {
  if (dtype == F32) return static_cast<const float*>(p)[i];
  if (dtype == BF16) return bf16f(static_cast<const uint16_t*>(p)[i]);
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void lin_load4(const void* p, int64_t i, int dtype, float (&v)[4]) {
  if (dtype == F32) {
    __builtin_memcpy(v, static_cast<const float*>(p) + i, 16);
  } else if (dtype == BF16) {
    uint16_t t[4];
    __builtin_memcpy(t, static_cast<const uint16_t*>(p) + i, 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = bf16f(t[j]);
  } else {
    _Float16 t[4];
    __builtin_memcpy(t, static_cast<const _Float16*>(p) + i, 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)t[j];
  }
}
__device__ __forceinline__ void lin_store4(void* p, int64_t i, int dtype, const float (&v)[4]) {
  if (dtype == F32) {
    __builtin_memcpy(static_cast<float*>(p) + i, v, 16);
  } else if (dtype == BF16) {
    uint16_t t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = f32_to_bf16(v[j]);
    __builtin_memcpy(static_cast<uint16_t*>(p) + i, t, 8);
  } else {
    _Float16 t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = (_Float16)v[j];
    __builtin_memcpy(static_cast<_Float16*>(p) + i, t, 8);
  }
}
__device__ __forceinline__ void lin_store(void* p, int64_t i, int dtype, float v) {
  if (dtype == F32) static_cast<float*>(p)[i] = v;
  else if (dtype == BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// outputs n .. n+3 of row m from their sums
__device__ __forceinline__ void lin_out4(const LinearArgs& a, int m, int n, float xs, const int (&acc)[4]) {
  if (n + 4 <= a.n) {
    float ws[4], v[4];
    __builtin_memcpy(ws, a.ws + n, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)acc[j] * (xs * ws[j]);
    if (a.bias) {
      float b[4];
      lin_load4(a.bias, n, a.dtype, b);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += b[j];
    }
    if (a.residual) {
      float r[4];
      lin_load4(a.residual, m * a.ldr + n, a.dtype, r);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += r[j];
    }
    lin_store4(a.out, m * a.ldo + n, a.dtype, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < a.n) {
        float v = (float)acc[j] * (xs * a.ws[n + j]);
        if (a.bias) v += lin_load(a.bias, n + j, a.dtype);
        if (a.residual) v += lin_load(a.residual, m * a.ldr + n + j, a.dtype);
        lin_store(a.out, m * a.ldo + n + j, a.dtype, v);
      }
  }
}

// the first `valid` of a chunk's 16 bytes (none for valid <= 0, all for valid >= 16)
__device__ __forceinline__ v4i lin_mask(v4i v, int valid) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = valid - 4 * j;
    v[j] &= n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
  }
  return v;
}

// ------------------------------------------------------------------ few rows
// MR rows of x, NR * 8 rows of w per workgroup, WAVES waves share K (wave w takes steps w, w + WAVES, ...: neighbouring
// cache lines at one time).
template <int MR, int NR, int WAVES, int U>
__global__ __launch_bounds__(WAVES * 64) void dot_kernel(LinearArgs a) {
  __shared__ int red[WAVES][MR][NR * 8];
  const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r8 = L >> 3, c = L & 7;
  const int n0 = blockIdx.x * (NR * 8);
  const int steps = (a.k + LIN_KS - 1) / LIN_KS;
  const int last_chunk = (a.k - 1) & ~15;
  const int8_t* wrow[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) wrow[i] = a.w + (int64_t)min(n0 + i * 8 + r8, a.n - 1) * a.ldw;
  const int8_t* xrow[MR];
#pragma unroll
  for (int i = 0; i < MR; ++i) xrow[i] = a.x + (int64_t)min(i, a.m - 1) * a.ldx;
  int acc[MR][NR] = {};
  auto step = [&](int s, bool tail) {
    const int kb = s * LIN_KS + c * 16, kc = min(kb, last_chunk);
    v4i w[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) w[i] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(wrow[i] + kc));
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      v4i x = *reinterpret_cast<const v4i*>(xrow[m] + kc);
      if (tail) x = lin_mask(x, a.k - kb);
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[m][i] = __builtin_amdgcn_sdot4(w[i][j], x[j], acc[m][i], false);
    }
  };
  const int full = a.k / LIN_KS;
  int s = wave;
  for (; s + (U - 1) * WAVES < full; s += U * WAVES) {
#pragma unroll
    for (int u = 0; u < U; ++u) step(s + u * WAVES, false);
  }
  for (; s < steps; s += WAVES) step(s, true);
  // the 8 lanes of a row, then the waves
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      int v = acc[m][i];
      v += __shfl_xor(v, 1);
      v += __shfl_xor(v, 2);
      v += __shfl_xor(v, 4);
      if (c == 0) red[wave][m][i * 8 + r8] = v;
    }
  __syncthreads();
  for (int o = threadIdx.x; o < MR * NR * 8; o += WAVES * 64) {
    const int m = o / (NR * 8), r = o % (NR * 8), n = n0 + r;
    if (m >= a.m || n >= a.n) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += red[w][m][r];
    float v = (float)sum * (a.xs[m] * a.ws[n]);
    if (a.bias) v += lin_load(a.bias, n, a.dtype);
    if (a.residual) v += lin_load(a.residual, m * a.ldr + n, a.dtype);
    lin_store(a.out, m * a.ldo + n, a.dtype, v);
  }
}

// ------------------------------------------------------------------ tiles
template <int S>
struct MfmaI8;
template <>
struct MfmaI8<16> {
  typedef int acc_t __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ acc_t run(v4i a, v4i b, acc_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};
template <>
struct MfmaI8<32> {
  typedef v16i acc_t;
  static __device__ __forceinline__ acc_t run(v4i a, v4i b, acc_t c) { return mfma_i8(a, b, c); }
};

// WM x WN waves, S x S MFMA blocks
template <int BM, int BN, int WM, int WN, int S, bool SPLIT>
__device__ __forceinline__ void linear_tile(const LinearArgs& a) {
  constexpr int WAVES = WM * WN, TM = BM / WM, TN = BN / WN, IM = TM / S, IN = TN / S;
  constexpr int CH = 64 / S;               // chunks of one MFMA (a lane's is L / S)
  constexpr int KK = 8 / CH;               // MFMAs of a step
  constexpr int PA = BM / 8, PB = BN / 8;  // loads (8 rows each) of a step
  constexpr int LA = (PA + WAVES - 1) / WAVES, LB = (PB + WAVES - 1) / WAVES;
  static_assert(TM % S == 0 && TN % S == 0 && BM % 8 == 0 && BN % 8 == 0, "whole MFMA blocks");
  using M = MfmaI8<S>;
  __shared__ __align__(16) int8_t lds0[(BM + BN) * LIN_KS], lds1[(BM + BN) * LIN_KS];

  const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the 8 XCDs in turn: give each XCD a run of neighbouring tiles (in groups of 8 tile rows, column by
  // column), so that its L2 serves the rows and columns that they share.
  const int total = a.tiles_m * a.tiles_n * a.splits;
  const int xcd = blockIdx.x & 7, q = total >> 3, rem = total & 7;
  int id = xcd * q + min(xcd, rem) + (blockIdx.x >> 3);
  const int split = id % a.splits;
  id /= a.splits;
  const int group = id / (8 * a.tiles_n), in_group = id - group * 8 * a.tiles_n;
  const int gm = min(8, a.tiles_m - group * 8);
  const int tn = in_group / gm, tm = group * 8 + in_group - tn * gm;
  const int m0 = tm * BM, n0 = tn * BN;
  const int steps = (a.k + LIN_KS - 1) / LIN_KS;
  const int s0 = split * a.per, s1 = min(steps, s0 + a.per);

  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.x + (int64_t)m0 * a.ldx), (short)0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.w + (int64_t)n0 * a.ldw), (short)0, 0x7fffffff, 0x00020000);
  const int chunk = (L & 7) ^ (L >> 3);  // (the row's low bits are L >> 3)
  int vx[LA], vw[LB];                    // this lane's byte offsets at K = 0
#pragma unroll
  for (int i = 0; i < LA; ++i)
    vx[i] = min((wave + i * WAVES) * 8 + (L >> 3), a.m - 1 - m0) * (int)a.ldx;
#pragma unroll
  for (int i = 0; i < LB; ++i)
    vw[i] = min((wave + i * WAVES) * 8 + (L >> 3), a.n - 1 - n0) * (int)a.ldw;
  const int last_chunk = (a.k - 1) & ~15;
  const int full = a.k / LIN_KS;  // steps whose 8 chunks all lie in the row
  auto issue = [&](int8_t* buf, int s) {
    const int koff = s < full ? chunk * 16 : min(s * LIN_KS + chunk * 16, last_chunk) - s * LIN_KS;
#pragma unroll
    for (int i = 0; i < LA; ++i)
      if (PA % WAVES == 0 || wave + i * WAVES < PA)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rx, (__attribute__((address_space(3))) void*)(buf + (wave + i * WAVES) * 1024), 16, vx[i] + koff,
            s * LIN_KS, 0, 0);
#pragma unroll
    for (int i = 0; i < LB; ++i)
      if (PB % WAVES == 0 || wave + i * WAVES < PB)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rw, (__attribute__((address_space(3))) void*)(buf + BM * LIN_KS + (wave + i * WAVES) * 1024), 16,
            vw[i] + koff, s * LIN_KS, 0, 0);
  };

  const int wm = wave % WM, wn = wave / WM, lr = L % S, lc = L / S;
  typename M::acc_t acc[IN][IM] = {};
  const int xa = (wm * TM + lr) * LIN_KS, wa = BM * LIN_KS + (wn * TN + lr) * LIN_KS, sw = lr & 7;
  auto compute = [&](const int8_t* buf, int s, bool tail) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int slot = ((kk * CH + lc) ^ sw) * 16;
      v4i fx[IM], fw[IN];
#pragma unroll
      for (int i = 0; i < IM; ++i) {
        fx[i] = *reinterpret_cast<const v4i*>(buf + xa + i * S * LIN_KS + slot);
        if (tail) fx[i] = lin_mask(fx[i], a.k - s * LIN_KS - (kk * CH + lc) * 16);
      }
#pragma unroll
      for (int i = 0; i < IN; ++i) fw[i] = *reinterpret_cast<const v4i*>(buf + wa + i * S * LIN_KS + slot);
#pragma unroll
      for (int i = 0; i < IN; ++i)
#pragma unroll
        for (int j = 0; j < IM; ++j) acc[i][j] = M::run(fw[i], fx[j], acc[i][j]);
    }
  };
  auto wait = [&]() {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
  issue(lds0, s0);
  int s = s0;
  const int whole = min(s1, full);
  // two steps per turn, so that each buffer is an object of its own to the compiler
  while (s + 1 < whole) {
    wait();  // step s has landed; every wave is done with the other buffer
    issue(lds1, s + 1);
    compute(lds0, s, false);
    wait();
    if (s + 2 < s1) issue(lds0, s + 2);
    compute(lds1, s + 1, false);
    s += 2;
  }
  if (s < whole) {
    wait();
    if (s + 1 < s1) issue(lds1, s + 1);
    compute(lds0, s, false);
    if (s + 1 < s1) {
      wait();
      compute(lds1, s + 1, true);
    }
  } else if (s < s1) {
    wait();
    compute(lds0, s, true);
  }

  // a lane's column of block (i, j) is m; its rows are n in runs of four
#pragma unroll
  for (int j = 0; j < IM; ++j) {
    const int m = m0 + wm * TM + j * S + lr;
    if (m >= a.m) continue;
    const float xs = SPLIT ? 0.0f : a.xs[m];
#pragma unroll
    for (int i = 0; i < IN; ++i)
#pragma unroll
      for (int g = 0; g < S / (64 / S * 4); ++g) {
        const int n = n0 + wn * TN + i * S + g * (64 / S * 4) + 4 * lc;
        const int v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        if constexpr (SPLIT) {
          int32_t* p = a.part + ((int64_t)split * a.m + m) * a.n + n;
          if (n + 4 <= a.n) __builtin_memcpy(p, v, 16);
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < a.n) p[e] = v[e];
        } else {
          if (n < a.n) lin_out4(a, m, n, xs, v);
        }
      }
  }
}

template <int BM, int BN, int WM, int WN, int S, bool SPLIT>
__global__ __launch_bounds__(WM * WN * 64) void tile_kernel(LinearArgs a) {
  linear_tile<BM, BN, WM, WN, S, SPLIT>(a);
}

// out from the splits' sums, four outputs per thread
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a) {
  const int nq = (a.n + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.m * nq) return;
  const int m = (int)(i / nq), n = (int)(i - (int64_t)m * nq) * 4;
  int v[4] = {};
  for (int s = 0; s < a.splits; ++s) {
    const int32_t* p = a.part + ((int64_t)s * a.m + m) * a.n + n;
    int t[4] = {};
    if (n + 4 <= a.n) __builtin_memcpy(t, p, 16);
    else
      for (int e = 0; e < 4; ++e)
        if (n + e < a.n) t[e] = p[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += t[e];
  }
  lin_out4(a, m, n, a.xs[m], v);
}

// ------------------------------------------------------------------ launches
// How one product is cut: `kind` 0 the dot kernel, otherwise a tile form; splits of `per` steps each.
struct LinearPlan {
  int kind, bm, bn, splits, per;
};

inline LinearPlan linear_plan(int m, int n, int k, int cus) {
  LinearPlan p{};
  const int steps = (k + LIN_KS - 1) / LIN_KS;
  p.splits = 1;
  p.per = steps;
  if (m <= 8) return p;
  if (m <= 16) p.kind = 1, p.bm = 16, p.bn = 64;
  else if (m <= 32) p.kind = 2, p.bm = 32, p.bn = 64;
  else if (m <= 64) p.kind = 3, p.bm = 64, p.bn = 64;
  else if ((int64_t)((m + 255) / 256) * ((n + 255) / 256) >= cus) p.kind = 5, p.bm = 256, p.bn = 256;
  else p.kind = 4, p.bm = 128, p.bn = 128;
  const int64_t tiles = (int64_t)((m + p.bm - 1) / p.bm) * ((n + p.bn - 1) / p.bn);
  if (p.kind < 5 && tiles < 2 * cus) {
    const int want = (int)std::min<int64_t>((2 * cus + tiles - 1) / tiles, std::max(1, steps / 8));
    p.per = (steps + want - 1) / want;
    p.splits = (steps + p.per - 1) / p.per;
  }
  return p;
}

template <int BM, int BN, int WM, int WN, int S>
inline void launch_tile(const LinearArgs& a, hipStream_t s) {
  const dim3 grid(a.tiles_m * a.tiles_n * a.splits), block(WM * WN * 64);
  if (a.splits > 1) tile_kernel<BM, BN, WM, WN, S, true><<<grid, block, 0, s>>>(a);
  else tile_kernel<BM, BN, WM, WN, S, false><<<grid, block, 0, s>>>(a);
}

template <int MR>
inline void launch_dot(const LinearArgs& a, hipStream_t s) {
  constexpr int NR = 2, WAVES = 4, U = 4;
  dot_kernel<MR, NR, WAVES, U><<<dim3((a.n + NR * 8 - 1) / (NR * 8)), dim3(WAVES * 64), 0, s>>>(a);
}

inline void launch_linear(LinearArgs a, const LinearPlan& p, hipStream_t s) {
  if (p.kind == 0) {
    if (a.m == 1) launch_dot<1>(a, s);
    else if (a.m == 2) launch_dot<2>(a, s);
    else if (a.m <= 4) launch_dot<4>(a, s);
    else launch_dot<8>(a, s);
    return;
  }
  a.tiles_m = (a.m + p.bm - 1) / p.bm;
  a.tiles_n = (a.n + p.bn - 1) / p.bn;
  a.splits = p.splits;
  a.per = p.per;
  switch (p.kind) {
    case 1: launch_tile<16, 64, 1, 4, 16>(a, s); break;
    case 2: launch_tile<32, 64, 1, 4, 16>(a, s); break;
    case 3: launch_tile<64, 64, 2, 2, 32>(a, s); break;
    case 4: launch_tile<128, 128, 2, 2, 32>(a, s); break;
    default: launch_tile<256, 256, 2, 4, 32>(a, s); break;
  }
  if (p.splits > 1) {
    const int64_t quads = (int64_t)a.m * ((a.n + 3) / 4);
    linear_join_kernel<<<dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s>>>(a);
  }
}

}  // namespace tri
