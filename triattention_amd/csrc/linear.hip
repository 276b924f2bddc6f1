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

template <typename T>
__device__ __forceinline__ float lin_f32(T v) { return (float)v; }
template <>
__device__ __forceinline__ float lin_f32<__bf16>(__bf16 v) { return bf16f(__builtin_bit_cast(uint16_t, v)); }

// `run` with a value of the output's type
template <typename F>
__device__ __forceinline__ void lin_typed(int dtype, F run) {
  if (dtype == BF16) run(__bf16{});
  else if (dtype == F32) run(float{});
  else run(_Float16{});
}

// p[base + off], the base uniform and the lane's offset 32 bits of bytes: addressed without a 64-bit sum per lane
template <typename T>
__device__ __forceinline__ T* lin_at(T* p, int64_t base, uint32_t off) {
  return reinterpret_cast<T*>(reinterpret_cast<uint64_t>(p + base) + off * (uint32_t)sizeof(T));
}
// Scales and biases of channels n .. n+C-1, n = nu + nl with nu uniform; WHOLE: all of them exist.  The vectors may be
// unaligned (odd row lengths).
template <typename T, bool WHOLE, int C>
__device__ __forceinline__ void lin_channels(const LinearArgs& a, int nu, int nl, float (&ws)[C], float (&bias)[C]) {
  const int n = nu + nl;
  if constexpr (WHOLE) __builtin_memcpy(ws, lin_at(a.ws, nu, nl), sizeof(ws));
  else
#pragma unroll
    for (int e = 0; e < C; ++e) ws[e] = n + e < a.n ? a.ws[n + e] : 0.0f;
  T t[C] = {};
  if (a.bias) {
    const T* b = static_cast<const T*>(a.bias);
    if constexpr (WHOLE) __builtin_memcpy(t, lin_at(b, nu, nl), sizeof(t));
    else
#pragma unroll
      for (int e = 0; e < C; ++e) t[e] = n + e < a.n ? b[n + e] : T{};
  }
#pragma unroll
  for (int e = 0; e < C; ++e) bias[e] = lin_f32(t[e]);
}
// The outputs of those channels of row m = mu + ml (mu uniform, ml < 32) from their sums.
template <typename T, bool WHOLE, int C>
__device__ __forceinline__ void lin_out(const LinearArgs& a, int mu, int ml, int nu, int nl, const float (&ws)[C],
                                        const float (&bias)[C], const int (&sums)[C]) {
  const int n = nu + nl;
  const float xs = a.xs[mu + ml];
  T* o = lin_at(static_cast<T*>(a.out), mu * a.ldo + nu, ml * (uint32_t)a.ldo + nl);
  float v[C];
#pragma unroll
  for (int e = 0; e < C; ++e) v[e] = (float)sums[e] * (xs * ws[e]) + bias[e];
  T t[C];
  if (a.residual) {
    const T* r = static_cast<const T*>(a.residual) + (mu + ml) * a.ldr + n;
    if constexpr (WHOLE) __builtin_memcpy(t, r, sizeof(t));
#pragma unroll
    for (int e = 0; e < C; ++e) {
      if constexpr (!WHOLE) t[e] = n + e < a.n ? r[e] : T{};
      v[e] += lin_f32(t[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < C; ++e) t[e] = (T)v[e];
  if constexpr (WHOLE) __builtin_memcpy(o, t, sizeof(t));
  else
#pragma unroll
    for (int e = 0; e < C; ++e)
      if (n + e < a.n) o[e] = t[e];
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
  const int full = a.k / LIN_KS;
  int s = wave;
  for (; s + (U - 1) * WAVES < full; s += U * WAVES) {
    v4i w[U][NR], x[U][MR];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kc = (s + u * WAVES) * LIN_KS + c * 16;
#pragma unroll
      for (int i = 0; i < NR; ++i) w[u][i] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(wrow[i] + kc));
#pragma unroll
      for (int m = 0; m < MR; ++m) x[u][m] = *reinterpret_cast<const v4i*>(xrow[m] + kc);
    }
    __builtin_amdgcn_sched_barrier(0);  // (every load of the turn in flight before the first is used)
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[m][i] = __builtin_amdgcn_sdot4(w[u][i][j], x[u][m][j], acc[m][i], false);
  }
  if (s < steps) {  // what is left: at most U steps, some past the row's end (masked)
    v4i w[U][NR], x[U][MR];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kc = min((s + u * WAVES) * LIN_KS + c * 16, last_chunk);
#pragma unroll
      for (int i = 0; i < NR; ++i) w[u][i] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(wrow[i] + kc));
#pragma unroll
      for (int m = 0; m < MR; ++m) x[u][m] = *reinterpret_cast<const v4i*>(xrow[m] + kc);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const v4i xm = lin_mask(x[u][m], a.k - (s + u * WAVES) * LIN_KS - c * 16);
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[m][i] = __builtin_amdgcn_sdot4(w[u][i][j], xm[j], acc[m][i], false);
      }
  }
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
    lin_typed(a.dtype, [&](auto type) {
      using T = decltype(type);
      float v = (float)sum * (a.xs[m] * a.ws[n]);
      if (a.bias) v += lin_f32(static_cast<const T*>(a.bias)[n]);
      if (a.residual) v += lin_f32(static_cast<const T*>(a.residual)[m * a.ldr + n]);
      static_cast<T*>(a.out)[m * a.ldo + n] = (T)v;
    });
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

// Waits for all but the last N loads of this wave and for its LDS reads, then for the workgroup.
template <int N>
__device__ __forceinline__ void lin_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A buffer descriptor of the rows from `p` on (32-bit byte offsets, uniform).
__device__ __forceinline__ v4i lin_rsrc(const void* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  return v4i{__builtin_amdgcn_readfirstlane((int)u), __builtin_amdgcn_readfirstlane((int)(u >> 32) & 0xffff),
             0x7fffffff, 0x00020000};
}
// 16 bytes a lane from byte `off` + `soff` of the rows to LDS byte `dst` + 16 * lane, awaited by lin_wait alone.  (The
// builtin would make the compiler wait for every load in flight before it reads LDS again.)  The five wait states cover
// a scalar operand that a vector instruction (readfirstlane) has just written: the compiler does not look into the asm
// for that hazard.  Nothing else in these kernels uses m0.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lin_lds_load(v4i rsrc, int off, int soff, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(
                   __builtin_amdgcn_readfirstlane(dst)),
               "v"(off), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(soff))
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lin_lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// WM x WN waves, S x S MFMA blocks, ST buffers of 128 bytes of K.  Workgroup w takes tiles w, w + gridDim.x, ...: with
// fewer workgroups than tiles, the next tile's first loads are in flight while this one's outputs are written.
template <int BM, int BN, int WM, int WN, int S, int ST, bool SPLIT>
__device__ __forceinline__ void linear_tile(const LinearArgs& a) {
  constexpr int WAVES = WM * WN, TM = BM / WM, TN = BN / WN, IM = TM / S, IN = TN / S;
  constexpr int CH = 64 / S;               // chunks of one MFMA (a lane's is L / S)
  constexpr int KK = 8 / CH;               // MFMAs of a step
  constexpr int PA = BM / 8, PB = BN / 8;  // loads (8 rows each) of a step
  constexpr int LA = (PA + WAVES - 1) / WAVES, LB = (PB + WAVES - 1) / WAVES, LPS = LA + LB;
  constexpr int RUN = 64 / S * 4;          // a lane's rows of a block come in runs of four, RUN apart
  constexpr bool ROWS = !SPLIT && S == 32;  // outputs pass through LDS
  static_assert(TM % S == 0 && TN % S == 0 && BM % 8 == 0 && BN % 8 == 0, "whole MFMA blocks");
  static_assert(ST >= 2 && ST <= 4 && KK % 2 == 0, "buffers");
  using M = MfmaI8<S>;
  constexpr int BUF = (BM + BN) * LIN_KS;
  __shared__ __align__(16) int8_t bufs[ST][BUF];
  __shared__ __align__(16) int8_t rows[ROWS ? WAVES : 1][ROWS ? 4096 : 16];

  const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM, lr = L % S, lc = L / S;
  const int total = a.tiles_m * a.tiles_n * a.splits, steps = (a.k + LIN_KS - 1) / LIN_KS;
  const int last_chunk = (a.k - 1) & ~15;
  const int full = a.k / LIN_KS;         // steps whose 8 chunks all lie in the row
  const int chunk = (L & 7) ^ (L >> 3);  // (the row's low bits are L >> 3)

  // The tile: its place, its steps, and this wave's loads: the 8-row pieces and this lane's byte offsets at K = 0 (a wave
  // without a piece of its own repeats the last one, so that every wave counts the same loads).
  int m0, n0, split, s0, whole, tail;
  v4i rx, rw;
  int vx[LA], vw[LB];
  auto locate = [&](int t) __attribute__((always_inline)) {
    // Workgroups go to the 8 XCDs in turn: give each XCD a run of neighbouring tiles (in groups of 8 tile rows, column
    // by column), so that its L2 serves the rows and columns that they share.
    const int xcd = t & 7, q = total >> 3, rem = total & 7;
    int id = xcd * q + min(xcd, rem) + (t >> 3);
    split = __builtin_amdgcn_readfirstlane(id % a.splits);
    id /= a.splits;
    const int group = id / (8 * a.tiles_n), in_group = id - group * 8 * a.tiles_n;
    const int gm = min(8, a.tiles_m - group * 8);
    const int tn = in_group / gm, tm = group * 8 + in_group - tn * gm;
    // (divisions run in vector registers: the results are uniform)
    m0 = __builtin_amdgcn_readfirstlane(tm * BM);
    n0 = __builtin_amdgcn_readfirstlane(tn * BN);
    s0 = split * a.per;
    const int s1 = min(steps, s0 + a.per);
    whole = min(s1, full);
    tail = s1 > full;
    rx = lin_rsrc(a.x + (int64_t)m0 * a.ldx);
    rw = lin_rsrc(a.w + (int64_t)n0 * a.ldw);
#pragma unroll
    for (int i = 0; i < LA; ++i)
      vx[i] = min(min(wave + i * WAVES, PA - 1) * 8 + (L >> 3), a.m - 1 - m0) * (int)a.ldx;
#pragma unroll
    for (int i = 0; i < LB; ++i)
      vw[i] = min(min(wave + i * WAVES, PB - 1) * 8 + (L >> 3), a.n - 1 - n0) * (int)a.ldw;
  };
  auto issue = [&](int8_t* buf, int s) __attribute__((always_inline)) {
    const int koff = s < full ? chunk * 16 : min(s * LIN_KS + chunk * 16, last_chunk) - s * LIN_KS;
    const uint32_t dst = lin_lds_addr(buf);
#pragma unroll
    for (int i = 0; i < LA; ++i)
      lin_lds_load(rx, vx[i] + koff, s * LIN_KS, dst + min(wave + i * WAVES, PA - 1) * 1024);
#pragma unroll
    for (int i = 0; i < LB; ++i)
      lin_lds_load(rw, vw[i] + koff, s * LIN_KS, dst + BM * LIN_KS + min(wave + i * WAVES, PB - 1) * 1024);
  };
  auto start = [&]() __attribute__((always_inline)) {  // the first ST steps' loads; the step that ends inside its 128 bytes first
#pragma unroll
    for (int u = 0; u < ST - 1; ++u)
      if (s0 + u < whole) issue(bufs[u], s0 + u);
    if (tail) issue(bufs[ST - 1], full);
    else if (s0 + ST - 1 < whole) issue(bufs[ST - 1], s0 + ST - 1);
  };

  typename M::acc_t acc[IN][IM];
  const int xa = (wm * TM + lr) * LIN_KS, wa = BM * LIN_KS + (wn * TN + lr) * LIN_KS, sw = lr & 7;
  v4i fx[2][IM], fw[2][IN];
  auto read = [&](const int8_t* buf, int kk) __attribute__((always_inline)) {
    const int slot = ((kk * CH + lc) ^ sw) * 16;
#pragma unroll
    for (int i = 0; i < IM; ++i) fx[kk & 1][i] = *reinterpret_cast<const v4i*>(buf + xa + i * S * LIN_KS + slot);
#pragma unroll
    for (int i = 0; i < IN; ++i) fw[kk & 1][i] = *reinterpret_cast<const v4i*>(buf + wa + i * S * LIN_KS + slot);
  };
  auto multiply = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < IN; ++i)
#pragma unroll
      for (int j = 0; j < IM; ++j) acc[i][j] = M::run(fw[kk & 1][i], fx[kk & 1][j], acc[i][j]);
  };

  int t = blockIdx.x;
  locate(t);
  start();
  for (bool first = true;; first = false) {
#pragma unroll
    for (int i = 0; i < IN; ++i)
#pragma unroll
      for (int j = 0; j < IM; ++j) acc[i][j] = typename M::acc_t{};
    if (tail) {
      lin_wait<0>();
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        read(bufs[ST - 1], kk);
#pragma unroll
        for (int i = 0; i < IM; ++i)
          fx[kk & 1][i] = lin_mask(fx[kk & 1][i], a.k - full * LIN_KS - (kk * CH + lc) * 16);
        multiply(kk);
      }
      lin_wait<0>();
      if (s0 + ST - 1 < whole) issue(bufs[ST - 1], s0 + ST - 1);
    } else if (first && s0 + ST - 1 < whole) {
      lin_wait<(ST - 1) * LPS>();
    } else {
      lin_wait<0>();  // (after a first tile the counter holds its stores too)
    }
    // Step s: the operands of one MFMA are read while the one before runs.  Before the last, every operand of the step
    // is in registers: the workgroup meets, its buffer takes step s + ST, and the next step's first operands are read.
    if (s0 < whole) read(bufs[0], 0);
    for (int s = s0; s < whole; s += ST) {
#pragma unroll
      for (int u = 0; u < ST; ++u) {
        if (s + u < whole) {
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            if (kk + 1 < KK) {
              read(bufs[u], kk + 1);
            } else if (s + u + 1 < whole) {
              if (s + u + ST - 1 < whole) lin_wait<(ST - 2) * LPS>();
              else lin_wait<0>();
              if (s + u + ST < whole) issue(bufs[u], s + u + ST);
              read(bufs[(u + 1) % ST], 0);
            }
            __builtin_amdgcn_sched_barrier(0);  // (the compiler would read each operand right before its use)
            multiply(kk);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }

    // a lane's column of block (i, j) is m; its rows are n
    const int tm0 = m0 + wm * TM, tn0 = n0 + wn * TN, tsplit = split;
    const bool whole_n = n0 + BN <= a.n;
    t += gridDim.x;
    if (t < total) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // every wave has read its last operands
      locate(t);
      start();
    }
    if constexpr (SPLIT) {
#pragma unroll
      for (int j = 0; j < IM; ++j) {
        const int m = tm0 + lr + j * S;
        if (m < a.m) {
          int32_t* p = a.part + ((int64_t)tsplit * a.m + m) * a.n;
#pragma unroll
          for (int i = 0; i < IN; ++i)
#pragma unroll
            for (int g = 0; g < S / RUN; ++g) {
              const int n = tn0 + i * S + g * RUN + 4 * lc;
              const int v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
              if (n + 4 <= a.n) __builtin_memcpy(p + n, v, 16);
              else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (n + e < a.n) p[n + e] = v[e];
            }
        }
      }
    } else {
      auto write = [&](auto type, auto whole_tile) __attribute__((always_inline)) {
        using T = decltype(type);
        constexpr bool WHOLE = decltype(whole_tile)::value;
        if constexpr (ROWS) {
          // A block's sums pass through the wave's own 4 KiB of LDS, row m at 128 bytes, 16-byte piece p at slot
          // p ^ (m & 7): four lanes then hold a row's 32 channels, eight each, with one set of scales for all rows.
          int8_t* own = rows[wave];
          const int row = L >> 2, c8 = (L & 3) * 8;
#pragma unroll
          for (int i = 0; i < IN; ++i) {
            float ws[8], bias[8];
            lin_channels<T, WHOLE>(a, tn0 + i * S, c8, ws, bias);
#pragma unroll
            for (int j = 0; j < IM; ++j) {
#pragma unroll
              for (int g = 0; g < S / RUN; ++g)
                *reinterpret_cast<v4i*>(own + lr * 128 + ((2 * g + lc) ^ (lr & 7)) * 16) =
                    v4i{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int mu = tm0 + j * S + h * 16, nu = tn0 + i * S;
                const int8_t* src = own + (h * 16 + row) * 128;
                v4i v[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  v[e] = *reinterpret_cast<const v4i*>(src + ((2 * (L & 3) + e) ^ (row & 7)) * 16);
                if (mu + row < a.m) {
                  const int sums[8] = {v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]};
                  lin_out<T, WHOLE>(a, mu, row, nu, c8, ws, bias, sums);
                }
              }
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < IN; ++i)
#pragma unroll
            for (int g = 0; g < S / RUN; ++g) {
              const int nu = tn0 + i * S + g * RUN;
              float ws[4], bias[4];
              lin_channels<T, WHOLE>(a, nu, 4 * lc, ws, bias);
#pragma unroll
              for (int j = 0; j < IM; ++j) {
                const int sums[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                if (tm0 + j * S + lr < a.m) lin_out<T, WHOLE>(a, tm0 + j * S, lr, nu, 4 * lc, ws, bias, sums);
              }
            }
        }
      };
      lin_typed(a.dtype, [&](auto type) __attribute__((always_inline)) {
        if (whole_n) write(type, std::true_type{});
        else write(type, std::false_type{});
      });
    }
    if (t >= total) return;
  }
}

template <int BM, int BN, int WM, int WN, int S, int ST, bool SPLIT>
__global__ __launch_bounds__(WM * WN * 64) void tile_kernel(LinearArgs a) {
  linear_tile<BM, BN, WM, WN, S, ST, SPLIT>(a);
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
  lin_typed(a.dtype, [&](auto type) {
    using T = decltype(type);
    float ws[4], bias[4];
    if (n + 4 <= a.n) {
      lin_channels<T, true>(a, 0, n, ws, bias);
      lin_out<T, true>(a, m, 0, 0, n, ws, bias, v);
    } else {
      lin_channels<T, false>(a, 0, n, ws, bias);
      lin_out<T, false>(a, m, 0, 0, n, ws, bias, v);
    }
  });
}

// ------------------------------------------------------------------ launches
// How one product is cut: `kind` 0 the dot kernel, otherwise a tile form; splits of `per` steps each.
struct LinearPlan {
  int kind, bm, bn, splits, per;
  int groups;  // workgroups, at most one a tile
};

// The tile forms.  step: us that a step takes a workgroup alone on its CU (the latency of its loads over its buffers);
// resident: workgroups of the form that a CU holds; fixed: us before the first and after the last step.
struct LinearForm {
  int bm, bn, resident;
  double step, fixed;
};
constexpr LinearForm LIN_FORMS[] = {
    {16, 64, 3, 0.13, 0.7},   {32, 64, 3, 0.20, 1.3},   {64, 64, 2, 0.32, 1.4},
    {128, 128, 2, 0.70, 3.4},  // two buffers, two workgroups a CU
    {128, 128, 1, 0.70, 3.0},  // four buffers: for fewer tiles than CUs
    {256, 256, 1, 0.90, 7.4},
};

// The form and the split that this model of their time holds fastest: rounds of resident workgroups, each step bound by
// its own latency, by the bytes that a CU takes from its L2 (63 GB/s) or by the matrix cores (12.7 Top/s a CU); never
// below the stream of both operands (5.75 TB/s); a split adds its launch and its partials' way through memory.  Fitted
// to 2,500 timings of 121 shapes (5 to 4,096 rows, 640 to 37,888 channels, K 1,000 to 18,944): its choice takes 0.5% more
// than the fastest of all forms and splits on the mean, 11% at most.
inline LinearPlan linear_plan(int m, int n, int k, int cus) {
  const int steps = (k + LIN_KS - 1) / LIN_KS;
  LinearPlan best{};
  best.splits = 1;
  best.per = steps;
  // Up to 4 rows v_dot4 keeps up with the stream (K 18,944 x 3,584 channels: 11.8 / 12.5 / 15.5 us for 1 / 2 / 4 rows, 23
  // for 8; the 16-row tile 15-16 us at any count).
  if (m <= 4) return best;
  double least = 1e300;
  const double stream = ((double)n * k + (double)m * k) / 5.75e6;
  for (int f = 0; f < 6; ++f) {
    const LinearForm& form = LIN_FORMS[f];
    const int64_t tiles = (int64_t)((m + form.bm - 1) / form.bm) * ((n + form.bn - 1) / form.bn);
    const int64_t slots = (int64_t)cus * form.resident;
    const double bytes = (form.bm + form.bn) * LIN_KS / 63e3, ops = 2.0 * form.bm * form.bn * LIN_KS / 12.7e6;
    for (int want = 1; want <= 16 && (want == 1 || (steps >= 4 * want && tiles * want <= 5 * (int64_t)cus)); ++want) {
      const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
      const int64_t work = tiles * splits, rounds = work / slots;
      const int left = (int)((work - rounds * slots + cus - 1) / cus);
      double t = rounds * (per * std::max(form.step, form.resident * std::max(bytes, ops)) + form.fixed);
      if (left) t += per * std::max(form.step, left * std::max(bytes, ops)) + form.fixed;
      t = std::max(t, stream);
      if (splits > 1) t += 2.2 + 0.17 * splits + 8.0 * splits * m * n / 3.4e6;
      if (t < least) {
        least = t;
        best = {f + 1, form.bm, form.bn, splits, per, INT32_MAX};
      }
    }
  }
  // (the largest form's workgroups take tile after tile; a multiple of the XCDs keeps a workgroup's tiles on its XCD)
  if (best.kind == 6) best.groups = std::max(8, cus & ~7);
  return best;
}

template <int BM, int BN, int WM, int WN, int S, int ST>
inline void launch_tile(const LinearArgs& a, int groups, hipStream_t s) {
  const dim3 grid(std::min(groups, a.tiles_m * a.tiles_n * a.splits)), block(WM * WN * 64);
  if (a.splits > 1) tile_kernel<BM, BN, WM, WN, S, ST, true><<<grid, block, 0, s>>>(a);
  else tile_kernel<BM, BN, WM, WN, S, ST, false><<<grid, block, 0, s>>>(a);
}

template <int MR, int U>
inline void launch_dot(const LinearArgs& a, hipStream_t s) {
  constexpr int NR = 2, WAVES = 8;
  dot_kernel<MR, NR, WAVES, U><<<dim3((a.n + NR * 8 - 1) / (NR * 8)), dim3(WAVES * 64), 0, s>>>(a);
}

inline void launch_linear(LinearArgs a, const LinearPlan& p, hipStream_t s) {
  if (p.kind == 0) {
    if (a.m == 1) launch_dot<1, 4>(a, s);
    else if (a.m == 2) launch_dot<2, 4>(a, s);
    else launch_dot<4, 2>(a, s);
    return;
  }
  a.tiles_m = (a.m + p.bm - 1) / p.bm;
  a.tiles_n = (a.n + p.bn - 1) / p.bn;
  a.splits = p.splits;
  a.per = p.per;
  switch (p.kind) {
    case 1: launch_tile<16, 64, 1, 4, 16, 4>(a, p.groups, s); break;
    case 2: launch_tile<32, 64, 1, 4, 16, 4>(a, p.groups, s); break;
    case 3: launch_tile<64, 64, 2, 2, 32, 3>(a, p.groups, s); break;
    case 4: launch_tile<128, 128, 2, 2, 32, 2>(a, p.groups, s); break;
    case 5: launch_tile<128, 128, 2, 2, 32, 4>(a, p.groups, s); break;
    default: launch_tile<256, 256, 2, 4, 32, 2>(a, p.groups, s); break;
  }
  if (p.splits > 1) {
    const int64_t quads = (int64_t)a.m * ((a.n + 3) / 4);
    linear_join_kernel<<<dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s>>>(a);
  }
}

}  // namespace tri
