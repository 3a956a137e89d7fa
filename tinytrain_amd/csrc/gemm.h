// Matrix products of bf16 operands with fp32 sums, gfx950: out[m][n] = sum_k X(m, k) W(n, k) as tiles
// of TM x TN, for the kernels whose epilogues differ (swiglu.hip, linear_mx.hip).
//
// An operand is read as it lies in memory: rows along k (row m holds its k's), or rows along the
// other index (row k holds its m's; TR), so no product needs a transposed copy.  Tiles go straight
// to LDS (16 bytes a lane, S stages: the next ones' loads run during this stage's products)
// and come back as operand registers of v_mfma_f32_32x32x16_bf16, TR ones through
// ds_read_b64_tr_b16.  LDS rows are swizzled in 16-byte chunks so that both reads are free of
// conflicts (fa_common.h: 16 rows at one chunk; 4 rows x 4 chunks).
//
// W is the instruction's first operand: a lane then holds, of column m = lane % 32 of a 32 x 32
// block, n = 8a + 4 (lane / 32) + e in register 4a + e, so runs of n, which lie together in memory.
//
// Edges: rows past an operand's end are past its buffer and load as zeros; k past the end of rows
// along k would be the next row's values, so those lanes are pointed past the buffer in the last
// stage.  Columns past the end of TR rows are other elements of the matrix, and give results that
// are not stored.  (Zeros, not multiplications by zero: a NaN or infinity stays in its own row.)
#pragma once

#include <algorithm>

#include "fa_bwd.h"  // allow_lds
#include "fa_common.h"
#include "product_cut.h"

namespace ttfa {

// D[i][j] of 16 x 16 in lane j + 16 (i / 4), register i % 4; operands: row i (or j) in lanes i + 16 (k / 8).
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The LDS reads of this wave, and all but its last N vector memory accesses, done; then the workgroup
// meets.  Memory accesses stay on their side of it.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
  static_assert(N < 64, "six bits");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 16 bytes to byte_off of a buffer; past its end they are dropped (the instruction is issued all the same,
// so what is counted by vmcnt does not depend on it).
__device__ __forceinline__ void buf_store16(__amdgpu_buffer_rsrc_t r, uint32_t byte_off, u32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(v, r, byte_off, 0, 0);
}

__device__ __forceinline__ void buf_store8(__amdgpu_buffer_rsrc_t r, uint32_t byte_off, u32x2 v) {
  __builtin_amdgcn_raw_buffer_store_b64(v, r, byte_off, 0, 0);
}

constexpr uint32_t kPastEnd = 0x80000000u;  // an offset that no tile's buffer covers

// One operand's tile of T rows (of the m or n index) x BK, loaded by NT threads, stage after stage along k.
template <int T, int BK, bool TR, int NT>
struct TileLoad {
  static constexpr int LOADS = T * BK * 2 / 16 / NT;
  static constexpr int CPR = TR ? T / 8 : BK / 8;  // 16-byte chunks of an LDS row
  static constexpr int BYTES = T * BK * 2;
  static constexpr int ROWS = NT / CPR;  // of one load of all threads
  static_assert(T * BK * 2 % (16 * NT) == 0 && (!TR || T >= 128), "tile");
  static_assert(NT % CPR == 0 && ROWS % 16 == 0, "a thread's loads have one swizzle");
  const char *base;  // of the next stage
  uint32_t bytes;    // that the tile's rows have from there on
  int64_t step;      // bytes to the stage after it
  uint32_t off;   // this thread's first load in the stage, the others `rows` bytes further on each
  uint32_t rows;

  static __device__ __forceinline__ int swizzle(int row) {
    return TR ? (row & 3) << 2 : (row / (16 / CPR)) & (CPR - 1);
  }

  // The matrix at p, rows of ld elements: tile from row (TR: column) r0 of R on.
  __device__ __forceinline__ void init(const bf16 *p, int64_t ld, int64_t r0, int64_t R) {
    start(p, ld, r0, R);
    step = TR ? ld * (BK * 2) : BK * 2;
    const int row = (int)threadIdx.x / CPR;
    off = (uint32_t)(row * ld * 2) + (((int)threadIdx.x % CPR) ^ swizzle(row)) * 16;
    rows = (uint32_t)(ROWS * ld * 2);
  }
  // The same tile of another matrix of the same shape (k from 0 again).
  __device__ __forceinline__ void start(const bf16 *p, int64_t ld, int64_t r0, int64_t R) {
    base = reinterpret_cast<const char *>(p + (TR ? r0 : r0 * ld));
    const int64_t n = R - r0 < T ? R - r0 : T;
    bytes = n <= 0 ? 0u : (uint32_t)((TR ? BK * ld - r0 : n * ld) * 2);
  }
  // Past the next n stages.
  __device__ __forceinline__ void skip(int n) {
    base += step * n;
    if (!TR) bytes -= (uint32_t)(BK * 2) * n;
  }
  // A stage of `left` < BK k's, the last one: what lies past them loads as zeros.
  __device__ __forceinline__ void shorten(int64_t ld, int left) {
    if constexpr (TR) {
      bytes -= (uint32_t)((BK - left) * ld * 2);
    } else {
      if (8 * (((int)threadIdx.x % CPR) ^ swizzle((int)threadIdx.x / CPR)) >= left) off = kPastEnd;
    }
  }
  // The stage, of the matrix that lies `beside` bytes further on.
  __device__ __forceinline__ void load_beside(int64_t beside, char *lds) const {
    char *dst = lds + wave_id() * 1024;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base + beside, bytes);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) buf_load16_lds(r, off + j * rows, dst + j * NT * 16);
  }
  __device__ __forceinline__ void load(char *lds) {
    load_beside(0, lds);
    base += step;
    if (!TR) bytes -= (uint32_t)(BK * 2);
  }
};

// Operand registers from such a tile: NB blocks of 32 of its rows, from row0 on every STRIDE rows
// (TR: row0 a multiple of 32 NB), k 16 s .. 16 s + 15.
template <int T, int BK, bool TR, int STRIDE = 32>
struct TileRead {
  static_assert(!TR || STRIDE == 32, "blocks of a TR tile lie together");
  static constexpr int CPR = TR ? T / 8 : BK / 8;
  static constexpr int STEPS = BK / 16;
  int at[TR ? 1 : STEPS];  // this lane's byte offsets in block 0, by s (TR: for s = 0)

  __device__ __forceinline__ void init(int row0) {
    const int lane = threadIdx.x & 63;
    if constexpr (TR) {
      const int k = 8 * (lane >> 5) + ((lane >> 2) & 3);
      const int col = row0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      at[0] = k * (T * 2) + (((col >> 3) ^ ((k & 3) << 2)) << 4) + (col & 7) * 2;
    } else {
      const int row = row0 + (lane & 31);
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        at[s] = row * (BK * 2) + (((2 * s + (lane >> 5)) ^ ((row / (16 / CPR)) & (CPR - 1))) << 4);
    }
  }

  __device__ __forceinline__ bf16x8 read(const char *__restrict__ lds, int b, int s) const {
    if constexpr (TR) {
      // Four chunks to a block: the swizzle XORs the block's index, which b does too.
      const bf16 *p = reinterpret_cast<const bf16 *>(lds + (at[0] ^ (b << 6)) + s * (16 * T * 2));
      const bf16x4 lo = lds_read_tr(p), hi = lds_read_tr(p + 4 * T);
      return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
      return *reinterpret_cast<const bf16x8 *>(lds + at[s] + b * (STRIDE * BK * 2));
    }
  }
};

// A 32 x 32 result block rounded to bf16, as two sets of 16-byte pieces of its rows: lane l holds, of set
// q, n = 8 piece_of(l) .. + 7 of column m = 16 q + l % 16, so that a store writes 64 bytes of each of 16
// rows.
__device__ __forceinline__ int piece_of(int lane) { return 2 * ((lane >> 4) & 1) + (lane >> 5); }

__device__ __forceinline__ void swap_rows(u32x4 &a, u32x4 &b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto x = __builtin_amdgcn_permlane16_swap(a[i], b[i], false, false);
    a[i] = x[0];
    b[i] = x[1];
  }
}

// From the block's registers in pairs: w[k] holds elements 2k and 2k + 1.
__device__ __forceinline__ void block_rows(const uint32_t (&w)[8], u32x4 (&set)[2]) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const auto x = __builtin_amdgcn_permlane32_swap(w[4 * p], w[4 * p + 2], false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(w[4 * p + 1], w[4 * p + 3], false, false);
    set[p] = u32x4{x[0], y[0], x[1], y[1]};
  }
  swap_rows(set[0], set[1]);
}

__device__ __forceinline__ void block_rows(const f32x16 &v, u32x4 (&set)[2]) {
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2 * k], v[2 * k + 1]}), bf16x2));
  block_rows(w, set);
}

// The same of a block of bytes, four to a word: pieces of eight.
__device__ __forceinline__ void block_rows_u8(const uint32_t (&w)[4], u32x2 (&set)[2]) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const auto x = __builtin_amdgcn_permlane32_swap(w[2 * p], w[2 * p + 1], false, false);
    set[p] = u32x2{x[0], x[1]};
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = set[0][i], v = set[1][i];
    const auto x = __builtin_amdgcn_permlane16_swap(u, v, false, false);
    set[0][i] = x[0];
    set[1][i] = x[1];
  }
}

// The block in fp32: set 2 c + q holds, of rows 16 q + lane % 16, n = 16 c + 8 (lane / 16 % 2) + 4 (lane / 32) .. + 3.
__device__ __forceinline__ void block_rows_f32(const f32x16 &v, u32x4 (&set)[4]) {
#pragma unroll
  for (int a = 0; a < 4; ++a)
    set[a] = __builtin_bit_cast(u32x4, (f32x4{v[4 * a], v[4 * a + 1], v[4 * a + 2], v[4 * a + 3]}));
  swap_rows(set[0], set[1]);
  swap_rows(set[2], set[3]);
}

// Both sums of M N elements as the backward reads them: 20 bits each, fp32 rounded to 12 significant bits,
// the high halves as two matrices of bf16 and the low four bits of both in a byte.
struct SavedSums {
  bf16 *high[2];
  uint8_t *low;
  __host__ __device__ SavedSums(uint8_t *p, int64_t n)
      : high{reinterpret_cast<bf16 *>(p), reinterpret_cast<bf16 *>(p) + n}, low(p + 4 * n) {}
};

// Four elements of both: their high halves in pairs, and a byte of low bits each, g's below u's.  Half a step is
// added and the bits past the twelfth are left out, so an infinity stays one, and a NaN does: its low bits are zero (an
// operand's, which has 16 bits) or it is the matrix unit's own.
__device__ __forceinline__ void saved_four(const float (&g)[4], const float (&u)[4], uint32_t *gh, uint32_t *uh,
                                           uint32_t &low) {
  uint32_t x[4], y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __float_as_uint(g[e]) + 0x800u, y[e] = __float_as_uint(u[e]) + 0x800u;
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    gh[e / 2] = __builtin_amdgcn_perm(x[e + 1], x[e], 0x07060302u);
    uh[e / 2] = __builtin_amdgcn_perm(y[e + 1], y[e], 0x07060302u);
  }
  // the second byte of each, whose upper half is wanted (0x0c: zero)
  const uint32_t p = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0501u) | __builtin_amdgcn_perm(x[3], x[2], 0x05010c0cu);
  const uint32_t q = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0501u) | __builtin_amdgcn_perm(y[3], y[2], 0x05010c0cu);
  low = (p >> 4 & 0x0f0f0f0fu) | (q & 0xf0f0f0f0u);
}

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + exp2f_fast(-x * kLog2e));
}

namespace {

// Work in tiles: `splits` parts of the contraction, z problems, tiles_m x tiles_n tiles of each.
struct Tiles {
  int splits, z, tiles_m, tiles_n;
  __host__ __device__ int total() const { return splits * z * tiles_m * tiles_n; }
};

struct Tile {
  int part, z, m, n;
};

// The i-th tile in the order of work.  Consecutive workgroup ids go to the 8 XCDs in turn, each with its own
// L2, so each XCD gets a run of tiles; a run goes down bands of 8 rows of tiles before the next column:
// those at work at one time share rows of X and of W.
__device__ __forceinline__ Tile tile_at(const Tiles &g, int i) {
  const int n = g.total(), x = i % 8, rem = n % 8;
  int t = x * (n / 8) + (x < rem ? x : rem) + i / 8;
  const int per = g.tiles_m * g.tiles_n, zs = t / per;
  t -= zs * per;
  const int band = 8 * g.tiles_n, b0 = t / band * 8, rows = min(8, g.tiles_m - b0), in = t - t / band * band;
  return Tile{zs / g.z, zs % g.z, b0 + in % rows, in / rows};
}

// The first of `stages` (at most 2^25: 64 of 2^31 rows each) stages that a part, of at most 32, takes.
__device__ __forceinline__ int first_stage(const Tiles &g, int stages, int part) {
  return (int)((uint32_t)(stages * part) / (uint32_t)g.splits);
}

// kPartial: kStore's sums in fp32, one of `splits` parts of the contraction.
// kGatedSave: kGated, and both sums for the backward.
enum Epilogue { kStore, kPartial, kGated, kGatedSave };

struct GemmArgs {
  const bf16 *x[2], *w[2];  // kStore, kPartial: segments of the sum (segs) or problems (z)
  int64_t ldx, ldw;
  int64_t M, N, K;          // K of one segment
  int segs, z;
  bf16 *out[2];             // [M][N]
  float *part;              // kPartial: [splits][z][M][N]
  uint8_t *saved;           // kGatedSave: SavedSums of M N elements
  Tiles tiles;
};

// Keeps a step's LDS reads among its first products, two to each, where the compiler would put them
// right before their use; nothing moves across.
template <int PRODUCTS>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instructions
  }
  __builtin_amdgcn_sched_barrier(0);
}

// Workgroups take tiles in turn, and load the next one's first stages during the last steps of the one
// before, so that its results are rounded and stored while those are on their way.
template <int TM, int TN, int WM, int WN, int BK, int S, bool XTR, bool WTR, Epilogue E>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs g) {
  constexpr int NT = 64 * WM * WN, MB = TM / WM / 32, NB = TN / WN / 32, STEPS = BK / 16;
  constexpr bool DUAL = E == kGated || E == kGatedSave;
  static_assert(!DUAL || (NB == 2 && !WTR), "a wave has 32 columns of both sums");
  static_assert(STEPS % 2 == 0, "operands alternate between two sets of registers");
  constexpr int WT = DUAL ? TN / 2 : TN, STORES = MB * (E == kGated ? 2 : E == kGatedSave ? 8 : E == kPartial ? 4 * NB : 2 * NB);
  using XL = TileLoad<TM, BK, XTR, NT>;
  using WL = TileLoad<WT, BK, WTR, NT>;
  constexpr int STAGE = (TM + TN) * BK * 2;
  extern __shared__ __align__(1024) char lds[];

  const int total = g.tiles.total();
  const int per_seg = (int)((g.K + BK - 1) / BK), all_stages = per_seg * g.segs;

  // Loads: a cursor over the stages of this workgroup's tiles.
  XL xl;
  WL wl;  // of a dual tile both weights' rows
  const int64_t beside = DUAL ? reinterpret_cast<const char *>(g.w[1]) - reinterpret_cast<const char *>(g.w[0]) : 0;
  int ahead = blockIdx.x, seg, to_do;  // stages of the tile at `at`
  int64_t left;
  Tile at;
  auto start = [&](int skip) {
    const int i = at.z + seg;
    xl.init(g.x[i], g.ldx, (int64_t)at.m * TM, g.M);
    wl.init(g.w[i], g.ldw, (int64_t)at.n * WT, g.N);
    if constexpr (E == kPartial) xl.skip(skip), wl.skip(skip);
    left = g.K - (int64_t)skip * BK;
  };
  auto next_tile = [&] {
    at = tile_at(g.tiles, ahead);
    const int first = first_stage(g.tiles, all_stages, at.part);
    to_do = first_stage(g.tiles, all_stages, at.part + 1) - first;
    seg = first / per_seg;
    start(first - seg * per_seg);
  };
  next_tile();
  auto load = [&](int buf) {
    if (ahead >= total) return;
    char *dst = lds + buf * STAGE;
    if (left < BK) {
      xl.shorten(g.ldx, (int)left);
      wl.shorten(g.ldw, (int)left);
    }
    xl.load(dst);
    if constexpr (DUAL) wl.load_beside(beside, dst + XL::BYTES + WL::BYTES);
    wl.load(dst + XL::BYTES);
    left -= BK;
    if (--to_do == 0) {
      ahead += gridDim.x;
      if (ahead < total) next_tile();
    } else if (left <= 0) {
      ++seg;
      start(0);
    }
  };

  const int wave = wave_id(), wm = wave / WN, wn = wave % WN, lane = threadIdx.x & 63;
  TileRead<TM, BK, XTR> xr;
  TileRead<TN, BK, WTR, DUAL ? TN / 2 : 32> wr;
  xr.init(wm * (TM / WM));
  wr.init(wn * (DUAL ? 32 : TN / WN));
  bf16x8 xf[2][MB], wf[2][NB];
  auto read = [&](int buf, int s, int into) {
    const char *from = lds + buf * STAGE;
#pragma unroll
    for (int b = 0; b < NB; ++b) wf[into][b] = wr.read(from + XL::BYTES, b, s);
#pragma unroll
    for (int b = 0; b < MB; ++b) xf[into][b] = xr.read(from, b, s);
  };

  // Operands of a step are read during the step before it.  All reads of a stage are so done before its
  // last step: there the workgroup meets, the stage's buffer takes the loads of the stage that is S
  // further on, and the next stage is read from.  Loads that were issued after the next stage's may still
  // be on their way, and so may a tile's stores, if they are younger than those.
  constexpr int LOADS = XL::LOADS + WL::LOADS * (DUAL ? 2 : 1);
#pragma unroll
  for (int b = 0; b < S; ++b) load(b);
  if (ahead < total) wait_and_meet<(S - 1) * LOADS>();
  else wait_and_meet<0>();
  read(0, 0, 0);
  int buf = 0;
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    const Tile t = tile_at(g.tiles, i);
    const int64_t m0 = (int64_t)t.m * TM, n0 = (int64_t)t.n * WT;
    const int stages = first_stage(g.tiles, all_stages, t.part + 1) - first_stage(g.tiles, all_stages, t.part);
    f32x16 acc[MB][NB] = {};
    const int row = wm * (TM / WM) + (lane & 15), col = wn * (DUAL ? 32 : TN / WN) + 8 * piece_of(lane);
    const uint32_t row_bytes = (uint32_t)g.N * (E == kPartial ? 4 : 2);
    const uint32_t bytes = (uint32_t)(g.M - m0 < TM ? g.M - m0 : TM) * row_bytes;
    // byte offset in the tile's rows of this lane's piece of set q of block (i, j): past the end with its column
    uint32_t piece0[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int n = (int)n0 + col + 32 * j;
      piece0[j] = n < (int)g.N ? row * row_bytes + 2 * n : kPastEnd;
    }
    auto piece_at = [&](int i, int j, int q) { return piece0[j] + (32 * i + 16 * q) * row_bytes; };
    for (int st = 0; st < stages; ++st) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (s + 1 < STEPS) {
          read(buf, s + 1, (s + 1) & 1);
        } else {
          if (ahead >= total) wait_and_meet<0>();
          else if (st <= S - 2 && i != (int)blockIdx.x) wait_and_meet<(S - 2) * LOADS + STORES>();
          else wait_and_meet<(S - 2) * LOADS>();
          load(buf);
          buf = buf + 1 == S ? 0 : buf + 1;
          read(buf, 0, (s + 1) & 1);  // after the last stage: values that nothing uses
        }
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[i][j] = mfma32(wf[s & 1][j], xf[s & 1][i], acc[i][j]);
        interleave<MB * NB>();
      }
    }

    if constexpr (E == kPartial) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(g.part + ((int64_t)(t.part * g.z + t.z) * g.M + m0) * g.N, bytes);
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          u32x4 set[4];
          block_rows_f32(acc[i][j], set);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n = (int)n0 + wn * (TN / WN) + 32 * j + 16 * (q / 2) + 8 * ((lane >> 4) & 1) + 4 * (lane >> 5);
            const uint32_t to = n < (int)g.N ? row * row_bytes + 4 * n : kPastEnd;
            buf_store16(r, to + (32 * i + 16 * (q % 2)) * row_bytes, set[q]);
          }
        }
      continue;
    }
    const __amdgpu_buffer_rsrc_t r0 = make_rsrc(g.out[E == kStore ? t.z : 0] + m0 * g.N, bytes);
    const SavedSums saved(g.saved, g.M * g.N);
    const __amdgpu_buffer_rsrc_t rg = make_rsrc(saved.high[0] + m0 * g.N, bytes);
    const __amdgpu_buffer_rsrc_t ru = make_rsrc(saved.high[1] + m0 * g.N, bytes);
    const __amdgpu_buffer_rsrc_t rl = make_rsrc(saved.low + m0 * g.N, bytes / 2);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      if constexpr (E == kStore) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          u32x4 set[2];
          block_rows(acc[i][j], set);
          buf_store16(r0, piece_at(i, j, 0), set[0]);
          buf_store16(r0, piece_at(i, j, 1), set[1]);
        }
      } else {
        f32x16 v;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[i][0][e] * sigmoid(acc[i][0][e]) * acc[i][1][e];
        u32x4 set[2];
        block_rows(v, set);
        buf_store16(r0, piece_at(i, 0, 0), set[0]);
        buf_store16(r0, piece_at(i, 0, 1), set[1]);
        if constexpr (E == kGatedSave) {
          uint32_t high[2][8], low[4];
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const f32x16 &g4 = acc[i][0], &u4 = acc[i][1];
            saved_four({g4[4 * a], g4[4 * a + 1], g4[4 * a + 2], g4[4 * a + 3]},
                       {u4[4 * a], u4[4 * a + 1], u4[4 * a + 2], u4[4 * a + 3]}, &high[0][2 * a], &high[1][2 * a], low[a]);
          }
          block_rows(high[0], set);
          buf_store16(rg, piece_at(i, 0, 0), set[0]);
          buf_store16(rg, piece_at(i, 0, 1), set[1]);
          block_rows(high[1], set);
          buf_store16(ru, piece_at(i, 0, 0), set[0]);
          buf_store16(ru, piece_at(i, 0, 1), set[1]);
          u32x2 bytes8[2];
          block_rows_u8(low, bytes8);
          buf_store8(rl, piece_at(i, 0, 0) / 2, bytes8[0]);
          buf_store8(rl, piece_at(i, 0, 1) / 2, bytes8[1]);
        }
      }
    }
  }
}

// Sums of parts [splits][n8 * 8], rounded to bf16: the first n0 pieces of 8 to out0, the others to out1.
__global__ __launch_bounds__(256) void sum_parts_kernel(const float *__restrict__ part, bf16 *__restrict__ out0,
                                                        bf16 *__restrict__ out1, int splits, int64_t n0, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  f32x4 a{}, b{};
  for (int s = 0; s < splits; ++s) {
    const f32x4 *p = reinterpret_cast<const f32x4 *>(part) + (s * n + i) * 2;
    a += p[0];
    b += p[1];
  }
  const bf16x4 x = pack4(a[0], a[1], a[2], a[3]), y = pack4(b[0], b[1], b[2], b[3]);
  reinterpret_cast<bf16x8 *>(i < n0 ? out0 : out1)[i < n0 ? i : i - n0] =
      bf16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
}

template <bool XTR, bool WTR, Epilogue E, int TM, int WM, int WN, int S>
hipError_t launch_tiles(GemmArgs g, int splits, hipStream_t stream) {
  constexpr int BK = 64, TN = TM, DUAL = E == kGated || E == kGatedSave, WT = DUAL ? TN / 2 : TN;
  constexpr int lds = S * (TM + TN) * BK * 2;
  constexpr auto kernel = gemm_kernel<TM, TN, WM, WN, BK, S, XTR, WTR, E>;
  g.tiles = Tiles{splits, g.z, (int)((g.M + TM - 1) / TM), (int)((g.N + WT - 1) / WT)};
  if constexpr (lds > 65536) {
    const hipError_t e = allow_lds<kernel>(lds);
    if (e != hipSuccess) return e;
  }
  const int slots = resident_slots<kernel>(64 * WM * WN, lds);
  kernel<<<dim3(std::min(slots, g.tiles.total())), dim3(64 * WM * WN), lds, stream>>>(g);
  return hipGetLastError();
}

hipError_t launch_sum_parts(const float *part, bf16 *out0, bf16 *out1, int splits, int64_t n0, int64_t n,
                            hipStream_t stream) {
  sum_parts_kernel<<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream>>>(part, out0, out1, splits, n0, n);
  return hipGetLastError();
}

template <bool XTR, bool WTR, Epilogue E>
hipError_t launch_cut(const GemmArgs &g, const Cut &c, hipStream_t stream) {
  if (c.wide) return launch_tiles<XTR, WTR, E, 256, 2, 4, 2>(g, c.splits, stream);
  return c.deep ? launch_tiles<XTR, WTR, E, 128, 4, 2, 4>(g, c.splits, stream)
                : launch_tiles<XTR, WTR, E, 128, 2, 2, 2>(g, c.splits, stream);
}

template <bool XTR, bool WTR, Epilogue E>
hipError_t launch_gemm(const GemmArgs &g, const Cut &c, hipStream_t stream) {
  if constexpr (E == kStore) {
    if (c.splits > 1) {
      const hipError_t e = launch_cut<XTR, WTR, kPartial>(g, c, stream);
      if (e != hipSuccess) return e;
      return launch_sum_parts(g.part, g.out[0], g.out[1], c.splits, g.M * g.N / 8, g.z * g.M * g.N / 8, stream);
    }
  }
  return launch_cut<XTR, WTR, E>(g, c, stream);
}

}  // namespace

}  // namespace ttfa
