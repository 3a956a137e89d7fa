// Matrix products of bf16 operands with fp32 sums, gfx950: out[m][n] = sum_k X(m, k) W(n, k) as tiles
// of TM x TN, for the kernels whose epilogues differ (swiglu.hip, linear_mx.hip).
//
// An operand is read as it lies in memory: rows along k (row m holds its k's), or rows along the
// other index (row k holds its m's; TR), so no product needs a transposed copy.  Tiles go straight
// to LDS (16 bytes a lane, double-buffered: the next stage's loads run during this stage's products)
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

#include "fa_common.h"

namespace ttfa {

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

constexpr uint32_t kPastEnd = 0x80000000u;  // an offset that no tile's buffer covers

// One operand's tile of T rows (of the m or n index) x BK, loaded by NT threads, stage after stage along k.
template <int T, int BK, bool TR, int NT>
struct TileLoad {
  static constexpr int LOADS = T * BK * 2 / 16 / NT;
  static constexpr int CPR = TR ? T / 8 : BK / 8;  // 16-byte chunks of an LDS row
  static constexpr int BYTES = T * BK * 2;
  static_assert(T * BK * 2 % (16 * NT) == 0 && (!TR || T >= 128), "tile");
  const char *base;  // of the next stage
  uint32_t bytes;    // that the tile's rows have from there on
  int64_t step;      // bytes to the stage after it
  uint32_t off[LOADS];

  static __device__ __forceinline__ int swizzle(int row) {
    return TR ? (row & 3) << 2 : (row / (16 / CPR)) & (CPR - 1);
  }

  // The matrix at p, rows of ld elements: tile from row (TR: column) r0 of R on.
  __device__ __forceinline__ void init(const bf16 *p, int64_t ld, int64_t r0, int64_t R) {
    start(p, ld, r0, R);
    step = TR ? ld * (BK * 2) : BK * 2;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int e = j * NT + (int)threadIdx.x, row = e / CPR;
      off[j] = (uint32_t)(row * ld * 2) + ((e % CPR) ^ swizzle(row)) * 16;
    }
  }
  // The same tile of another matrix of the same shape (k from 0 again).
  __device__ __forceinline__ void start(const bf16 *p, int64_t ld, int64_t r0, int64_t R) {
    base = reinterpret_cast<const char *>(p + (TR ? r0 : r0 * ld));
    const int64_t rows = R - r0 < T ? R - r0 : T;
    bytes = rows <= 0 ? 0u : (uint32_t)((TR ? BK * ld - r0 : rows * ld) * 2);
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
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int e = j * NT + (int)threadIdx.x, row = e / CPR;
        if (8 * ((e % CPR) ^ swizzle(row)) >= left) off[j] = kPastEnd;
      }
    }
  }
  __device__ __forceinline__ void load(char *lds) {
    char *dst = lds + wave_id() * 1024;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base, bytes);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) buf_load16_lds(r, off[j], dst + j * NT * 16);
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
// rows.  (With 32 bytes of 32 rows, as the halves of the wave have them, stores took about twice the time.)
__device__ __forceinline__ int piece_of(int lane) { return 2 * ((lane >> 4) & 1) + (lane >> 5); }

__device__ __forceinline__ void swap_rows(u32x4 &a, u32x4 &b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto x = __builtin_amdgcn_permlane16_swap(a[i], b[i], false, false);
    a[i] = x[0];
    b[i] = x[1];
  }
}

__device__ __forceinline__ void block_rows(const f32x16 &v, u32x4 (&set)[2]) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const u32x2 a = __builtin_bit_cast(u32x2, pack4(v[8 * p], v[8 * p + 1], v[8 * p + 2], v[8 * p + 3]));
    const u32x2 b = __builtin_bit_cast(u32x2, pack4(v[8 * p + 4], v[8 * p + 5], v[8 * p + 6], v[8 * p + 7]));
    const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
    set[p] = u32x4{x[0], y[0], x[1], y[1]};
  }
  swap_rows(set[0], set[1]);
}

// The block in fp32: set 2 c + q holds, of rows 16 q + lane % 16, n = 16 c + 8 (lane / 16 % 2) + 4 (lane / 32) .. + 3.
__device__ __forceinline__ void block_rows_f32(const f32x16 &v, u32x4 (&set)[4]) {
#pragma unroll
  for (int a = 0; a < 4; ++a)
    set[a] = __builtin_bit_cast(u32x4, (f32x4{v[4 * a], v[4 * a + 1], v[4 * a + 2], v[4 * a + 3]}));
  swap_rows(set[0], set[1]);
  swap_rows(set[2], set[3]);
}

// The inverse: a block's registers from such pieces.
__device__ __forceinline__ f32x16 block_regs(u32x4 a, u32x4 b) {
  swap_rows(a, b);
  f32x16 v;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const u32x4 c = p ? b : a;
    const auto x = __builtin_amdgcn_permlane32_swap(c[0], c[2], false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(c[1], c[3], false, false);
    const bf16x8 w = __builtin_bit_cast(bf16x8, (u32x4{x[0], y[0], x[1], y[1]}));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * p + i] = (float)w[i];
  }
  return v;
}

}  // namespace ttfa
