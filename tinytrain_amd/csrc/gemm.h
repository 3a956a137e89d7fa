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

// Rows of `ld` elements from p; `rows` of them.
struct Operand {
  const bf16 *p;
  int64_t ld;
  int64_t rows;
};

// Buffer resource over [p, end), at most 2^31 - 1 bytes of it.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_to(const bf16 *p, const bf16 *end) {
  const int64_t left = (end - p) * 2;
  return make_rsrc(p, left <= 0 ? 0u : left > 0x7fffffff ? 0x7fffffffu : (uint32_t)left);
}

constexpr uint32_t kPastEnd = 0x80000000u;  // an offset that no resource covers

// One operand's tile of T rows (of the m or n index) x BK, loaded by NT threads.
template <int T, int BK, bool TR, int NT>
struct TileLoad {
  static constexpr int LOADS = T * BK * 2 / 16 / NT;
  static constexpr int CPR = TR ? T / 8 : BK / 8;  // 16-byte chunks of an LDS row
  static constexpr int BYTES = T * BK * 2;
  static_assert(T * BK * 2 % (16 * NT) == 0 && (!TR || T >= 128), "tile");
  uint32_t off[LOADS];
  int chunk[LOADS];

  static __device__ __forceinline__ int swizzle(int row) {
    return TR ? (row & 3) << 2 : (row / (16 / CPR)) & (CPR - 1);
  }
  // Rows from `half` on are row - half of a second source (dual tiles).
  __device__ __forceinline__ void init(int64_t ld, int half = T) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int e = j * NT + (int)threadIdx.x, row = e / CPR, ch = (e % CPR) ^ swizzle(row);
      chunk[j] = ch;
      off[j] = (uint32_t)((row >= half ? row - half : row) * ld * 2 + ch * 16);
    }
  }
  // Loads j0 .. j1 - 1 from the buffer r; `left`: the k's that rows along k still have.
  template <int J0, int J1>
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, char *lds, int64_t left) const {
    char *dst = lds + wave_id() * 1024;
    if (TR || left >= BK) {
#pragma unroll
      for (int j = J0; j < J1; ++j) buf_load16_lds(r, off[j], dst + j * NT * 16);
    } else {
#pragma unroll
      for (int j = J0; j < J1; ++j)
        buf_load16_lds(r, 8 * chunk[j] < left ? off[j] : kPastEnd, dst + j * NT * 16);
    }
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

// Registers of a 32 x 32 result block, rounded to bf16, as 16-byte pieces of rows: lane's piece p is
// n = 16 p + 8 (lane / 32) .. + 7 of its column m.
__device__ __forceinline__ u32x4 row_piece(const f32x16 &v, int p) {
  const u32x2 a = __builtin_bit_cast(u32x2, pack4(v[8 * p], v[8 * p + 1], v[8 * p + 2], v[8 * p + 3]));
  const u32x2 b = __builtin_bit_cast(u32x2, pack4(v[8 * p + 4], v[8 * p + 5], v[8 * p + 6], v[8 * p + 7]));
  const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
  return u32x4{x[0], y[0], x[1], y[1]};
}

// The inverse: registers 8p .. 8p + 7 of a block from piece p of bf16 rows.
__device__ __forceinline__ void block_regs(u32x4 piece, f32x16 &v, int p) {
  const auto x = __builtin_amdgcn_permlane32_swap(piece[0], piece[2], false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(piece[1], piece[3], false, false);
  const bf16x8 b = __builtin_bit_cast(bf16x8, (u32x4{x[0], y[0], x[1], y[1]}));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[8 * p + i] = (float)b[i];
}

}  // namespace ttfa
