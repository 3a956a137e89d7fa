// How a product of M x N over a contraction of K is cut into work for 256 CUs: the rules by which gemm.h, swiglu.hip
// and linear_mx.hip choose their kernels.  Sizes alone decide, in host code that needs no HIP, so that a test can ask
// which kernel a size takes.
#pragma once

#include <cstdint>

namespace ttfa {

// How a product is cut: tiles of 256 x 256 (one workgroup a CU) or 128 x 128 (two, or one with four stages
// in LDS where there are no more than CUs: deep), and parts of the contraction that sum_parts_kernel joins.
struct Cut {
  bool wide;
  int splits;
  bool deep;
};

inline int64_t tiles_of(int64_t M, int64_t N, int tm, int tn) { return (M + tm - 1) / tm * ((N + tn - 1) / tn); }

constexpr double kMostPartFloats = 1 << 26;  // 256 MB, what the last-level cache holds

// The cut that is estimated to take least time, in microseconds on 256 CUs: a stage of 64 k's of a wide
// tile takes 1.5, of a narrow one 0.6 alone on its CU and 0.97 beside another; 3 stages more for a tile's
// start and end; parts go out and in at 4 TB/s, with a launch of 4 us.  What a forward keeps for its backward is the
// same for every cut and not counted.  (Whole rounds of narrow tiles take 0.9 to
// 1.06 a stage; 0.97 decides the near draws as they were measured: forward 2048 x 2048 x 6144 wide 110, narrow 101;
// 4096 x 1024 x 2816: 58, 52; dx of 4096 x 2048 x 6144: wide in two parts 232 with the kernel before it, narrow 262.)
inline Cut cut_of(int64_t M, int64_t N, int64_t K, int segs, int z, bool dual) {
  const int64_t stages = (K + 63) / 64 * segs;
  Cut best{true, 1, false};
  double least = 1e30;
  for (int wide = 1; wide >= 0; --wide) {
    const int64_t tiles = z * (wide ? tiles_of(M, N, 256, dual ? 128 : 256) : tiles_of(M, N, 128, dual ? 64 : 128));
    for (int s = 1; s <= (dual ? 1 : 32) && s <= stages; ++s) {
      if (s > 1 && (double)s * z * M * N > kMostPartFloats) break;
      const int64_t n = tiles * s;
      const double len = (double)((stages + s - 1) / s) + 3;
      const bool deep = !wide && n <= 256;
      double t = len * (wide ? (double)((n + 255) / 256) * 1.5 : deep ? 0.6 : (double)((n + 511) / 512) * 0.97);
      if (s > 1) t += 4 + (double)s * z * M * N * 8 / 4e6;
      if (t < least) least = t, best = Cut{wide != 0, s, deep};
    }
  }
  return best;
}

inline int64_t part_bytes(const Cut &c, int64_t M, int64_t N, int z) {
  return c.splits > 1 ? 4 * c.splits * z * M * N : 0;
}

// Rows of x up to which swiglu's kernel for few rows is faster than tiles (us, K x N: rows, tiles).  768 x 2304, 64
// rows: 7.2, 11.2; 2048 x 6144: 20.7, 22.0; 4096 x 8192: 39.6, 39.2.  More columns give a tile to each CU, and reading
// x again for every 16 of them counts: 4096 x 12288, 1 row: 36.7, 41.1; 16: 45.3, 42.0; 32: 52.7, 44.5; 2048 x 12288,
// 16: 23.9, 24.0.
inline bool swiglu_few_rows(int M, int N) { return M <= (N <= 8192 ? 64 : 16); }

// Whether a call of linear_mx takes the kernel for few rows.  Measured at the borders, us (rows, tiles), K 4096, x and
// W in 8 and 4 bits: N 8192, 64 rows: 15.1, 18.2; N 12288, 32 rows: 11.3, 18.6; 48 rows: 21.8, 20.0; N 20480, 16 rows:
// 19.5, 20.9; 24 rows: 22.7, 21.6.  x in bf16: 21.4, 20.5; 16.3, 23.6; 33.3, 24.5; 23.8, 27.0; 32 rows: 33.8, 28.1;
// 768 x 2304, 64 rows: 5.4, 9.1.  W in 8 bits, x in 8: 18.0, 17.3; 15.6, 20.6; 28.1, 21.8; 29.4, 25.9.
inline bool linear_mx_few_rows(int M, int N) { return M <= (N <= 8192 ? 64 : N <= 16384 ? 32 : 16); }

// With x in 8 bits 128 k's take the time of 64 in bf16.  With x in bf16 (tiles of 128 x 256: wide, or 128 x 128) they
// take 1.6 and 0.95 us.
inline Cut mx_cut(int M, int K, int N, bool x_quantised) {
  if (x_quantised) return cut_of(M, N, K / 2, 1, 1, false);
  const int64_t stages = (K + 127) / 128;
  Cut best{true, 1, false};
  double least = 1e30;
  for (int wide = 1; wide >= 0; --wide)
    for (int s = 1; s <= 32 && s <= stages; ++s) {
      if (s > 1 && (double)s * M * N > kMostPartFloats) break;
      const int64_t n = tiles_of(M, N, 128, wide ? 256 : 128) * s;
      double t = (double)((n + 255) / 256) * (wide ? 1.6 : 0.95) * (double)((stages + s - 1) / s + 3);
      if (s > 1) t += 4 + (double)s * M * N * 8 / 4e6;
      if (t < least) least = t, best = Cut{wide != 0, s, false};
    }
  return best;
}

}  // namespace ttfa
