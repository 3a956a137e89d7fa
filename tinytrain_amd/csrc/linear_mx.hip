// Products with a quantised weight, gfx950: y[m][n] = sum_k x[m][k] W[n][k], W in 4 or 8 bits with a
// power of two per 32 elements (kv_cache_mx.hip describes the format), x in bf16 or in 8 bits as the
// norm's kernel gives it.  The reference has no counterpart (its linear layers are bf16 products).
//
// Every value of either format is a bf16 as it stands, so with x in bf16 the products are bf16 ones with
// fp32 sums, of values that are formed in registers.  With x in 8 bits the matrix unit takes both as they lie, with
// their scales (v_mfma_scale_f32_16x16x128_f8f6f4, twice the rate, no conversions); of every eight consecutive
// products it drops the bits below 2^-13 of the largest before it adds in fp32 (fa_decode_mx.hip), so a
// sum is off by less than 2^-10 of those largest ones' sum, on random values by 2^-19 of sum |x w|, far
// below the 2^-9 of y's own rounding.
//
// Few rows: bound by reading W once, and by the cache lines that its loads touch.  A workgroup takes 16 NB rows
// of W and each of its eight waves an eighth of the columns, in blocks of 128, two or four of these at once (as
// many as registers hold).  A lane has, of its row, 32 consecutive elements of a block (e4m3 with x in 8 bits: 16
// and the 16 that are 64 further on, the matrix unit's layout).  The waves' sums are joined through LDS.  4096 x
// 12288 in 4 bits, us: one row 8.0 (3.3 TB/s, of which a launch and one round of loads are half), 32 rows 11.3;
// with every eighth block to a wave, and so a load for each scale, 8.8 and 14.0.
#include <type_traits>

#include "fa_common.h"
#include "fa_kernels.h"
#include "gemm.h"
#include "mx.h"
#include "ttfa.h"

namespace ttfa {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kRowWaves = 8;

// Scale bytes of a lane's row in U blocks of four groups, of group q of each: the row's bytes lie together, so one
// load of 4 U of them where the row has as many left, and not U of one byte each.
template <int U>
struct Scales {
  uint32_t w[U];
  int shift;
  // at: the first block's first byte, `left` groups from there to the row's end
  __device__ __forceinline__ void load(const uint8_t *at, int left, int q) {
    if (left >= 4 * U) {
      __builtin_memcpy(w, at, 4 * U);
      shift = 8 * q;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = 4 * u + q < left ? at[4 * u + q] : 127;
      shift = 0;
    }
  }
  __device__ __forceinline__ uint32_t byte(int u) const { return w[u] >> shift & 255; }
};

// 32 consecutive elements (a group) of a row of W, as bf16 for the product with x in bf16.
template <int BITS>
struct Group {
  u32x4 c[BITS / 4];
  __device__ __forceinline__ void load(const uint8_t *codes, int64_t group, bool ok) {
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i)
      c[i] = ok ? reinterpret_cast<const u32x4 *>(codes + group * (4 * BITS))[i] : u32x4{};
  }
  // elements 8 j .. 8 j + 7
  __device__ __forceinline__ bf16x8 values(int j, uint32_t byte) const {
    const float scale = __uint_as_float(byte << 23);
    if constexpr (BITS == 4) return mx_values8<4>(u32x2{c[0][j], 0u}, scale);
    else return mx_values8<8>(u32x2{c[j / 2][2 * (j % 2)], c[j / 2][2 * (j % 2) + 1]}, scale);
  }
};

struct Rows32 {
  u32x4 c[4];
  __device__ __forceinline__ void load(const bf16 *x, int64_t group, bool ok) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = ok ? reinterpret_cast<const u32x4 *>(x + group * 32)[j] : u32x4{};
  }
  __device__ __forceinline__ bf16x8 values(int j) const { return __builtin_bit_cast(bf16x8, c[j]); }
};

// A lane's part of 128 k's of a row as an operand of the scaled product: lane i + 16 q has the scale of
// elements 32 q .. 32 q + 31 and those elements (BITS 4), or 16 q .. and 64 + 16 q .. (BITS 8).
template <int BITS>
struct Scaled {
  u32x4 c[BITS / 4];
  // group0: the first of the row's four groups, `left` groups from there to the row's end
  __device__ __forceinline__ void load(const uint8_t *codes, int64_t group0, int left, int q) {
    if constexpr (BITS == 4) {
      c[0] = q < left ? *reinterpret_cast<const u32x4 *>(codes + (group0 + q) * 16) : u32x4{};
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        c[i] = 2 * i + q / 2 < left ? *reinterpret_cast<const u32x4 *>(codes + group0 * 32 + 64 * i + 16 * q) : u32x4{};
    }
  }
  __device__ __forceinline__ i32x8 operand() const {
    i32x8 v{};
#pragma unroll
    for (int i = 0; i < BITS; ++i) v[i] = (int)c[i / 4][i % 4];
    return v;
  }
};

template <int BITS, bool XMX, int MB, int NB>
__global__ __launch_bounds__(64 * kRowWaves) void linear_mx_rows_kernel(
    const void *__restrict__ x, const uint8_t *__restrict__ x_scales, const uint8_t *__restrict__ codes,
    const uint8_t *__restrict__ scales, bf16 *__restrict__ y, int M, int K, int N) {
  constexpr int U = XMX && MB <= 2 && NB * BITS / 4 + 2 * MB <= 10 ? 4 : 2;
  __shared__ f32x4 part[kRowWaves][NB * MB][64];
  const int lane = threadIdx.x & 63, wave = wave_id(), row = lane & 15, quarter = lane >> 4;
  const int n0 = blockIdx.x * 16 * NB, groups = K / 32, blocks = (groups + 3) / 4;
  const int each = (blocks + kRowWaves - 1) / kRowWaves, end = min(blocks, each * (wave + 1));
  int64_t wrow[NB], xrow[MB];  // rows past the end: the last one's, not stored
#pragma unroll
  for (int c = 0; c < NB; ++c) wrow[c] = (int64_t)min(n0 + 16 * c + row, N - 1) * groups;
#pragma unroll
  for (int b = 0; b < MB; ++b) xrow[b] = (int64_t)min(16 * b + row, M - 1) * groups;
  f32x4 acc[NB][MB] = {};
  for (int k = each * wave; k < end; k += U) {
    const int left = groups - 4 * k;  // to the row's end
    Scales<U> ws[NB];
#pragma unroll
    for (int c = 0; c < NB; ++c) ws[c].load(scales + wrow[c] + 4 * k, left, quarter);
    if constexpr (XMX) {
      Scaled<BITS> w[U][NB];
      Scaled<8> v[U][MB];
      Scales<U> xs[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) xs[b].load(x_scales + xrow[b] + 4 * k, left, quarter);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = 4 * (k + u), of = k + u < end ? groups - at : 0;
#pragma unroll
        for (int c = 0; c < NB; ++c) w[u][c].load(codes, wrow[c] + at, of, quarter);
#pragma unroll
        for (int b = 0; b < MB; ++b) v[u][b].load((const uint8_t *)x, xrow[b] + at, of, quarter);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
          for (int b = 0; b < MB; ++b)
            acc[c][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                w[u][c].operand(), v[u][b].operand(), acc[c][b], BITS == 4 ? 4 : 0, 0, 0, (int)ws[c].byte(u), 0,
                (int)xs[b].byte(u));
    } else {
      Group<BITS> w[U][NB];
      Rows32 v[U][MB];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = 4 * (k + u) + quarter;
        const bool ok = k + u < end && at < groups;
#pragma unroll
        for (int c = 0; c < NB; ++c) w[u][c].load(codes, wrow[c] + at, ok);
#pragma unroll
        for (int b = 0; b < MB; ++b) v[u][b].load((const bf16 *)x, xrow[b] + at, ok);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int c = 0; c < NB; ++c) {
            const bf16x8 wv = w[u][c].values(j, ws[c].byte(u));
#pragma unroll
            for (int b = 0; b < MB; ++b)
              acc[c][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, v[u][b].values(j), acc[c][b], 0, 0, 0);
          }
    }
  }
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int b = 0; b < MB; ++b) part[wave][c * MB + b][lane] = acc[c][b];
  __syncthreads();
  if (wave >= NB * MB) return;
  f32x4 t{};
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) t += part[w][wave][lane];
  const int m = 16 * (wave % MB) + row, n = n0 + 16 * (wave / MB) + 4 * quarter;
  if (m < M && n < N) *reinterpret_cast<bf16x4 *>(y + (int64_t)m * N + n) = pack4(t[0], t[1], t[2], t[3]);
}

// Many rows: tiles of TM x TN, stages of 128 k's, with the order of gemm_kernel (gemm.h): a persistent
// workgroup, loads S stages ahead, operands read before they are needed.  128 k's of a row of x are 128 or 256
// bytes and of W 64 or 128, loaded as gemm.h's tiles of bf16 of that many bytes; the scales of a stage, four bytes a
// row, go to LDS beside them.  With x in 8 bits a step is 16 rows of x by the wave's columns, whose operands stay in
// registers for a stage.  With x in bf16 it is a quarter of the stage's k's, eight of each group, for which the
// wave's columns become bf16.  What a last stage has past K loads as zeros; rows of scales that are no whole dwords
// are laid out anew first (pad_scales_kernel).
// 4096 x 4096 x 12288 in 4 bits: x in 8 bits 166 to 173 us (2480 to 2380 TFLOP/s), x in bf16 332 (1240); 128 rows: 25
// and 29.  W in 8 bits: 194 and 368.
// With W written out in bf16 first and tiles of that, x in bf16 took 346 and 52, and 2 N K bytes of workspace.
struct MxArgs {
  const uint8_t *x, *x_scales, *codes, *scales;
  bf16 *out;
  float *part;  // PARTIAL: [splits][M][N]
  int64_t M, N, K;
  int sld;      // bytes of a row of scales
  Tiles tiles;
};

// Rows of K / 32 scales of x (rows 0 .. m - 1) and W as rows of whole dwords, the bytes behind them a scale of one.
__global__ __launch_bounds__(256) void pad_scales_kernel(const uint8_t *__restrict__ x_scales,
                                                         const uint8_t *__restrict__ scales, uint32_t *__restrict__ x_out,
                                                         uint32_t *__restrict__ out, int groups, int dwords, int64_t m,
                                                         int64_t rows) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * dwords; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / dwords;
    const int g = 4 * (int)(i - row * dwords);
    const uint8_t *from = row < m ? x_scales + row * groups : scales + (row - m) * groups;
    uint32_t w = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) w |= (g + b < groups ? from[g + b] : 127u) << (8 * b);
    if (row < m) x_out[i] = w;
    else out[i - m * dwords] = w;
  }
}

// The scales of T rows, one dword each, into LDS: waves W0 .. W0 + T / 64 - 1 load one instruction each.
template <int T, int W0>
__device__ __forceinline__ void load_scales(const uint8_t *p, uint32_t bytes, uint32_t ld, char *lds) {
  const int w = wave_id() - W0;
  if (w < 0 || w >= T / 64) return;
  const __amdgpu_buffer_rsrc_t r = make_rsrc(p, bytes);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (TTFA_LDS void *)(lds + w * 256), 4,
                                           (w * 64 + (threadIdx.x & 63)) * ld, 0, 0, 0);
}

template <int TM, int TN, int WM, int WN, int S, int BITS, bool XMX, bool PARTIAL>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_mx_tile_kernel(MxArgs g) {
  constexpr int NT = 64 * WM * WN, MB = TM / WM / 16, NB = TN / WN / 16, STORES = MB * NB / (PARTIAL ? 1 : 2);
  constexpr int XK = XMX ? 64 : 128, WK = BITS == 4 ? 32 : 64;  // bf16's as long as 128 elements of x, W
  using XL = TileLoad<TM, XK, false, NT>;
  using WL = TileLoad<TN, WK, false, NT>;
  static_assert(((XMX ? TM : 0) + TN) / 64 <= NT / 64, "a wave loads scales once a stage");
  constexpr int XS = XL::BYTES + WL::BYTES, WS = XS + (XMX ? 4 * TM : 0), STAGE = WS + 4 * TN;
  extern __shared__ __align__(1024) char lds[];
  const int total = g.tiles.total(), all_stages = (int)((g.K + 127) / 128);
  const uint32_t sld = (uint32_t)g.sld;

  XL xl;
  WL wl;
  const uint8_t *xs, *ws;
  uint32_t xs_bytes, ws_bytes;
  int ahead = blockIdx.x, to_do, left;
  auto next_tile = [&] {
    const Tile at = tile_at(g.tiles, ahead);
    const int first = first_stage(g.tiles, all_stages, at.part);
    const int64_t m0 = (int64_t)at.m * TM, n0 = (int64_t)at.n * TN;
    to_do = first_stage(g.tiles, all_stages, at.part + 1) - first;
    xl.init(reinterpret_cast<const bf16 *>(g.x), XMX ? g.K / 2 : g.K, m0, g.M);
    wl.init(reinterpret_cast<const bf16 *>(g.codes), g.K * BITS / 16, n0, g.N);
    xl.skip(first);
    wl.skip(first);
    left = (int)g.K - 128 * first;
    if constexpr (XMX) {
      xs = g.x_scales + m0 * sld + 4 * first;
      xs_bytes = (uint32_t)((g.M - m0 < TM ? g.M - m0 : TM) * sld) - 4 * first;
    }
    ws = g.scales + n0 * sld + 4 * first;
    ws_bytes = (uint32_t)((g.N - n0 < TN ? g.N - n0 : TN) * sld) - 4 * first;
  };
  next_tile();
  auto load = [&](int buf) {
    if (ahead >= total) return;
    char *dst = lds + buf * STAGE;
    if (left < 128) {
      xl.shorten(0, XMX ? left / 2 : left);
      wl.shorten(0, left * BITS / 16);
    }
    left -= 128;
    xl.load(dst);
    wl.load(dst + XL::BYTES);
    if constexpr (XMX) {
      load_scales<TM, 0>(xs, xs_bytes, sld, dst + XS);
      xs += 4, xs_bytes -= 4;
    }
    load_scales<TN, XMX ? TM / 64 : 0>(ws, ws_bytes, sld, dst + WS);
    ws += 4, ws_bytes -= 4;
    if (--to_do == 0) {
      ahead += gridDim.x;
      if (ahead < total) next_tile();
    }
  };

  const int wave = wave_id(), wm = wave / WN, wn = wave % WN, lane = threadIdx.x & 63;
  const int i16 = lane & 15, q = lane >> 4;
  // Offsets in a stage of this lane's pieces of block 0 (16 rows on: the same swizzle).  With x in 8 bits a second
  // piece is four chunks on: that bit flipped.  With x in bf16 lane q has group q of W (e4m3: its second half in the
  // next chunk), and of x the same 32 elements, four chunks.
  const int xrow = wm * (TM / WM) + i16, wrow = wn * (TN / WN) + i16;
  const int x0 = xrow * (2 * XK) + (((XMX ? q : 4 * q) ^ XL::swizzle(xrow)) << 4);
  const int w0 = XL::BYTES + wrow * (2 * WK) + (((XMX || BITS == 4 ? q : 2 * q) ^ WL::swizzle(wrow)) << 4);
  u32x4 xf[2][XMX ? 2 : MB], wf[NB][BITS / 4];
  uint32_t sx[2], sw[NB];
  // block b (x in bf16: chunk b of all blocks)
  auto read_x = [&](int buf, int b, int into) {
    const char *from = lds + buf * STAGE;
    if constexpr (XMX) {
      xf[into][0] = *reinterpret_cast<const u32x4 *>(from + x0 + b * 2048);
      xf[into][1] = *reinterpret_cast<const u32x4 *>(from + (x0 ^ 64) + b * 2048);
      sx[into] = *reinterpret_cast<const uint8_t *>(from + XS + 4 * xrow + q + b * 64);
    } else {
#pragma unroll
      for (int i = 0; i < MB; ++i) xf[into][i] = *reinterpret_cast<const u32x4 *>(from + (x0 ^ (b << 4)) + i * 4096);
    }
  };
  auto read_w = [&](int buf, int c) {
    const char *from = lds + buf * STAGE;
    wf[c][0] = *reinterpret_cast<const u32x4 *>(from + w0 + c * (32 * WK));
    if constexpr (BITS == 8) wf[c][1] = *reinterpret_cast<const u32x4 *>(from + (w0 ^ (XMX ? 64 : 16)) + c * (32 * WK));
    sw[c] = *reinterpret_cast<const uint8_t *>(from + WS + 4 * wrow + q + c * 64);
  };
  auto operand = [](const u32x4 *c, int n) {
    i32x8 v{};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) v[i] = (int)c[i / 4][i % 4];
    return v;
  };
  // x in bf16: elements 8 j .. 8 j + 7 of the lane's group of block c
  auto values = [&](int c, int j) {
    const u32x4 &v = wf[c][BITS == 4 ? 0 : j / 2];
    const u32x2 codes = BITS == 4 ? u32x2{v[j], 0u} : u32x2{v[2 * (j % 2)], v[2 * (j % 2) + 1]};
    return mx_values8<BITS>(codes, __uint_as_float(sw[c] << 23));
  };
  constexpr int XSTEPS = XMX ? MB : 4;  // of a stage: blocks of rows, or chunks of k's

  constexpr int LOADS = XL::LOADS + WL::LOADS;  // and one of scales in some waves: not counted
#pragma unroll
  for (int b = 0; b < S; ++b) load(b);
  if (ahead < total) wait_and_meet<(S - 1) * LOADS>();
  else wait_and_meet<0>();
#pragma unroll
  for (int c = 0; c < NB; ++c) read_w(0, c);
  read_x(0, 0, 0);
  int buf = 0;
  bf16x8 wv[NB];
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    const Tile t = tile_at(g.tiles, i);
    const int64_t m0 = (int64_t)t.m * TM, n0 = (int64_t)t.n * TN;
    const int stages = first_stage(g.tiles, all_stages, t.part + 1) - first_stage(g.tiles, all_stages, t.part);
    f32x4 acc[MB][NB] = {};
    for (int st = 0; st < stages; ++st) {
#pragma unroll
      for (int b = 0; b < XSTEPS; ++b) {
        if constexpr (!XMX)
#pragma unroll
          for (int c = 0; c < NB; ++c) wv[c] = values(c, b);
        if (b + 1 < XSTEPS) {
          read_x(buf, b + 1, (b + 1) & 1);
        } else {
          if (ahead >= total) wait_and_meet<0>();
          else if (st <= S - 2 && i != (int)blockIdx.x) wait_and_meet<(S - 2) * LOADS + STORES>();
          else wait_and_meet<(S - 2) * LOADS>();
          load(buf);
          buf = buf + 1 == S ? 0 : buf + 1;
          read_x(buf, 0, (b + 1) & 1);  // after the last stage: values that nothing uses
        }
        if constexpr (XMX) {
#pragma unroll
          for (int c = 0; c < NB; ++c) {
            acc[b][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                operand(wf[c], BITS), operand(xf[b & 1], 8), acc[b][c], BITS == 4 ? 4 : 0, 0, 0, (int)sw[c], 0,
                (int)sx[b & 1]);
            if (b + 1 == XSTEPS) {
              read_w(buf, c);  // into the registers that the product has read
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        } else {
          if (b + 1 == XSTEPS)
#pragma unroll
            for (int c = 0; c < NB; ++c) read_w(buf, c);
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int c = 0; c < NB; ++c)
              acc[i][c] = mfma16(wv[c], __builtin_bit_cast(bf16x8, xf[b & 1][i]), acc[i][c]);
        }
        // The products of the step before (of this one, with x in bf16) are done here: without a use they would all
        // be moved behind the last step's wait, and every operand of the stage be held until then.
        if constexpr (XMX) {
          if (b > 0)
#pragma unroll
            for (int c = 0; c < NB; ++c) asm volatile("" : "+v"(acc[b - 1][c]));
        } else if (b + 1 < XSTEPS) {
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int c = 0; c < NB; ++c) asm volatile("" : "+v"(acc[i][c]));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // Byte offsets of rows, a step further for each block.  The lane's part is formed here, not kept over the
    // stages, whose registers it would spill.
    const int64_t rows = g.M - m0 < TM ? g.M - m0 : TM;
    const uint32_t row_bytes = (uint32_t)g.N * (PARTIAL ? 4 : 2);
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    const int lq = l >> 4;
    uint32_t to = (wm * (TM / WM) + (l & 15)) * row_bytes;
    if constexpr (PARTIAL) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(g.part + ((int64_t)t.part * g.M + m0) * g.N, (uint32_t)(rows * g.N * 4));
#pragma unroll
      for (int b = 0; b < MB; ++b, to += 16 * row_bytes)
#pragma unroll
        for (int c = 0; c < NB; ++c) {
          const int n = (int)n0 + wn * (TN / WN) + 16 * c + 4 * lq;
          buf_store16(r, n < g.N ? to + 4 * n : kPastEnd, __builtin_bit_cast(u32x4, acc[b][c]));
        }
    } else {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(g.out + m0 * g.N, (uint32_t)(rows * g.N * 2));
#pragma unroll
      for (int b = 0; b < MB; ++b, to += 16 * row_bytes)
#pragma unroll
        for (int c = 0; c < NB; c += 2) {
          // lanes of odd q take the second block's halves: 16 bytes a lane, 64 of a row
          const f32x4 u = acc[b][c], v = acc[b][c + 1];
          const u32x2 e = __builtin_bit_cast(u32x2, pack4(u[0], u[1], u[2], u[3]));
          const u32x2 f = __builtin_bit_cast(u32x2, pack4(v[0], v[1], v[2], v[3]));
          const auto y0 = __builtin_amdgcn_permlane16_swap(e[0], f[0], false, false);
          const auto y1 = __builtin_amdgcn_permlane16_swap(e[1], f[1], false, false);
          const int n = (int)n0 + wn * (TN / WN) + 16 * c + 16 * (lq & 1) + 8 * (lq >> 1);
          buf_store16(r, n < g.N ? to + 2 * n : kPastEnd, u32x4{y0[0], y1[0], y0[1], y1[1]});
        }
    }
  }
}

// f(bits, whether x is quantised) as compile-time values
template <class F>
hipError_t by_types(int bits, bool xmx, F f) {
  using std::integral_constant;
  if (bits == 4) return xmx ? f(integral_constant<int, 4>{}, std::true_type{}) : f(integral_constant<int, 4>{}, std::false_type{});
  return xmx ? f(integral_constant<int, 8>{}, std::true_type{}) : f(integral_constant<int, 8>{}, std::false_type{});
}

// f(blocks of 16 rows of x, of 16 columns of W) for M rows: as many columns a workgroup as leave 256 of them
// (more than 32 rows come with at most 8192 columns: linear_mx_few_rows).
template <class F>
hipError_t by_blocks(int M, int N, F f) {
  using std::integral_constant;
  const int nb = (N + 16 * 256 - 1) / (16 * 256);
  auto go = [&](auto m, auto most) {
    constexpr int MOST = decltype(most)::value;
    if (nb <= 1) return f(m, integral_constant<int, 1>{});
    if constexpr (MOST > 2) {
      if (nb == 3) return f(m, integral_constant<int, 3>{});
      if (nb > 3) return f(m, integral_constant<int, 4>{});
    }
    return f(m, integral_constant<int, 2>{});
  };
  if (M <= 16) return go(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  if (M <= 32) return go(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  if (M <= 48) return go(integral_constant<int, 3>{}, integral_constant<int, 2>{});
  return go(integral_constant<int, 4>{}, integral_constant<int, 2>{});
}

// Bytes of the scales of `rows` rows in whole dwords, to where the next piece of a workspace begins.
int64_t padded_scales(int64_t rows, int K) { return (rows * ((K + 127) / 128 * 4) + 15) / 16 * 16; }

template <int TM, int TN, int WM, int WN, int S, int BITS, bool XMX, bool PARTIAL>
hipError_t launch_mx_tiles(MxArgs g, int splits, hipStream_t stream) {
  constexpr int lds = S * (TM * (XMX ? 132 : 256) + TN * (16 * BITS + 4));
  constexpr auto kernel = linear_mx_tile_kernel<TM, TN, WM, WN, S, BITS, XMX, PARTIAL>;
  g.tiles = Tiles{splits, 1, (int)((g.M + TM - 1) / TM), (int)((g.N + TN - 1) / TN)};
  if constexpr (lds > 65536) {
    const hipError_t e = allow_lds<kernel>(lds);
    if (e != hipSuccess) return e;
  }
  const int slots = resident_slots<kernel>(64 * WM * WN, lds);
  kernel<<<dim3(std::min(slots, g.tiles.total())), dim3(64 * WM * WN), lds, stream>>>(g);
  return hipGetLastError();
}

template <int BITS, bool XMX, bool PARTIAL>
hipError_t launch_mx_cut(const MxArgs &g, const Cut &c, hipStream_t stream) {
  if constexpr (!XMX)
    return c.wide ? launch_mx_tiles<128, 256, 2, 4, BITS == 4 ? 3 : 2, BITS, false, PARTIAL>(g, c.splits, stream)
                  : launch_mx_tiles<128, 128, 4, 2, 3, BITS, false, PARTIAL>(g, c.splits, stream);
  else if (c.wide) return launch_mx_tiles<256, 256, 2, 4, 2, BITS, true, PARTIAL>(g, c.splits, stream);
  else if (c.deep)  // eight waves: 256 x 4096 x 12288 in 4 bits 28.7 us, four 26.5
    return launch_mx_tiles<128, 128, 2, 2, 4, BITS, true, PARTIAL>(g, c.splits, stream);
  else return launch_mx_tiles<128, 128, 2, 2, 2, BITS, true, PARTIAL>(g, c.splits, stream);
}

template <int BITS, bool XMX>
hipError_t launch_mx(const MxArgs &g, hipStream_t stream) {
  const Cut c = mx_cut((int)g.M, (int)g.K, (int)g.N, XMX);
  if (c.splits == 1) return launch_mx_cut<BITS, XMX, false>(g, c, stream);
  const hipError_t e = launch_mx_cut<BITS, XMX, true>(g, c, stream);
  return e != hipSuccess ? e : launch_sum_parts(g.part, g.out, nullptr, c.splits, g.M * g.N / 8, g.M * g.N / 8, stream);
}

}  // namespace

int64_t linear_mx_workspace(int M, int K, int N, bool x_quantised) {
  if (linear_mx_few_rows(M, N)) return 0;
  return (K % 128 ? padded_scales(x_quantised ? M : 0, K) + padded_scales(N, K) : 0) +
         part_bytes(mx_cut(M, K, N, x_quantised), M, N, 1);
}

hipError_t launch_linear_mx(const void *x, const void *x_scales, const void *codes, const void *scales,
                            void *y, void *workspace, int M, int K, int N, int bits, hipStream_t stream) {
  MxArgs g{(const uint8_t *)x, (const uint8_t *)x_scales, (const uint8_t *)codes, (const uint8_t *)scales,
           (bf16 *)y, (float *)workspace, M, N, K, K / 32, {}};
  if (linear_mx_few_rows(M, N))
    return by_types(bits, x_scales != nullptr, [&](auto b, auto xmx) {
      return by_blocks(M, N, [&](auto mb, auto nb) {
        constexpr int NB = decltype(nb)::value;
        linear_mx_rows_kernel<decltype(b)::value, decltype(xmx)::value, decltype(mb)::value, NB>
            <<<dim3((N + 16 * NB - 1) / (16 * NB)), dim3(64 * kRowWaves), 0, stream>>>(
                x, g.x_scales, g.codes, g.scales, g.out, M, K, N);
        return hipGetLastError();
      });
    });
  if (K % 128) {
    const int64_t x_rows = x_scales ? M : 0, rows = x_rows + N;
    uint8_t *xp = (uint8_t *)workspace, *wp = xp + padded_scales(x_rows, K);
    const int dwords = (K + 127) / 128;
    const int64_t blocks = (rows * dwords + 255) / 256;
    pad_scales_kernel<<<dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(256), 0, stream>>>(
        g.x_scales, g.scales, (uint32_t *)xp, (uint32_t *)wp, K / 32, dwords, x_rows, rows);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    g.x_scales = xp, g.scales = wp, g.sld = 4 * dwords, g.part = (float *)(wp + padded_scales(N, K));
  }
  return by_types(bits, x_scales != nullptr, [&](auto b, auto xmx) {
    return launch_mx<decltype(b)::value, decltype(xmx)::value>(g, stream);
  });
}

}  // namespace ttfa
