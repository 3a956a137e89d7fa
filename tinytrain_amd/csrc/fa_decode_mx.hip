// Decode attention over a quantised KV cache (kv_cache_mx.hip describes the format), gfx950: Tq new
// query rows per (batch, head) against a cache of L_b keys in 4 or 8 bits.  The mathematics is that
// of fa_decode.hip (the last Tq rows of the reference's causal attention, model.py:94-98) on the
// values the cache stands for, and so are the split over keys and the merge pass.
//
// Layout: a wave takes blocks of 64 keys, in halves of 32, and 16 or 32 query columns (R = G * Tq <= 32
// of them are real; the others repeat them).  S^T = K Q^T is formed as two tiles of 16 keys a half, tile
// t's row 4q + r being key q + 16t + 4r of it, so that the result (D[i][j] in lane j + 16 * (i / 4), register
// i % 4) leaves lane (j, q) with the scores of keys q + 4e, e = 4t + r, of column j: the B operand of
// O^T += V^T P^T through v_mfma_f32_16x16x32_bf16 as it stands, and every load instruction reads
// whole consecutive rows.
//  * K stays as it lies in the cache: v_mfma_scale_f32_16x16x128_f8f6f4 takes e2m1 or e4m3 elements
//    with one power of two per 32.  Its k index runs, for e2m1, 32 elements in lane i + 16 * (k / 32);
//    for e4m3 the elements 16c .. 16c + 15 and 64 + 16c .. of lane i + 16 c; the scale of elements
//    32c .. 32c + 31 comes from lane i + 16 c (checked element by element on gfx950).  Q is split
//    once into two e4m3 terms, q = hi + lo: a bf16 has 8 significant bits and each term 4, so the sum
//    is exact but for elements below 2^-13 of the row's largest, which lose at most 2^-21 of that.
//    Rows of less than 2^-108, whose powers of two the instruction's scales would not reach, enter it
//    scaled up, and their scores are scaled down with the softmax scale.
//    At D = 64 both terms share one product: k = 0..63 are hi, 64..127 lo, and K is given twice.
//    (K through bf16 conversions took 32 more of about 200 vector instructions a half.)
//    The instruction adds in fp32, but within every eight consecutive products it drops the bits below
//    2^-13 of the largest (seen with pairs of products, in one eight and in two).  A score is off by less than
//    2^-10 of the sum of those largest ones (at a sum of 30, by 0.03 at worst, and LSE by as much), most where
//    one product outweighs its eight; measured, relative to sum |q k|, 2^-22 on average and 2^-16.4 at most
//    of 4096 random scores in 4 bits, 2^-19 and 2^-14.9 in 8 bits.  At sums of a few hundred that is on average
//    below the 2^-8 to which the weights are rounded, and far below what 4 or 8 bits left of K.
//  * V: lane (i, q) loads D / 16 consecutive elements of each of the rows q + 4e, converts each
//    row's to bf16 with that row's scale, and pairs up rows with v_perm, giving the A operands of
//    D / 16 tiles whose row i is d = D / 16 * i + tile.  The scale goes by row, so it cannot move into
//    the product, whose scales go along the keys.
// No LDS in the loop, but for the one case that reads its queries there (below).
//
// What bounds it: up to 16 query columns, memory (1.5 GB of caches in turn: 64 x 8 heads of up to 16384
// keys, 678 MB, 131 us, 5.2 TB/s; 32 x 8 of 4096, 143 MB, 27.8 us, where a kernel of nothing but these loads
// takes 26.8); 17 to 32 columns on few heads, the vector instructions of a block, about 1.2 us for a wave
// (16 x 4 heads of 5000 keys, 32 columns: 18.8 us, 16 columns 15.0, and 8.3 without keys).
#include "decode_split.h"
#include "fa_bwd.h"  // allow_lds
#include "fa_common.h"
#include "fa_kernels.h"
#include "mx.h"

#include <algorithm>

namespace ttfa {

namespace {

constexpr float kMxSlack = 8.0f;
// Running maximum before any key: finite, so that differences from it are no NaN.
constexpr float kMxLowest = -3.402823466e38f;
constexpr int kMxBlock = 64;  // keys per block: two halves of 32
constexpr int kMxMerged = 16;  // partials of a row that one wave merges

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// max / sum over the four lanes j, j + 16, j + 32, j + 48 of a column
__device__ __forceinline__ float quarters_max(float x) {
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xhalf_max(fmax2(__uint_as_float(p[0]), __uint_as_float(p[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xhalf_sum(__uint_as_float(p[0]) + __uint_as_float(p[1]));
}

template <int D, int BITS>
struct MxShape {
  static constexpr int CODE = D * BITS / 8, GR = D / 32;  // bytes of a row: codes, scales
  static constexpr int DT = D / 16;                       // output tiles; V elements of a lane's row
  static constexpr bool PAIRED = D == 64 && BITS == 4;    // a lane's load serves two K tiles / V rows
  static constexpr int KW = D == 128 && BITS == 8 ? 8 : 4;  // words of a lane's K piece
  static constexpr int KL = PAIRED ? 1 : 2, VL = PAIRED ? 4 : 8;  // loads of a half: K tiles, V rows
  static constexpr int VW = D == 128 && BITS == 8 ? 2 : 1;  // words of a V load
};

// What a lane holds of a half block, as it lies in the cache.
//  * K: for tile t its 16 or 32 bytes of row q' + 4 r' + 16 t, where i = 4 q' + r'.  e2m1 at D = 64
//    needs the same two pieces of a row in lanes q and q + 2: the lower half of the wave loads tile
//    0, the upper one tile 1, and they are exchanged at use.
//  * V: D / 16 elements of each of the rows q + 4e; those 2 bytes of e2m1 at D = 64 come as words,
//    an even lane's from row e = 2r, an odd lane's from row 2r + 1, and neighbours exchange halves.
template <int D, int BITS>
struct MxK {
  using P = MxShape<D, BITS>;
  uint32_t x[P::KL][P::KW];
};
template <int D, int BITS>
struct MxV {
  using P = MxShape<D, BITS>;
  uint32_t x[P::VL][P::VW];
};

// Scale bytes of a block: of K row q' + 4 r' + 16 q (tile q of the block's four) and of V row
// q + 4 (i & 7) + 32 (i >> 3).  A block's scales come in two loads of 64 rows each: loads of 32 rows
// at a time took 2 to 4 of 20 us at 64 x 12 caches of D = 64.
struct MxScales {
  uint32_t k, v;
};

// This lane's byte offsets within a half (codes) or a block (scales).
template <int D, int BITS>
struct MxLane {
  using P = MxShape<D, BITS>;
  uint32_t k, v, ks, vs;
  __device__ explicit MxLane(int lane) {
    const int i = lane & 15, q = lane >> 4, row = (i >> 2) + 4 * (i & 3);
    if constexpr (P::PAIRED) {
      k = (row + 16 * (q >> 1)) * P::CODE + 16 * (q & 1);
      v = (q + 4 * (i & 1)) * P::CODE + 4 * (i >> 1);
    } else {
      k = row * P::CODE + 16 * q;
      v = q * P::CODE + i * (P::CODE / 16);
    }
    ks = (row + 16 * q) * P::GR;
    vs = (q + 4 * (i & 7) + 32 * (i >> 3)) * P::GR;
  }
};

struct MxSrc {  // one (batch, KV head) of the cache
  const uint8_t *kc, *ks, *vc, *vs;
};

// Loads of rows past `end` read nothing and give zeros (codes 0 of scale 2^-127: exact zeros).
template <int D, int BITS>
__device__ __forceinline__ void load_k(MxK<D, BITS> &k, const MxSrc &s, const MxLane<D, BITS> &o,
                                       int k0, int end) {
  using P = MxShape<D, BITS>;
  const auto kc = make_rsrc(s.kc + (int64_t)k0 * P::CODE, (uint32_t)max(end - k0, 0) * P::CODE);
#pragma unroll
  for (int t = 0; t < P::KL; ++t)
#pragma unroll
    for (int c = 0; c < P::KW / 4; ++c) {  // e4m3, D = 128: elements 16q .. and 64 + 16q ..
      const u32x4 w = buf_load16(kc, o.k + 16 * t * P::CODE + 64 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) k.x[t][4 * c + e] = w[e];
    }
}

template <int D, int BITS>
__device__ __forceinline__ void load_v(MxV<D, BITS> &v, const MxSrc &s, const MxLane<D, BITS> &o,
                                       int k0, int end) {
  using P = MxShape<D, BITS>;
  const auto vc = make_rsrc(s.vc + (int64_t)k0 * P::CODE, (uint32_t)max(end - k0, 0) * P::CODE);
#pragma unroll
  for (int r = 0; r < P::VL; ++r) {
    const uint32_t at = o.v + (32 / P::VL) * r * P::CODE;
    if constexpr (P::VW == 1) v.x[r][0] = buf_load4(vc, at);
    else {
      const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(vc, at, 0, 0);
      v.x[r][0] = w[0], v.x[r][1] = w[1];
    }
  }
}

template <int D, int BITS>
__device__ __forceinline__ MxScales load_scales(const MxSrc &s, const MxLane<D, BITS> &o, int k0, int end) {
  using P = MxShape<D, BITS>;
  const uint32_t bytes = (uint32_t)max(end - k0, 0) * P::GR;
  const auto ks = make_rsrc(s.ks + (int64_t)k0 * P::GR, bytes);
  const auto vs = make_rsrc(s.vs + (int64_t)k0 * P::GR, bytes);
  if constexpr (P::GR == 4) return {buf_load4(ks, o.ks), buf_load4(vs, o.vs)};
  else
    return {(uint32_t)__builtin_amdgcn_raw_buffer_load_b16(ks, o.ks, 0, 0),
            (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(vs, o.vs, 0, 0)};
}

// x of row (of 16 lanes) T of the wave, in every row, for T = 0..3
__device__ __forceinline__ void spread_rows(uint32_t (&out)[4], uint32_t x) {
  const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const auto p = __builtin_amdgcn_permlane16_swap(h[u], h[u], false, false);
    out[2 * u] = p[0], out[2 * u + 1] = p[1];
  }
}

// x of lane S of each row of 16
template <int S>
__device__ __forceinline__ uint32_t row_bcast(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x150 + S, 0xF, 0xF, true);
}

// Scales of this lane's group in its eight V rows of half U, on the exponent bits (the conversions
// look at nothing else): `turn` rotates the group's byte of a row's there.
template <int U>
__device__ __forceinline__ void v_scales(uint32_t (&sc)[8], uint32_t vs, uint32_t turn) {
  sc[0] = row_bcast<8 * U>(vs), sc[1] = row_bcast<8 * U + 1>(vs);
  sc[2] = row_bcast<8 * U + 2>(vs), sc[3] = row_bcast<8 * U + 3>(vs);
  sc[4] = row_bcast<8 * U + 4>(vs), sc[5] = row_bcast<8 * U + 5>(vs);
  sc[6] = row_bcast<8 * U + 6>(vs), sc[7] = row_bcast<8 * U + 7>(vs);
#pragma unroll
  for (int r = 0; r < 8; ++r) sc[r] = __builtin_amdgcn_alignbit(sc[r], sc[r], turn);
}

// 1 in the slot of every row whose group is NaN, whose scale becomes 2^-127 (its codes are zeros).
__device__ __forceinline__ bf16x8 take_out_nans(uint32_t (&sc)[8]) {
  bf16x8 mark;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const bool nan = (sc[r] & 0x7f800000u) == 0x7f800000u;
    mark[r] = (bf16)(nan ? 1.f : 0.f);
    sc[r] = nan ? 0 : sc[r];
  }
  return mark;
}

// The words v_pair takes.  PAIRED: even lanes take the low halves of their own row's word and their
// neighbour's, odd lanes the high halves of the neighbour's and their own: row 2r's elements, then
// row 2r + 1's.
template <int D, int BITS>
__device__ __forceinline__ MxV<D, BITS> v_words(const MxV<D, BITS> &v, int lane) {
  using P = MxShape<D, BITS>;
  MxV<D, BITS> out;
  // bytes of (neighbour's word, own word) = bytes (7..4, 3..0)
  const uint32_t halves = lane & 1 ? 0x03020706u : 0x05040100u;
#pragma unroll
  for (int r = 0; r < P::VL; ++r)
#pragma unroll
    for (int w = 0; w < P::VW; ++w) {
      const uint32_t own = v.x[r][w];
      if constexpr (P::PAIRED) {
        const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xF, 0xF, true);
        out.x[r][w] = __builtin_amdgcn_perm(other, own, halves);
      } else {
        out.x[r][w] = own;
      }
    }
  return out;
}

// A operands of output tiles 2W and 2W + 1: slot r = V[key q + 4r][d = DT * i + 2W, + 1]
template <int D, int BITS, int W>
__device__ __forceinline__ void v_pair(bf16x8 &even, bf16x8 &odd, const MxV<D, BITS> &v,
                                       const uint32_t (&sc)[8]) {
  using P = MxShape<D, BITS>;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const float scale = __uint_as_float(sc[r]);
    bf16x2 y;
    if constexpr (P::PAIRED)
      y = r & 1 ? mx_values2<4, W + 2>(v.x[r / 2][0], scale) : mx_values2<4, W>(v.x[r / 2][0], scale);
    else if constexpr (BITS == 4) y = mx_values2<4, W>(v.x[r % P::VL][0], scale);
    else y = mx_values2<8, W & 1>(v.x[r % P::VL][W >> 1], scale);
    even[r] = y[0], odd[r] = y[1];
  }
}

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The query rows of a workgroup in LDS: per row D bytes of hi, then D bytes of lo, in 16-byte pieces
// whose place is turned by the row (a fragment read takes the same piece of 16 rows), and the rows'
// exponents e + 127: -8 (subnormals) to 247, or 255 for a row with a NaN or an infinity.  The product
// takes a lower one than kLeastExp as that, whose lo term, 4 below, is then in reach too.
constexpr int kLeastExp = 10;

template <int D>
__device__ __forceinline__ uint8_t *query_piece(uint8_t *rows, int row, int piece) {
  return rows + row * 2 * D + ((piece ^ (row & (D / 8 - 1))) << 4);
}

// x / scale, y / scale as e4m3 in half H of a word
template <int H>
__device__ __forceinline__ s16x2 put_fp8(uint32_t word, float x, float y, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(__builtin_bit_cast(s16x2, word), x, y, scale, H);
}

// Splits the workgroup's query rows into e4m3 terms; a lane takes eight elements, N times.
template <int D, int N>
__device__ __forceinline__ void split_queries(const u32x4 (&q)[N], int n_rows, uint8_t *rows,
                                              int16_t *exps, int threads) {
  constexpr int LPR = D / 8;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int at = threadIdx.x + j * threads;
    if (at >= n_rows * LPR) break;  // whole rows, so whole groups of lanes
    const u32x4 w = q[j];
    u16x2 m{};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    uint32_t top = (uint32_t)max(m[0], m[1]) << 16;
    auto with = [&](auto dpp) {
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, decltype(dpp)::value, 0xF, 0xF,
                                                           true));
    };
    with(std::integral_constant<int, 0xB1>{});   // lane ^ 1
    with(std::integral_constant<int, 0x4E>{});   // lane ^ 2
    with(std::integral_constant<int, 0x141>{});  // mirrored in eight
    if constexpr (LPR == 16) with(std::integral_constant<int, 0x140>{});  // in sixteen
    // As mx_scale_byte<8>, not clamped: no cache value has to hold these.
    const int e = (int)((top + (0x7fffff - 0x680000)) >> 23) - 8;
    const int exp = top >= 0x7f800000u ? 255 : e;
    u32x2 hi{}, lo{};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y0 = __builtin_ldexpf(__uint_as_float(w[i] << 16), 127 - exp);
      const float y1 = __builtin_ldexpf(__uint_as_float(w[i] & 0xffff0000u), 127 - exp);
      const uint32_t h_old = hi[i >> 1], l_old = lo[i >> 1];
      const s16x2 h = i & 1 ? put_fp8<1>(h_old, y0, y1, 1.f) : put_fp8<0>(h_old, y0, y1, 1.f);
      hi[i >> 1] = __builtin_bit_cast(uint32_t, h);
      const uint32_t code = hi[i >> 1];
      const f32x2 v = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code, 1.f, 1)
                            : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code, 1.f, 0);
      const s16x2 l = i & 1 ? put_fp8<1>(l_old, y0 - v[0], y1 - v[1], 0x1p-4f)
                            : put_fp8<0>(l_old, y0 - v[0], y1 - v[1], 0x1p-4f);
      lo[i >> 1] = __builtin_bit_cast(uint32_t, l);
    }
    const int row = at / LPR, part = at % LPR;
    *reinterpret_cast<u32x2 *>(query_piece<D>(rows, row, part >> 1) + 8 * (part & 1)) = hi;
    *reinterpret_cast<u32x2 *>(query_piece<D>(rows, row, D / 16 + (part >> 1)) + 8 * (part & 1)) = lo;
    if (part == 0) exps[row] = (int16_t)exp;
  }
}

// One column's query row as a lane holds it: the B operands (D = 64: hi and lo in one) and the bytes of
// their powers of two.
template <int D>
struct MxQuery {
  static constexpr int N = D / 64;
  i32x8 t[N];
  int scale[N];

  __device__ __forceinline__ void read(uint8_t *rows, const int16_t *exps, int row, int q4) {
    // D = 128: elements 16 q .. and 64 + 16 q .. of each term; D = 64: 16 q .. of both
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(query_piece<D>(rows, row, 8 * n + 4 * r + q4));
#pragma unroll
        for (int e = 0; e < 4; ++e) t[n][4 * r + e] = (int)w[e];
      }
    const int hi = max((int)exps[row], kLeastExp), lo = hi == 255 ? 255 : hi - 4;  // 255: the row is NaN
    if constexpr (D == 128) scale[0] = hi, scale[1] = lo;
    else scale[0] = q4 < 2 ? hi : lo;
  }
};

// A operands of a half's two K tiles
template <int D, int BITS>
__device__ __forceinline__ void k_operands(i32x8 (&a)[2], const MxK<D, BITS> &k) {
  using P = MxShape<D, BITS>;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    a[t] = i32x8{};
#pragma unroll
    for (int w = 0; w < P::KW; ++w) a[t][w] = (int)k.x[t % P::KL][w];
    if constexpr (D == 64 && BITS == 8) {
#pragma unroll
      for (int w = 0; w < 4; ++w) a[t][4 + w] = (int)k.x[t][w];
    }
  }
  if constexpr (P::PAIRED) {
#pragma unroll
    for (int w = 0; w < P::KW; ++w) {
      const auto p = __builtin_amdgcn_permlane32_swap(k.x[0][w], k.x[0][w], false, false);
      a[0][w] = (int)p[0], a[1][w] = (int)p[1];
    }
  }
}

// S^T tile of one column tile; `scale`: byte 0 is that of the row's group q (D = 64: q & 1)
template <int D, int BITS>
__device__ __forceinline__ f32x4 scores(i32x8 a, uint32_t scale, const MxQuery<D> &q) {
  constexpr int type = BITS == 4 ? 4 : 0;  // e2m1, e4m3
  f32x4 s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q.t[0], f32x4{}, type, 0, 0, (int)scale, 0,
                                                             q.scale[0]);
  if constexpr (D == 128)
    s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q.t[1], s, type, 0, 0, (int)scale, 0,
                                                         q.scale[1]);
  return s;
}

// x - y, not fused with the product that x comes from
__device__ __forceinline__ float minus(float x, float y) {
#pragma clang fp contract(off)
  return x - y;
}

// Whether one of the row's scale bytes is 255 (a NaN group)
__device__ __forceinline__ bool any_nan_scale(uint32_t bytes) {
  const uint32_t x = ~bytes;  // has a zero byte?
  return (x - 0x01010101u) & ~x & 0x80808080u;
}

}  // namespace

// Grid: (B * Hkv units, n_chunks), workgroups of NW waves; NC tiles of 16 query columns.  Partial rows
// are indexed as q's, each with n_chunks slots.
template <int D, int BITS, int NW, int NC, bool SPLIT>
__global__ __launch_bounds__(64 * NW, 2) void fa_decode_mx_kernel(
    const bf16 *Q, KvCache cache, const int *__restrict__ cache_seqlens,
    bf16 *__restrict__ O, float *__restrict__ LSE, float *__restrict__ part_o,
    float *__restrict__ part_ml, Divisor units, Divisor heads, int G, Divisor new_rows, int Lmax,
    int n_chunks, int log2_min, int turn_units, float scale_log2) {
  using P = MxShape<D, BITS>;
  constexpr int DT = P::DT, COLS = 16 * NC;
  // first the query rows' terms, in the end per wave the partial rows of min(R, 16) columns
  extern __shared__ __attribute__((aligned(16))) float stage[];
  __shared__ float wm[NW][COLS], wsum[NW][COLS];
  __shared__ int16_t query_exps[COLS];
  uint8_t *query_rows = reinterpret_cast<uint8_t *>(stage);
  // The way to the first loads has no branches, and neither have they: a load behind one would have to
  // be waited for before the query rows, which come first.
  const int chunk = SPLIT ? blockIdx.y : 0;
  uint32_t bhk = blockIdx.x;
  if (SPLIT) {
    bhk += chunk * turn_units;
    bhk -= units.quotient(bhk) * units.n;
  }
  const int b = (int)heads.quotient(bhk), Tq = (int)new_rows.n, R = G * Tq;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int i16 = lane & 15, q4 = lane >> 4;
  const int64_t row0 = (int64_t)bhk * R;  // the unit's rows of q, O and the partials follow each other
  constexpr int NQ = (COLS * D / 8 + 64 * NW - 1) / (64 * NW);
  const auto q_rows = make_rsrc(Q + row0 * D, (uint32_t)(R * D) * sizeof(bf16));
  u32x4 q[NQ];
#pragma unroll
  for (int j = 0; j < NQ; ++j) q[j] = buf_load16(q_rows, 16 * (threadIdx.x + j * 64 * NW));
  asm volatile("" ::: "memory");  // keeps them here: they are used behind a branch

  // Rows past the capacity were dropped: their keys are missing, the queries' positions stay.
  const int len = max(cache_seqlens[b], 0), L = min(len, Lmax);
  const int nb = (L + kMxBlock - 1) / kMxBlock;
  const int used = SPLIT ? used_chunks(nb, n_chunks, log2_min) : 1, step = used * NW;
  const int blk0 = chunk * NW + wave, end = !SPLIT || chunk < used ? L : 0;
  // The next block's K is loaded into the registers of this one's once its scores are formed, its V
  // once this one's is added, its scales before both.
  const int64_t slab = (int64_t)bhk * Lmax;
  const MxSrc src{cache.codes[0] + slab * P::CODE, cache.scales[0] + slab * P::GR,
                  cache.codes[1] + slab * P::CODE, cache.scales[1] + slab * P::GR};
  const MxLane<D, BITS> off(lane);
  MxK<D, BITS> kx[2];
  MxV<D, BITS> vx[2];
  __builtin_amdgcn_sched_barrier(0);  // in this order: the waits count on it
  MxScales sc = load_scales(src, off, blk0 * kMxBlock, end);
#pragma unroll
  for (int u = 0; u < 2; ++u) load_k(kx[u], src, off, blk0 * kMxBlock + 32 * u, end);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < 2; ++u) load_v(vx[u], src, off, blk0 * kMxBlock + 32 * u, end);
  __builtin_amdgcn_sched_barrier(0);
  if (SPLIT && chunk >= used) {  // an empty partial, whose O the merge does not read
    if (threadIdx.x < R)
      *reinterpret_cast<f32x2 *>(part_ml + ((row0 + threadIdx.x) * n_chunks + chunk) * 2) =
          f32x2{-INFINITY, 0.f};
    return;
  }
  split_queries<D>(q, R, query_rows, query_exps, 64 * NW);
  __syncthreads();

  f32x4 oacc[NC][DT];
  float m_t[NC], l_part[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m_t[c] = kMxLowest, l_part[c] = 0.f;
#pragma unroll
    for (int n = 0; n < DT; ++n) oacc[c][n] = f32x4{};
  }

  if (blk0 < nb) {
    // 32 columns of 8 bits at D = 128 read their query rows again for every block, one tile's at a
    // time: held, those 36 registers push others to scratch (16 x 4 units of 5000 keys 28.6 us, read
    // again 23.7; 64 x 4 uneven ones 64.7 and 54.4).
    constexpr bool kReread = NC == 2 && D == 128 && BITS == 8;
    MxQuery<D> query[NC];
    int pos[NC];  // last key that this lane's query column of a tile sees; none past the cache
    float scale[NC];  // of its scores, in log2 units
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = min(16 * c + i16, R - 1);  // columns past the last repeat it
      pos[c] = min(len - Tq + col - (int)new_rows.quotient((uint32_t)col) * Tq, L - 1);
      scale[c] = __builtin_ldexpf(scale_log2, min((int)query_exps[col] - kLeastExp, 0));
      if (!kReread) query[c].read(query_rows, query_exps, col, q4);
    }
    // rotates byte g of a row's scale bytes to bits 30:23
    const uint32_t turn = (8 * (i16 * P::GR / 16) + 9) & 31;
    const int first_masked = min(len - Tq, L - 1);  // keys past this need the mask for some column

    const uint32_t kshift = 8 * (q4 & (P::GR - 1));  // brings the byte of this lane's K group down

#pragma unroll 1
    for (int blk = blk0; blk < nb; blk += step) {
      const int k0 = blk * kMxBlock, kn = k0 + step * kMxBlock;
      uint32_t ks[4];
      spread_rows(ks, sc.k);
      const uint32_t vs = sc.v;
      sc = load_scales(src, off, kn, L);
      f32x4 s[NC][4];  // of keys k0 + q + 4 (4t + r)
      if constexpr (kReread) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          asm volatile("" ::: "memory");  // keeps the reads inside the loop, one tile's at a time
          query[0].read(query_rows, query_exps, min(16 * c + i16, R - 1), q4);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            i32x8 a[2];
            k_operands<D, BITS>(a, kx[u]);
#pragma unroll
            for (int t = 0; t < 2; ++t)
              s[c][2 * u + t] = scores<D, BITS>(a[t], ks[2 * u + t] >> kshift, query[0]);
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(s[c][t]));  // formed here, not at first use
        }
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          i32x8 a[2];
          k_operands<D, BITS>(a, kx[u]);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c)
              s[c][2 * u + t] = scores<D, BITS>(a[t], ks[2 * u + t] >> kshift, query[c]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 2; ++u) load_k(kx[u], src, off, kn + 32 * u, L);
      __builtin_amdgcn_sched_barrier(0);

      const bool masked = k0 + kMxBlock - 1 > first_masked;
      bf16x8 pb[NC][2];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        // Scaled before the maximum is taken off, each with its own rounding: fused, the largest
        // score's rounding error would be left there, an exponent of any size for scores past 2^30
        // (0 to 1% of a call's time).
#pragma unroll
        for (int e = 0; e < 16; ++e) s[c][e >> 2][e & 3] *= scale[c];
        if (masked) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (k0 + q4 + 4 * e > pos[c]) s[c][e >> 2][e & 3] = -INFINITY;
        }
        float mx = max16(f32x16{s[c][0][0], s[c][0][1], s[c][0][2], s[c][0][3], s[c][1][0], s[c][1][1],
                                s[c][1][2], s[c][1][3], s[c][2][0], s[c][2][1], s[c][2][2], s[c][2][3],
                                s[c][3][0], s[c][3][1], s[c][3][2], s[c][3][3]}, -INFINITY);
        mx = quarters_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m_t[c] + kMxSlack)) {
          // each column by itself: its bits do not depend on when others rescale
          const float m_new = mx > m_t[c] + kMxSlack ? mx : m_t[c];
          const float alpha = exp2f_fast(m_t[c] - m_new);  // 0 from the lowest; 1 if unchanged
          m_t[c] = m_new;
          l_part[c] *= alpha;
#pragma unroll
          for (int n = 0; n < DT; ++n) oacc[c][n] *= alpha;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float p[8], rs = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] = exp2f_fast(minus(s[c][2 * u + (e >> 2)][e & 3], m_t[c]));
            rs += p[e];
          }
          l_part[c] += rs;
          // The weights are rounded to bf16, as the product takes them beside V, whose values are bf16
          // exactly: up to 2^-8 of each, which averages out over the keys; their sum is fp32 of the unrounded.
          const bf16x4 lo = pack4(p[0], p[1], p[2], p[3]), hi = pack4(p[4], p[5], p[6], p[7]);
          pb[c][u] = bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
      }
      // Where rows see different keys (several new rows), a NaN group of a key that a row does not
      // see must not reach it through 0 * NaN: those blocks count the NaN keys that each row sees,
      // make NaN what they add to, and go on without them.
      const bool nans = masked && Tq > 1 && __builtin_amdgcn_ballot_w64(any_nan_scale(vs));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t vsc[8];
        if (u == 0) v_scales<0>(vsc, vs, turn);
        else v_scales<1>(vsc, vs, turn);
        if (nans) {
          int key = k0 + 32 * u + q4;
          asm volatile("" : "+v"(key));  // keeps this block's comparisons in it
          const bf16x8 mark = take_out_nans(vsc);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            bf16x8 seen;
#pragma unroll
            for (int e = 0; e < 8; ++e) seen[e] = (bf16)(key + 4 * e > pos[c] ? 0.f : 1.f);
            const f32x4 count = mfma16(mark, seen, f32x4{});
#pragma unroll
            for (int n = 0; n < DT; ++n)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (count[r] > 0.f) oacc[c][n][r] = __builtin_nanf("");
          }
        }
        const MxV<D, BITS> v = v_words(vx[u], lane);
        auto add = [&](auto w) {
          constexpr int W = decltype(w)::value;
          bf16x8 even, odd;
          v_pair<D, BITS, W>(even, odd, v, vsc);
#pragma unroll
          for (int c = 0; c < NC; ++c) oacc[c][2 * W] = mfma16(even, pb[c][u], oacc[c][2 * W]);
#pragma unroll
          for (int c = 0; c < NC; ++c) oacc[c][2 * W + 1] = mfma16(odd, pb[c][u], oacc[c][2 * W + 1]);
        };
        add(std::integral_constant<int, 0>{});
        add(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
          add(std::integral_constant<int, 2>{});
          add(std::integral_constant<int, 3>{});
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 2; ++u) load_v(vx[u], src, off, kn + 32 * u, L);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Merge of the workgroup's waves, as in fa_decode.hip: every wave scales its partial to the
  // workgroup's running max and stages it as fp32 rows, then the threads add the waves in order.
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float l = quarters_sum(l_part[c]);
    if (q4 == 0) {
      // A wave without visible keys (l exactly 0) weighs nothing; the NaN of one that saw a NaN score
      // goes on through the maximum and the weights.
      wm[wave][16 * c + i16] = l == 0.f ? -INFINITY : l == l ? m_t[c] : l;
      wsum[wave][16 * c + i16] = l;
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = 16 * c + i16, cols = min(R - 16 * c, 16);  // cols > 0: R > 16 where NC is 2
    const int rows = min(R, 16);
    if (c) __syncthreads();  // the first tile's rows are read
    float M = wm[0][col];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmax2(M, wm[w][col]);
    const float mw = wm[wave][col], alpha = mw == -INFINITY ? 0.f : exp2f_fast(mw - M);
    if (i16 < cols) {
      // register r of tile n is d = DT * (4 * q4 + r) + n: DT consecutive ones per r
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < DT; n += 4) {
          const int ch = (DT * (4 * q4 + r) + n) / 4;
          *reinterpret_cast<f32x4 *>(&stage[(wave * rows + i16) * D + ((ch ^ (i16 & 7)) << 2)]) =
              alpha != 0.f ? f32x4{oacc[c][n][r] * alpha, oacc[c][n + 1][r] * alpha,
                                   oacc[c][n + 2][r] * alpha, oacc[c][n + 3][r] * alpha}
                           : f32x4{};
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < cols * (D / 4); e += 64 * NW) {
      const int j = e / (D / 4), ch = e % (D / 4), k = 16 * c + j;
      f32x4 t{};
      float mx = wm[0][k], ls = 0.f;
#pragma unroll
      for (int w = 1; w < NW; ++w) mx = fmax2(mx, wm[w][k]);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        t += *reinterpret_cast<const f32x4 *>(&stage[(w * rows + j) * D + ((ch ^ (j & 7)) << 2)]);
        ls += wm[w][k] == -INFINITY ? 0.f : wsum[w][k] * exp2f_fast(wm[w][k] - mx);
      }
      const int64_t row = row0 + k;
      if (!SPLIT) {
        const float inv = ls == 0.f ? 0.f : 1.f / ls;  // NaN sums reach O and LSE
        *reinterpret_cast<bf16x4 *>(O + row * D + 4 * ch) =
            pack4(t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv);
        if (ch == 0) LSE[row] = ls == 0.f ? -INFINITY : (mx + __log2f(ls)) * kLn2;
      } else {
        const int64_t slot = row * n_chunks + chunk;
        *reinterpret_cast<f32x4 *>(part_o + slot * D + 4 * ch) = t;
        if (ch == 0) *reinterpret_cast<f32x2 *>(part_ml + slot * 2) = f32x2{mx, ls};
      }
    }
  }
}

// Merge of up to kMxMerged partials per query row (fa_decode_combine_kernel's rule), a wave per row: lane c
// sums D / 64 columns over the partials in order, all of whose loads go out at once.
template <int D>
__global__ __launch_bounds__(256) void fa_decode_mx_merge_kernel(const float *__restrict__ part_o,
                                                                 const float *__restrict__ part_ml,
                                                                 bf16 *__restrict__ O,
                                                                 float *__restrict__ LSE, int rows,
                                                                 int n_splits) {
  typedef float vec __attribute__((ext_vector_type(D / 64)));
  const int row = blockIdx.x * 4 + wave_id(), lane = threadIdx.x & 63;
  if (row >= rows) return;
  const f32x2 *ml = reinterpret_cast<const f32x2 *>(part_ml) + (int64_t)row * n_splits;
  const vec *po = reinterpret_cast<const vec *>(part_o + (int64_t)row * n_splits * D) + lane;
  const f32x2 mine = lane < n_splits ? ml[lane] : f32x2{-INFINITY, 0.f};
  vec x[kMxMerged];
#pragma unroll
  for (int s = 0; s < kMxMerged; ++s)
    if (s < n_splits) x[s] = po[s * 64];
  float M = mine[1] != 0.f ? mine[0] : -INFINITY;
#pragma unroll
  for (int m = 1; m < kMxMerged; m <<= 1) M = fmax2(M, __shfl_xor(M, m));
  M = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(M)));
  const float w = mine[1] != 0.f ? exp2f_fast(mine[0] - M) : 0.f;
  float sum = w * mine[1];
#pragma unroll
  for (int m = 1; m < kMxMerged; m <<= 1) sum += __shfl_xor(sum, m);
  sum = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(sum)));
  vec acc{};
#pragma unroll
  for (int s = 0; s < kMxMerged; ++s) {
    const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
    // an unused chunk wrote no O
    if (s < n_splits && ws != 0.f) {
#pragma unroll
      for (int e = 0; e < D / 64; ++e) acc[e] = __builtin_fmaf(x[s][e], ws, acc[e]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < D / 64; ++e) O[(int64_t)row * D + lane * (D / 64) + e] = (bf16)(acc[e] * inv);
  if (lane == 0) LSE[row] = sum == 0.f ? -INFINITY : (M + __log2f(sum)) * kLn2;
}

// Workgroups per unit and the blocks that one takes at least; four waves each.  Times in us
// back to back, caches rotated through 1.5 GB, D 128, 4 bits and full caches unless said; "uneven" is
// lengths from a tenth of the capacity up.
//  * One chunk, and one launch, up to 768 keys, or 1024 where there would be two chunks (8 units of 768
//    keys: 6.9, two launches 7.6; of 1000: 8.0, 7.6; 64 of 768: 7.3, 8.0; 128 of 1000: 8.4, 9.2; of 1500:
//    11.0, 10.9; 32 columns, 8 units of 768: 10.2, 9.8).  A call by itself gains 3 us more on the host.
//  * Otherwise as many as stay within 256 workgroups, one per CU, of at least a block per wave:
//      96 units of 3000 keys: 2 chunks 14.3, 1 17.1, 3 16.1; 160 units: 1 16.6, 2 20.8, 3 18.6;
//      256 of 4096: 1 27.8, 2 30.6; 48 of 3000: 5 chunks 10.8, 2 13.5, 11 12.9;
//      8 of 16384: 32 chunks 10.3, 16 11.7, 64 11.5; 8 of 131072: 32 32.6, 16 43.4, 64 32.7.
//    More than kMxMerged chunks need the slower merge, which pays from 32768 elements a chunk (8 units
//    of 8192: 32 chunks 8.6, 16 9.3; 12 units of 8000, D 64: 21 chunks 9.0, 16 7.6).
//  * A long cache among short ones: with several sequences and a capacity over 4096, chunks of about
//    2048 keys, up to 4096 workgroups (16 caches of 8 heads, one of 16384, the others of 300: 8 chunks
//    19.5, 2 38.4; full and uneven calls lose nothing: 64 x 8 of up to 16384: 8 chunks 131, 1 133).
//  * A chunk's least is its share of a full cache, so that short caches cost one workgroup each; with up
//    to 32 units, which leave the device idle, a block for every wave.
DecodeSplit decode_mx_split(int B, int Hkv, int Lmax, int D) {
  const int64_t units = (int64_t)B * Hkv;
  const int64_t blocks = ((int64_t)Lmax + kMxBlock - 1) / kMxBlock;
  int64_t n = std::max<int64_t>(256 / units, 1);
  if (n > kMxMerged && (int64_t)Lmax * D < n * 32768) n = kMxMerged;
  if (B > 1 && Lmax > 4096) {
    const int64_t even = std::min(blocks / 32, 4096 / units);  // chunks of 2048 keys
    n = std::max(n, even);
  }
  n = std::min(n, (blocks + 3) / 4);
  n = std::min<int64_t>(n, 512);
  if (blocks <= 12 || (n == 2 && blocks <= 16)) n = 1;
  if (n <= 1) return {4, 1, 0};
  const int64_t least = units <= 32 ? 4 : (blocks + n - 1) / n;
  int log2_min = 0;
  while (least >> (log2_min + 1)) ++log2_min;
  return {4, (int)n, log2_min};
}

namespace {

// Waves of a one-chunk call: four, or eight, which halve a long cache's time where a CU has one
// workgroup, and keep fewer caches on the device at once where it has several.  Times of eight waves
// against four, uneven caches, then full ones:
//  * up to 256 units, rows of 64 bytes or less: from 24 blocks on, which calls of 129 units or more have in
//    one chunk (192 units, D 128, 4 bits: 600 keys 0.94, 1.01; 1000 1.01, 0.97; 1500 0.98, 0.94; 4000 0.89,
//    0.94; 132, 144 and 256 units, uneven: 1536 0.97; 2000 0.94 to 0.95; 4000 0.90 to 0.93); with 32 columns
//    from 9 on, whose vector instructions then come in shorter runs (64 units, 512 keys 0.94; 768 0.91; 192,
//    600 0.92; 520 to 768 keys of 1 to 128 units: D 128, 4 bits 0.89 to 0.92, D 64 0.94 to 0.97).  Rows of 128
//    bytes have enough on the way with four (192 units: 1500 1.09, 1.09; 4000 1.05, 1.03).
//  * up to 447 units: from 32 blocks on (320 units: 600 keys 1.29, 1.25; 1000 1.11, 1.16; 2000 0.90, 1.08;
//    4000 0.88, 1.05; 8 bits: 1000 1.01, 1.15; 2000 0.89, 1.06; 4000 0.87, 1.03; 32 columns: 600 1.38,
//    2000 1.03, 4000 0.86).
//  * more: four (448 units of 3000: 0.94, 1.03; 1024 of 1500: 1.17, 1.08; 512 of 2000, 32 columns 1.11).
int one_chunk_waves(int64_t units, int Lmax, int row_bytes, bool wide) {
  const int blocks = (Lmax + kMxBlock - 1) / kMxBlock;
  if (units <= 256) return row_bytes <= 64 && blocks >= (wide ? 9 : 24) ? 8 : 4;
  return units < 448 && blocks >= 32 ? 8 : 4;
}

// Places by which a chunk turns its units against the chunk before it (units are the grid's width, its
// chunks follow each other).  Consecutive workgroups go to the XCDs in turn, and those of an XCD to its
// 32 CUs: without a turn every chunk of a unit would share an XCD, or a CU, where the number of units is
// a multiple of 8 (or 256), and a long cache would be read by few (16 caches of 8 heads, one of 16384
// keys: 52 us without, 23 with).  37 = 4 * 8 + 5 moves a unit's chunks to other XCDs and other CUs.
// fa_decode.hip turns by the chunk's number, fewer than 32 units by its last three bits.
int chunk_turn(int units) { return (units >= 64 ? 37 : 5) % units; }

struct MxCall {
  const bf16 *q;
  KvCache cache;
  const int *cache_seqlens;
  bf16 *o;
  float *lse, *workspace;
  int B, Hq, Hkv, Tq, Lmax;
  DecodeSplit sp;
  float scale_log2;
  hipStream_t stream;
};

template <int D, int BITS, int NW, int NC, bool SPLIT>
hipError_t launch_waves(const MxCall &a) {
  const int rows = a.B * a.Hq * a.Tq, cols = a.Hq / a.Hkv * a.Tq, n = a.sp.n_chunks;
  float *part_o = a.workspace, *part_ml = a.workspace + (int64_t)rows * n * D;
  constexpr size_t most = NW * 16 * D * sizeof(float);
  const size_t lds = most * (cols < 16 ? cols : 16) / 16;
  // the kernel's static arrays come on top of the dynamic stages
  if (lds + 2 * NW * 16 * NC * sizeof(float) > 65536) {
    hipError_t e = allow_lds<fa_decode_mx_kernel<D, BITS, NW, NC, SPLIT>>(most);
    if (e != hipSuccess) return e;
  }
  const int units = a.B * a.Hkv;
  const dim3 grid((unsigned)units, (unsigned)n), block(64 * NW);
  fa_decode_mx_kernel<D, BITS, NW, NC, SPLIT><<<grid, block, lds, a.stream>>>(
      a.q, a.cache, a.cache_seqlens, a.o, a.lse, part_o, part_ml, Divisor(units), Divisor(a.Hkv),
      a.Hq / a.Hkv, Divisor(a.Tq), a.Lmax, n, a.sp.log2_min, units - chunk_turn(units), a.scale_log2);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !SPLIT) return e;
  if (n > kMxMerged) return launch_decode_combine(part_o, part_ml, a.o, a.lse, rows, n, D, a.stream);
  fa_decode_mx_merge_kernel<D><<<dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, a.stream>>>(
      part_o, part_ml, a.o, a.lse, rows, n);
  return hipGetLastError();
}

template <int D, int BITS, int NC>
hipError_t launch_shape(const MxCall &a) {
  if (a.sp.n_chunks > 1) return launch_waves<D, BITS, 4, NC, true>(a);
  if (a.sp.n_waves == 8) return launch_waves<D, BITS, 8, NC, false>(a);
  return launch_waves<D, BITS, 4, NC, false>(a);
}

}  // namespace

hipError_t launch_decode_mx(const void *q, const KvCache &cache, const int *cache_seqlens, void *o,
                            float *lse, float *workspace, int B, int Hq, int Hkv, int Tq, int Lmax,
                            int D, int bits, float scale, hipStream_t stream) {
  MxCall a{(const bf16 *)q, cache, cache_seqlens, (bf16 *)o, lse, workspace, B, Hq, Hkv, Tq,
           Lmax, decode_mx_split(B, Hkv, Lmax, D), scale * kLog2e, stream};
  const bool wide = Hq / Hkv * Tq > 16;
  if (a.sp.n_chunks == 1) a.sp.n_waves = one_chunk_waves((int64_t)B * Hkv, Lmax, D * bits / 8, wide);
  if (D == 64) {
    if (bits == 4) return wide ? launch_shape<64, 4, 2>(a) : launch_shape<64, 4, 1>(a);
    return wide ? launch_shape<64, 8, 2>(a) : launch_shape<64, 8, 1>(a);
  }
  if (bits == 4) return wide ? launch_shape<128, 4, 2>(a) : launch_shape<128, 4, 1>(a);
  return wide ? launch_shape<128, 8, 2>(a) : launch_shape<128, 8, 1>(a);
}

}  // namespace ttfa
