// Decode attention over a quantised KV cache (kv_cache_mx.hip describes the format), gfx950: Tq new
// query rows per (batch, head) against a cache of L_b keys in 4 or 8 bits.  The mathematics is that
// of fa_decode.hip (the last Tq rows of the reference's causal attention, model.py:94-98) on the
// values the cache stands for, and so are the split over keys and the merge pass.
//
// Layout: a wave takes 32 keys at a time and 16 or 32 query columns (R = G * Tq <= 32 of them are
// real; the others repeat them) through v_mfma_f32_16x16x32_bf16,
//      A[i][k] in lane i + 16 * (k / 8), slot k % 8      (16 rows, 32 deep)
//      B[k][j] in lane j + 16 * (k / 8), slot k % 8
//      D[i][j] in lane j + 16 * (i / 4), register i % 4,
// chosen over the 32x32 shape because a lane then holds a quarter of a K row: at D = 128 exactly one
// group of 32 with its one scale, loaded straight into registers.  S^T = K Q^T is formed as two
// tiles t whose row 4q + r is key 8q + 4t + r of the block.  Lane (j, q) then ends up with the
// scores of keys 8q .. 8q + 7 of column j, which is the B operand of O^T += V^T P^T as it stands.
// Its A operand has keys 8q .. 8q + 7 of one d in lane (i, q): the lane loads D / 16 consecutive
// elements of each of the eight rows, converts each row's with that row's scale, and pairs up
// rows with v_perm, giving D / 16 tiles whose row i is d = D / 16 * i + tile.  No LDS in the loop.
#include "fa_common.h"
#include "fa_kernels.h"
#include "mx.h"

namespace ttfa {

namespace {

constexpr float kMxSlack = 8.0f;
constexpr int kMxBlock = 32;  // keys per block

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
  static constexpr int KS = D / 32;                       // products of a score tile
  static constexpr int DT = D / 16;                       // output tiles; V elements of a lane's row
  static constexpr int KW = CODE / 16;                    // words of a lane's K quarter row
  static constexpr int VB = CODE / 16;                    // bytes of a lane's V row piece
};

// What a lane holds of one block: its quarter row of each K tile and its piece of eight V rows, as
// they lie in the cache.
template <int D, int BITS>
struct MxBlock {
  using P = MxShape<D, BITS>;
  uint32_t k[2][P::KW];
  uint32_t v[8][P::VB > 4 ? 2 : 1];
  uint32_t ks[2];  // scale byte of the K piece
  uint32_t vs;     // scale bytes of V row 8q + (i & 7)
};

// This lane's byte offsets within a block.
template <int D, int BITS>
struct MxLane {
  using P = MxShape<D, BITS>;
  uint32_t k, ks, v, vs;
  __device__ explicit MxLane(int lane) {
    const int i = lane & 15, q = lane >> 4, row = 8 * (i >> 2) + (i & 3);
    k = row * P::CODE + q * (P::CODE / 4);
    ks = row * P::GR + q * P::GR / 4;
    v = 8 * q * P::CODE + i * P::VB;
    vs = (8 * q + (i & 7)) * P::GR;
  }
};

struct MxSrc {  // one (batch, KV head) of the cache, L rows of it
  const uint8_t *kc, *ks, *vc, *vs;
  int L;
};

// Loads past row L give zeros (codes 0 of scale 2^-127: exact zeros), so no block needs a bound.
template <int D, int BITS>
__device__ __forceinline__ void load_block(MxBlock<D, BITS> &x, const MxSrc &s,
                                           const MxLane<D, BITS> &o, int k0) {
  using P = MxShape<D, BITS>;
  const uint32_t left = (uint32_t)max(s.L - k0, 0);
  const auto kc = make_rsrc(s.kc + (int64_t)k0 * P::CODE, left * P::CODE);
  const auto ks = make_rsrc(s.ks + (int64_t)k0 * P::GR, left * P::GR);
  const auto vc = make_rsrc(s.vc + (int64_t)k0 * P::CODE, left * P::CODE);
  const auto vs = make_rsrc(s.vs + (int64_t)k0 * P::GR, left * P::GR);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t at = o.k + 4 * t * P::CODE;
    if constexpr (P::KW == 2) {
      const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(kc, at, 0, 0);
      x.k[t][0] = w[0], x.k[t][1] = w[1];
    } else {
#pragma unroll
      for (int c = 0; c < P::KW / 4; ++c) {
        const u32x4 w = buf_load16(kc, at + 16 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e) x.k[t][4 * c + e] = w[e];
      }
    }
    x.ks[t] = __builtin_amdgcn_raw_buffer_load_b8(ks, o.ks + 4 * t * P::GR, 0, 0);
  }
  x.vs = P::GR == 4 ? buf_load4(vs, o.vs) : (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(vs, o.vs, 0, 0);
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const uint32_t at = o.v + r * P::CODE;
    if constexpr (P::VB == 2) x.v[r][0] = __builtin_amdgcn_raw_buffer_load_b16(vc, at, 0, 0);
    else if constexpr (P::VB == 4) x.v[r][0] = buf_load4(vc, at);
    else {
      const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(vc, at, 0, 0);
      x.v[r][0] = w[0], x.v[r][1] = w[1];
    }
  }
}

// x of lane S of each row of 16
template <int S>
__device__ __forceinline__ uint32_t row_bcast(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x150 + S, 0xF, 0xF, true);
}

// Scale of V row S for this lane's group, on the exponent bits (the conversions look at nothing
// else): `turn` rotates the byte of the group there.
template <int S, class Block>
__device__ __forceinline__ uint32_t v_scale(const Block &x, uint32_t turn) {
  const uint32_t sc = row_bcast<S>(x.vs);
  return __builtin_amdgcn_alignbit(sc, sc, turn);
}

// The lane's V piece of row S as bf16 pairs (DT / 2 of them).  CLEAN: values of a NaN group are
// zeros, and mark[S] is 1 for one.
template <int D, int BITS, bool CLEAN, int S>
__device__ __forceinline__ void v_row(bf16x2 (&out)[D / 32], const MxBlock<D, BITS> &x, uint32_t turn,
                                      bf16x8 &mark) {
  uint32_t sc = v_scale<S>(x, turn);
  if constexpr (CLEAN) {
    const bool nan = (sc & 0x7f800000u) == 0x7f800000u;
    mark[S] = (bf16)(nan ? 1.f : 0.f);
    sc = nan ? 0 : sc;
  }
  const float scale = __uint_as_float(sc);
  if constexpr (BITS == 4) {
    out[0] = mx_values2<4, 0>(x.v[S][0], scale);
    out[1] = mx_values2<4, 1>(x.v[S][0], scale);
    if constexpr (D == 128) {
      out[2] = mx_values2<4, 2>(x.v[S][0], scale);
      out[3] = mx_values2<4, 3>(x.v[S][0], scale);
    }
  } else {
    out[0] = mx_values2<8, 0>(x.v[S][0], scale);
    out[1] = mx_values2<8, 1>(x.v[S][0], scale);
    if constexpr (D == 128) {
      out[2] = mx_values2<8, 0>(x.v[S][1], scale);
      out[3] = mx_values2<8, 1>(x.v[S][1], scale);
    }
  }
}

// A operands of all output tiles: tile[n] slot s = V[key 8q + s][d = DT * i + n]
template <int D, int BITS, bool CLEAN>
__device__ __forceinline__ void v_tiles(bf16x8 (&tile)[D / 16], const MxBlock<D, BITS> &x, uint32_t turn,
                                        bf16x8 &mark) {
  bf16x2 a[8][D / 32];
  v_row<D, BITS, CLEAN, 0>(a[0], x, turn, mark);
  v_row<D, BITS, CLEAN, 1>(a[1], x, turn, mark);
  v_row<D, BITS, CLEAN, 2>(a[2], x, turn, mark);
  v_row<D, BITS, CLEAN, 3>(a[3], x, turn, mark);
  v_row<D, BITS, CLEAN, 4>(a[4], x, turn, mark);
  v_row<D, BITS, CLEAN, 5>(a[5], x, turn, mark);
  v_row<D, BITS, CLEAN, 6>(a[6], x, turn, mark);
  v_row<D, BITS, CLEAN, 7>(a[7], x, turn, mark);
#pragma unroll
  for (int n = 0; n < D / 16; ++n)
#pragma unroll
    for (int s = 0; s < 8; ++s) tile[n][s] = a[s][n >> 1][n & 1];
}

// Whether one of the row's scale bytes is 255 (a NaN group)
__device__ __forceinline__ bool any_nan_scale(uint32_t bytes) {
  const uint32_t x = ~bytes;  // has a zero byte?
  return (x - 0x01010101u) & ~x & 0x80808080u;
}

}  // namespace

// Grid: (B * Hkv units, n_chunks), workgroups of NW waves; NC tiles of 16 query columns.  Partial rows
// are indexed (b * Hq + h) * Tq + i, each with n_chunks slots.
template <int D, int BITS, int NW, int NC, bool SPLIT>
__global__ __launch_bounds__(64 * NW) void fa_decode_mx_kernel(
    const bf16 *__restrict__ Q, KvCache cache, const int *__restrict__ cache_seqlens,
    bf16 *__restrict__ O, float *__restrict__ LSE, float *__restrict__ part_o,
    float *__restrict__ part_ml, int B, int Hq, int Hkv, int Tq, int Lmax, int n_chunks, int log2_min,
    float scale_log2) {
  using P = MxShape<D, BITS>;
  constexpr int KS = P::KS, DT = P::DT, COLS = 16 * NC;
  __shared__ __attribute__((aligned(16))) float stage[NW][16 * D];
  __shared__ float wm[NW][COLS], wsum[NW][COLS];
  const int chunk = SPLIT ? blockIdx.y : 0;
  const int bhk = blockIdx.x;
  const int b = bhk / Hkv, hk = bhk - b * Hkv;
  const int G = Hq / Hkv, R = G * Tq;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int i16 = lane & 15, q4 = lane >> 4;
  const int L = min(max(cache_seqlens[b], 0), Lmax);

  const int nb = (L + kMxBlock - 1) / kMxBlock;
  const int used = SPLIT ? max(min((nb + (1 << log2_min) - 1) >> log2_min, n_chunks), 1) : 1;
  const int step = used * NW, blk0 = chunk < used ? chunk * NW + wave : nb;

  // the query columns of this lane, one per tile
  int pos[NC];  // last visible key
  const bf16 *qp[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (16 * c + i16) % R, g = col / Tq, i = col - g * Tq;
    pos[c] = L - Tq + i;
    qp[c] = Q + (((int64_t)b * Hq + hk * G + g) * Tq + i) * D;
  }

  f32x4 oacc[NC][DT];
  float m_t[NC], l_part[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m_t[c] = -INFINITY, l_part[c] = 0.f;
#pragma unroll
    for (int n = 0; n < DT; ++n) oacc[c][n] = f32x4{};
  }

  if (blk0 < nb) {
    bf16x8 qf[NC][KS];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
        qf[c][kk] = *reinterpret_cast<const bf16x8 *>(qp[c] + q4 * (D / 4) + 8 * kk);
    const int64_t slab = (int64_t)bhk * Lmax;
    const MxSrc src{cache.codes[0] + slab * P::CODE, cache.scales[0] + slab * P::GR,
                    cache.codes[1] + slab * P::CODE, cache.scales[1] + slab * P::GR, L};
    const MxLane<D, BITS> off(lane);
    // rotates byte g of a row's scale bytes to bits 30:23
    const uint32_t turn = (8 * (i16 * P::GR / 16) + 9) & 31;
    const int first_masked = L - Tq;  // keys past this need the mask for some column

#pragma unroll 1
    for (int blk = blk0; blk < nb; blk += step) {
      const int k0 = blk * kMxBlock;
      MxBlock<D, BITS> x;
      load_block(x, src, off, k0);
      f32x4 s[NC][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float scale = __uint_as_float(x.ks[t] << 23);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          const u32x2 w = BITS == 4 ? u32x2{x.k[t][kk], 0}
                                    : u32x2{x.k[t][2 * kk % P::KW], x.k[t][(2 * kk + 1) % P::KW]};
          const bf16x8 kf = mx_values8<BITS>(w, scale);
#pragma unroll
          for (int c = 0; c < NC; ++c) s[c][t] = mfma16(kf, qf[c][kk], kk ? s[c][t] : f32x4{});
        }
      }
      const bool masked = k0 + kMxBlock - 1 > first_masked;
      bf16x8 pb[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (masked) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k0 + 8 * q4 + e > pos[c]) s[c][e >> 2][e & 3] = -INFINITY;
        }
        float mx = fmax2(s[c][0][0], s[c][0][1]);
#pragma unroll
        for (int e = 2; e < 8; e += 2) mx = fmax3(mx, s[c][e >> 2][e & 3], s[c][e >> 2][(e + 1) & 3]);
        mx = quarters_max(mx) * scale_log2;
        if (__builtin_amdgcn_ballot_w64(mx > m_t[c] + kMxSlack)) {
          // each column by itself: its bits do not depend on when others rescale
          const float m_new = mx > m_t[c] + kMxSlack ? mx : m_t[c];
          // 0 when m_t is still -inf; 1 for a column that stays all-masked (m_new = -inf; its
          // sums are still 0), where exp2(-inf - -inf) would be NaN
          const float alpha = m_new == -INFINITY ? 1.f : exp2f_fast(m_t[c] - m_new);
          m_t[c] = m_new;
          l_part[c] *= alpha;
#pragma unroll
          for (int n = 0; n < DT; ++n) oacc[c][n] *= alpha;
        }
        const float m_use = m_t[c] == -INFINITY ? 0.f : m_t[c];
        float p[8], rs = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = exp2f_fast(__builtin_fmaf(s[c][e >> 2][e & 3], scale_log2, -m_use));
          rs += p[e];
        }
        l_part[c] += rs;
        const bf16x4 lo = pack4(p[0], p[1], p[2], p[3]), hi = pack4(p[4], p[5], p[6], p[7]);
        pb[c] = bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      }
      bf16x8 vt[DT], mark;
      // Where rows see different keys (several new rows), a NaN group of a key that a row does not
      // see must not reach it through 0 * NaN: those blocks count the NaN keys that each row sees.
      const bool nans = masked && Tq > 1 && __builtin_amdgcn_ballot_w64(any_nan_scale(x.vs));
      if (!nans) {
        v_tiles<D, BITS, false>(vt, x, turn, mark);
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
          for (int c = 0; c < NC; ++c) oacc[c][n] = mfma16(vt[n], pb[c], oacc[c][n]);
      } else {
        v_tiles<D, BITS, true>(vt, x, turn, mark);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          bf16x8 seen;
#pragma unroll
          for (int e = 0; e < 8; ++e) seen[e] = (bf16)(k0 + 8 * q4 + e > pos[c] ? 0.f : 1.f);
          const f32x4 count = mfma16(mark, seen, f32x4{});
#pragma unroll
          for (int n = 0; n < DT; ++n) {
            oacc[c][n] = mfma16(vt[n], pb[c], oacc[c][n]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (count[r] > 0.f) oacc[c][n][r] = __builtin_nanf("");
          }
        }
      }
    }
  }

  if (SPLIT && chunk >= used) {  // an empty partial, whose O the merge does not read
    if (threadIdx.x < R) {
      const int g = threadIdx.x / Tq;
      const int64_t row = ((int64_t)b * Hq + hk * G + g) * Tq + (threadIdx.x - g * Tq);
      *reinterpret_cast<f32x2 *>(part_ml + (row * n_chunks + chunk) * 2) = f32x2{-INFINITY, 0.f};
    }
    return;
  }

  // Merge of the workgroup's waves, as in fa_decode.hip: every wave scales its partial to the
  // workgroup's running max and stages it as fp32 rows, then the threads add the waves in order.
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float l = quarters_sum(l_part[c]);
    if (q4 == 0) {
      // A wave without visible keys (l exactly 0) weighs nothing.  A NaN sum is no empty one: its
      // max may still be -inf (no score compares greater), and then the sum is relative to 0.
      wm[wave][16 * c + i16] = l == 0.f ? -INFINITY : m_t[c] == -INFINITY ? 0.f : m_t[c];
      wsum[wave][16 * c + i16] = l;
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = 16 * c + i16, cols = min(R - 16 * c, 16);  // cols > 0: R > 16 where NC is 2
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
          *reinterpret_cast<f32x4 *>(&stage[wave][i16 * D + ((ch ^ (i16 & 7)) << 2)]) =
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
        t += *reinterpret_cast<const f32x4 *>(&stage[w][j * D + ((ch ^ (j & 7)) << 2)]);
        ls += wm[w][k] == -INFINITY ? 0.f : wsum[w][k] * exp2f_fast(wm[w][k] - mx);
      }
      const int g = k / Tq;
      const int64_t row = ((int64_t)b * Hq + hk * G + g) * Tq + (k - g * Tq);
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

// Workgroups per unit, waves per workgroup, and the blocks a workgroup takes at least (see
// decode_split).
DecodeSplit decode_mx_split(int B, int Hkv, int Lmax, int D, int bits) {
  const int64_t units = (int64_t)B * Hkv;
  const int64_t blocks = ((int64_t)Lmax + kMxBlock - 1) / kMxBlock;
  if (blocks <= 16) return {4, 1, 0};
  int64_t n = 1024 / units;
  if (n < 1) n = 1;
  const int64_t most = (blocks + 3) / 4;
  n = n > most ? most : n > 512 ? 512 : n;
  const int64_t least = units <= 32 ? 4 : (blocks + n - 1) / n;
  int log2_min = 0;
  while (least >> (log2_min + 1)) ++log2_min;
  return {4, (int)n, log2_min};
}

template <int D, int BITS, int NC>
static hipError_t launch_shape(const void *q, const KvCache &cache, const int *cache_seqlens, void *o,
                               float *lse, float *workspace, int B, int Hq, int Hkv, int Tq, int Lmax,
                               const DecodeSplit &sp, float scale_log2, hipStream_t stream) {
  const int rows = B * Hq * Tq;
  float *part_o = workspace, *part_ml = workspace + (int64_t)rows * sp.n_chunks * D;
  const dim3 grid((unsigned)((int64_t)B * Hkv), (unsigned)sp.n_chunks), block(256);
  auto go = [&](auto kernel) {
    kernel<<<grid, block, 0, stream>>>((const bf16 *)q, cache, cache_seqlens, (bf16 *)o, lse, part_o,
                                       part_ml, B, Hq, Hkv, Tq, Lmax, sp.n_chunks, sp.log2_min,
                                       scale_log2);
    return hipGetLastError();
  };
  if (sp.n_chunks == 1) return go(fa_decode_mx_kernel<D, BITS, 4, NC, false>);
  const hipError_t e = go(fa_decode_mx_kernel<D, BITS, 4, NC, true>);
  return e != hipSuccess ? e : launch_decode_combine(part_o, part_ml, o, lse, rows, sp.n_chunks, D, stream);
}

hipError_t launch_decode_mx(const void *q, const KvCache &cache, const int *cache_seqlens, void *o,
                            float *lse, float *workspace, int B, int Hq, int Hkv, int Tq, int Lmax,
                            int D, int bits, float scale, hipStream_t stream) {
  const DecodeSplit sp = decode_mx_split(B, Hkv, Lmax, D, bits);
  auto go = [&](auto launch) {
    return launch(q, cache, cache_seqlens, o, lse, workspace, B, Hq, Hkv, Tq, Lmax, sp,
                  scale * kLog2e, stream);
  };
  const bool wide = Hq / Hkv * Tq > 16;
  if (D == 64) {
    if (bits == 4) return wide ? go(launch_shape<64, 4, 2>) : go(launch_shape<64, 4, 1>);
    return wide ? go(launch_shape<64, 8, 2>) : go(launch_shape<64, 8, 1>);
  }
  if (bits == 4) return wide ? go(launch_shape<128, 4, 2>) : go(launch_shape<128, 4, 1>);
  return wide ? go(launch_shape<128, 8, 2>) : go(launch_shape<128, 8, 1>);
}

}  // namespace ttfa
