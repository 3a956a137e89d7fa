// Gated feed-forward input, gfx950: a = silu(x Wg^T) * (x Wu^T) in one kernel, and its backward.
// (model.py:111-125: act(gate_proj(x)) * up_proj(x); the down projection stays a product of its own.)
//
//   g = x Wg^T, u = x Wu^T, a = g u / (1 + e^-g)
//   du = da silu(g), dg = da u sig(g) (1 + g (1 - sig(g)))
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
// g and u never leave the registers in fp32: a workgroup's W tile holds rows of Wg and the same rows
// of Wu, so a wave has both sums of an element.  The backward forms them again (4MNK more operations
// on top of 8MNK): kept in fp32 they would be written and read back at 8 bytes an element each way,
// which takes as long and as much memory; kept in bf16 they would round every gradient once more.
// dg and du are rounded to bf16 once, as operands of the last two products.
#include <algorithm>
#include <type_traits>

#include "fa_bwd.h"  // allow_lds
#include "fa_kernels.h"
#include "gemm.h"

namespace ttfa {

namespace {

// kPartial: kStore's sums in fp32, one of `splits` parts of the contraction.
enum Epilogue { kStore, kPartial, kGated, kGatedGrad };

struct GemmArgs {
  const bf16 *x[2], *w[2];  // kStore, kPartial: segments of the sum (segs) or problems (z)
  int64_t ldx, ldw;
  int64_t M, N, K;          // K of one segment
  int segs, z;
  const bf16 *da;           // kGatedGrad
  bf16 *out[2];             // [M][N]
  float *part;              // kPartial: [splits][z][M][N]
  int splits, tiles_m, tiles_n;
};

// The i-th of n tiles in the order of work -> tile.  Consecutive workgroup ids go to the 8 XCDs in turn,
// each with its own L2, so each XCD gets a run of tiles.
__device__ __forceinline__ int tile_of(int i, int n) {
  const int per = n / 8, rem = n % 8, x = i % 8;
  return x * per + (x < rem ? x : rem) + i / 8;
}

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
template <int TM, int TN, int WM, int WN, int BK, bool XTR, bool WTR, Epilogue E>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs g) {
  constexpr int NT = 64 * WM * WN, MB = TM / WM / 32, NB = TN / WN / 32, STEPS = BK / 16;
  constexpr bool DUAL = E == kGated || E == kGatedGrad;
  static_assert(!DUAL || (NB == 2 && !WTR), "a wave has 32 columns of both sums");
  static_assert(STEPS % 2 == 0, "operands alternate between two sets of registers");
  constexpr int WT = DUAL ? TN / 2 : TN, STORES = MB * (E == kGated ? 2 : E == kPartial ? 4 * NB : 4);
  using XL = TileLoad<TM, BK, XTR, NT>;
  using WL = TileLoad<WT, BK, WTR, NT>;
  constexpr int STAGE = (TM + TN) * BK * 2;
  extern __shared__ __align__(1024) char lds[];

  struct Tile {
    int part, z;  // part of the contraction, problem
    int64_t m0, n0;
  };
  const int per = g.tiles_m * g.tiles_n, total = g.splits * g.z * per;
  const int per_seg = (int)((g.K + BK - 1) / BK), all_stages = per_seg * g.segs;
  auto first_stage = [&](int part) { return E == kPartial ? (int)((int64_t)all_stages * part / g.splits) : part * all_stages; };
  // Tiles go down bands of 8 rows of tiles before the next column: those at work at one time share rows
  // of X and of W.
  auto tile_at = [&](int i) {
    int t = tile_of(i, total);
    const int zs = t / per;
    t -= zs * per;
    const int band = 8 * g.tiles_n, b0 = t / band * 8, rows = min(8, g.tiles_m - b0), in = t - t / band * band;
    return Tile{zs / g.z, zs % g.z, (int64_t)(b0 + in % rows) * TM, (int64_t)(in / rows) * WT};
  };

  // Loads: a cursor over the stages of this workgroup's tiles.
  XL xl;
  WL wl, ul;  // ul: the second weight's rows of a dual tile
  int ahead = blockIdx.x, seg, to_do;  // stages of the tile at `at`
  int64_t left;
  Tile at;
  auto start = [&](int skip) {
    const int i = at.z + seg;
    xl.init(g.x[i], g.ldx, at.m0, g.M);
    wl.init(g.w[i], g.ldw, at.n0, g.N);
    if constexpr (DUAL) ul.init(g.w[1], g.ldw, at.n0, g.N);
    if constexpr (E == kPartial) xl.skip(skip), wl.skip(skip);
    left = g.K - (int64_t)skip * BK;
  };
  auto next_tile = [&] {
    at = tile_at(ahead);
    const int first = first_stage(at.part);
    to_do = first_stage(at.part + 1) - first;
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
      if constexpr (DUAL) ul.shorten(g.ldw, (int)left);
    }
    xl.load(dst);
    wl.load(dst + XL::BYTES);
    if constexpr (DUAL) ul.load(dst + XL::BYTES + WL::BYTES);
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
  // last step: there the workgroup meets, the stage's buffer takes the loads of the stage after next,
  // and the next stage, whose loads had a whole stage's time, is read from.
  load(0);
  wait_and_meet<0>();
  load(1);
  read(0, 0, 0);
  int buf = 0;
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    const Tile t = tile_at(i);
    const int stages = first_stage(t.part + 1) - first_stage(t.part);
    f32x16 acc[MB][NB] = {};
    const int row = wm * (TM / WM) + (lane & 15), col = wn * (DUAL ? 32 : TN / WN) + 8 * piece_of(lane);
    const uint32_t bytes = (uint32_t)((g.M - t.m0 < TM ? g.M - t.m0 : TM) * g.N * 2);
    // byte offset in the tile's rows of this lane's piece of set q of block (i, j)
    auto piece_at = [&](int i, int j, int q) {
      const int64_t n = t.n0 + col + 32 * j;
      return n < g.N ? (uint32_t)((row + 32 * i + 16 * q) * g.N * 2 + n * 2) : kPastEnd;
    };
    u32x4 da[MB][2];
    for (int st = 0; st < stages; ++st) {
      if (E == kGatedGrad && st == 0) {  // a tile's time to arrive (in its last stage: 728 us for 713 at 16384 x 2048 x 6144)
        const __amdgpu_buffer_rsrc_t r = make_rsrc(g.da + t.m0 * g.N, bytes);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int p = 0; p < 2; ++p) da[i][p] = buf_load16(r, piece_at(i, 0, p));
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (s + 1 < STEPS) {
          read(buf, s + 1, (s + 1) & 1);
        } else {
          // After a tile's results were stored: its stores are younger than the loads waited for.
          if (st == 0 && i != (int)blockIdx.x) wait_and_meet<STORES>();
          else wait_and_meet<0>();
          load(buf);
          read(buf ^ 1, 0, (s + 1) & 1);  // after the last stage: values that nothing uses
        }
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[i][j] = mfma32(wf[s & 1][j], xf[s & 1][i], acc[i][j]);
        interleave<MB * NB>();
      }
      buf ^= 1;
    }

    if constexpr (E == kPartial) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(g.part + ((int64_t)(t.part * g.z + t.z) * g.M + t.m0) * g.N, 2 * bytes);
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          u32x4 set[4];
          block_rows_f32(acc[i][j], set);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int64_t n = t.n0 + wn * (TN / WN) + 32 * j + 16 * (q / 2) + 8 * ((lane >> 4) & 1) + 4 * (lane >> 5);
            buf_store16(r, n < g.N ? (uint32_t)((row + 32 * i + 16 * (q % 2)) * g.N * 4 + n * 4) : kPastEnd, set[q]);
          }
        }
      continue;
    }
    const __amdgpu_buffer_rsrc_t r0 = make_rsrc(g.out[E == kStore ? t.z : 0] + t.m0 * g.N, bytes);
    const __amdgpu_buffer_rsrc_t r1 = make_rsrc(g.out[1] + t.m0 * g.N, bytes);
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
        f32x16 d, v0, v1;
        if constexpr (E == kGatedGrad) d = block_regs(da[i][0], da[i][1]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float gate = acc[i][0][e], up = acc[i][1][e];
          const float sig = __builtin_amdgcn_rcpf(1.f + exp2f_fast(-gate * kLog2e));
          if constexpr (E == kGated) {
            v0[e] = gate * sig * up;
          } else {
            v0[e] = d[e] * up * sig * fmaf(gate, 1.f - sig, 1.f);
            v1[e] = d[e] * gate * sig;
          }
        }
        u32x4 set[2];
        block_rows(v0, set);
        buf_store16(r0, piece_at(i, 0, 0), set[0]);
        buf_store16(r0, piece_at(i, 0, 1), set[1]);
        if constexpr (E == kGatedGrad) {
          block_rows(v1, set);
          buf_store16(r1, piece_at(i, 0, 0), set[0]);
          buf_store16(r1, piece_at(i, 0, 1), set[1]);
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

// How a product is cut: tiles of 256 x 256 (one workgroup a CU) or 128 x 128 (two), and parts of the
// contraction that sum_parts_kernel joins.
struct Cut {
  bool wide;
  int splits;
};

int64_t tiles_of(int64_t M, int64_t N, int tm, int tn) { return (M + tm - 1) / tm * ((N + tn - 1) / tn); }

constexpr double kMostPartFloats = 1 << 26;  // 256 MB, what the last-level cache holds

// The cut that is estimated to take least time, in microseconds on 256 CUs: a stage of 64 k's of a wide
// tile takes 1.5, of a narrow one 0.6 alone on its CU and 1.0 beside another; 3 stages more for a tile's
// start and end; parts go out and in at 4 TB/s, with a launch of 4 us.
Cut cut_of(int64_t M, int64_t N, int64_t K, int segs, int z, bool dual) {
  const int64_t stages = (K + 63) / 64 * segs;
  Cut best{true, 1};
  double least = 1e30;
  for (int wide = 1; wide >= 0; --wide) {
    const int64_t tiles = z * (wide ? tiles_of(M, N, 256, dual ? 128 : 256) : tiles_of(M, N, 128, dual ? 64 : 128));
    for (int s = 1; s <= (dual ? 1 : 32) && s <= stages; ++s) {
      if (s > 1 && (double)s * z * M * N > kMostPartFloats) break;
      const int64_t n = tiles * s;
      const double len = (double)((stages + s - 1) / s) + 3;
      double t;
      if (wide) {
        t = (double)((n + 255) / 256) * len * 1.5;
      } else {
        const int64_t full = n / 512, rest = n % 512;
        t = ((double)full * 1.0 + (rest == 0 ? 0 : rest <= 256 ? 0.6 : 1.0)) * len;
      }
      if (s > 1) t += 4 + (double)s * z * M * N * 8 / 4e6;
      if (t < least) least = t, best = Cut{wide != 0, s};
    }
  }
  return best;
}

int64_t part_bytes(const Cut &c, int64_t M, int64_t N, int z) { return c.splits > 1 ? 4 * c.splits * z * M * N : 0; }

template <bool XTR, bool WTR, Epilogue E, int TM, int WM, int WN>
hipError_t launch_tiles(GemmArgs g, hipStream_t stream) {
  constexpr int BK = 64, TN = TM, DUAL = E == kGated || E == kGatedGrad, WT = DUAL ? TN / 2 : TN;
  constexpr int lds = 2 * (TM + TN) * BK * 2;
  constexpr auto kernel = gemm_kernel<TM, TN, WM, WN, BK, XTR, WTR, E>;
  g.tiles_m = (int)((g.M + TM - 1) / TM);
  g.tiles_n = (int)((g.N + WT - 1) / WT);
  if constexpr (lds > 65536) {
    const hipError_t e = allow_lds<kernel>(lds);
    if (e != hipSuccess) return e;
  }
  const int slots = resident_slots<kernel>(64 * WM * WN, lds);
  kernel<<<dim3(std::min(slots, g.splits * g.z * g.tiles_m * g.tiles_n)), dim3(64 * WM * WN), lds, stream>>>(g);
  return hipGetLastError();
}

template <bool XTR, bool WTR, Epilogue E>
hipError_t launch_gemm(GemmArgs g, const Cut &c, hipStream_t stream) {
  g.splits = c.splits;
  if constexpr (E == kStore) {
    if (c.splits > 1) {
      const hipError_t e = c.wide ? launch_tiles<XTR, WTR, kPartial, 256, 2, 4>(g, stream)
                                  : launch_tiles<XTR, WTR, kPartial, 128, 2, 2>(g, stream);
      if (e != hipSuccess) return e;
      const int64_t n0 = g.M * g.N / 8, n = g.z * n0;
      sum_parts_kernel<<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream>>>(g.part, g.out[0], g.out[1],
                                                                                   c.splits, n0, n);
      return hipGetLastError();
    }
  }
  return c.wide ? launch_tiles<XTR, WTR, E, 256, 2, 4>(g, stream) : launch_tiles<XTR, WTR, E, 128, 2, 2>(g, stream);
}

const bf16 *in(const void *p) { return static_cast<const bf16 *>(p); }

}  // namespace

hipError_t launch_swiglu_fwd(const void *x, const void *w_gate, const void *w_up, void *a, int M, int K,
                             int N, hipStream_t stream) {
  GemmArgs g{{in(x), in(x)}, {in(w_gate), in(w_up)}, K, K, M, N, K, 1, 1, nullptr, {(bf16 *)a, nullptr}, nullptr};
  return launch_gemm<false, false, kGated>(g, cut_of(M, N, K, 1, 1, true), stream);
}

int64_t swiglu_bwd_workspace(int M, int K, int N) {
  const int64_t dx = part_bytes(cut_of(M, K, N, 2, 1, false), M, K, 1);
  const int64_t dw = part_bytes(cut_of(N, K, M, 1, 2, false), N, K, 2);
  return 4ll * M * N + std::max(dx, dw);
}

hipError_t launch_swiglu_bwd(const void *da, const void *x, const void *w_gate, const void *w_up, void *dx,
                             void *dw_gate, void *dw_up, void *workspace, int M, int K, int N,
                             hipStream_t stream) {
  bf16 *dg = static_cast<bf16 *>(workspace), *du = dg + (int64_t)M * N;
  float *part = reinterpret_cast<float *>(du + (int64_t)M * N);
  GemmArgs g{{in(x), in(x)}, {in(w_gate), in(w_up)}, K, K, M, N, K, 1, 1, in(da), {dg, du}, nullptr};
  hipError_t e = launch_gemm<false, false, kGatedGrad>(g, cut_of(M, N, K, 1, 1, true), stream);
  if (e == hipSuccess && dx) {
    GemmArgs d{{dg, du}, {in(w_gate), in(w_up)}, N, K, M, K, N, 2, 1, nullptr, {(bf16 *)dx, nullptr}, part};
    e = launch_gemm<false, true, kStore>(d, cut_of(M, K, N, 2, 1, false), stream);
  }
  if (e == hipSuccess && dw_gate) {
    GemmArgs d{{dg, du}, {in(x), in(x)}, N, K, N, K, M, 1, 2, nullptr, {(bf16 *)dw_gate, (bf16 *)dw_up}, part};
    e = launch_gemm<true, true, kStore>(d, cut_of(N, K, M, 1, 2, false), stream);
  }
  return e;
}

}  // namespace ttfa
