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
#include <type_traits>

#include "fa_kernels.h"
#include "gemm.h"

namespace ttfa {

namespace {

enum Epilogue { kStore, kGated, kGatedGrad };

struct GemmArgs {
  const bf16 *x[2], *w[2];  // kStore: segments of the sum (segs) or problems (z)
  int64_t ldx, ldw;
  int64_t M, N, K;          // K of one segment
  int segs, z, tiles_m, tiles_n;
  const bf16 *da;           // kGatedGrad
  bf16 *out[2];             // [M][N]
};

// Workgroup -> tile.  Consecutive workgroup ids go to the 8 XCDs in turn, each with its own L2, so
// each XCD gets a run of tiles; within it, tiles go down groups of 8 rows of tiles before the next
// column, so that the tiles at work at one time share rows of X and of W.
__device__ __forceinline__ int tile_of(int bid, int n) {
  const int per = n / 8, rem = n % 8, x = bid % 8, i = bid / 8;
  return x * per + (x < rem ? x : rem) + i;
}

template <int TM, int TN, int WM, int WN, int BK, bool XTR, bool WTR, Epilogue E>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs g) {
  constexpr int NT = 64 * WM * WN, MB = TM / WM / 32, NB = TN / WN / 32;
  constexpr bool DUAL = E != kStore;
  static_assert(!DUAL || (NB == 2 && !WTR), "a wave has 32 columns of both sums");
  using XL = TileLoad<TM, BK, XTR, NT>;
  using WL = TileLoad<TN, BK, WTR, NT>;
  constexpr int STAGE = XL::BYTES + WL::BYTES;
  __shared__ __align__(1024) char lds[2 * STAGE];

  int tile = tile_of(blockIdx.x, gridDim.x);
  const int per = g.tiles_m * g.tiles_n, z = tile / per;
  tile -= z * per;
  const int band = 8 * g.tiles_n, b0 = tile / band * 8, rows = min(8, g.tiles_m - b0);
  const int in = tile - tile / band * band;
  const int64_t m0 = (int64_t)(b0 + in % rows) * TM;
  const int64_t n0 = (int64_t)(in / rows) * (DUAL ? TN / 2 : TN);

  XL xl;
  WL wl;
  xl.init(g.ldx);
  wl.init(g.ldw, DUAL ? TN / 2 : TN);
  const int wave = wave_id(), wm = wave / WN, wn = wave % WN, lane = threadIdx.x & 63;
  TileRead<TM, BK, XTR> xr;
  TileRead<TN, BK, WTR, DUAL ? TN / 2 : 32> wr;
  xr.init(wm * (TM / WM));
  wr.init(wn * (DUAL ? 32 : TN / WN));

  const int64_t xrows = XTR ? g.K : g.M, wrows = WTR ? g.K : g.N;
  const int per_seg = (int)((g.K + BK - 1) / BK), stages = per_seg * g.segs;
  int seg = z;
  int64_t k0 = 0;
  auto load = [&](char *dst) {  // the next stage
    const int64_t left = g.K - k0;
    const bf16 *x = g.x[seg], *w = g.w[seg];
    xl.template load<0, XL::LOADS>(rsrc_to(x + (XTR ? k0 * g.ldx + m0 : m0 * g.ldx + k0), x + xrows * g.ldx),
                                   dst, left);
    const int64_t at = WTR ? k0 * g.ldw + n0 : n0 * g.ldw + k0;
    dst += XL::BYTES;
    if constexpr (DUAL) {
      wl.template load<0, WL::LOADS / 2>(rsrc_to(g.w[0] + at, g.w[0] + wrows * g.ldw), dst, left);
      wl.template load<WL::LOADS / 2, WL::LOADS>(rsrc_to(g.w[1] + at, g.w[1] + wrows * g.ldw), dst, left);
    } else {
      wl.template load<0, WL::LOADS>(rsrc_to(w + at, w + wrows * g.ldw), dst, left);
    }
    k0 += BK;
    if (k0 >= g.K) k0 = 0, ++seg;
  };

  f32x16 acc[MB][NB] = {};
  load(lds);
  for (int st = 0; st < stages; ++st) {
    const char *cur = lds + (st & 1) * STAGE;
    wait_vm_all();
    __syncthreads();
    if (st + 1 < stages) load(lds + (~st & 1) * STAGE);
#pragma unroll
    for (int s = 0; s < BK / 16; ++s) {
      bf16x8 xf[MB], wf[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) wf[b] = wr.read(cur + XL::BYTES, b, s);
#pragma unroll
      for (int b = 0; b < MB; ++b) xf[b] = xr.read(cur, b, s);
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mfma32(wf[j], xf[i], acc[i][j]);
    }
  }

  const int64_t nw = n0 + wn * (DUAL ? 32 : TN / WN) + 8 * (lane >> 5);
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t m = m0 + wm * (TM / WM) + 32 * i + (lane & 31);
    if constexpr (E == kStore) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const u32x4 v = row_piece(acc[i][j], p);
          const int64_t n = nw + 32 * j + 16 * p;
          if (m < g.M && n < g.N) *reinterpret_cast<u32x4 *>(g.out[z] + m * g.N + n) = v;
        }
    } else {
      f32x16 da;
      if constexpr (E == kGatedGrad) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          u32x4 piece{};
          if (m < g.M && nw + 16 * p < g.N)
            piece = *reinterpret_cast<const u32x4 *>(g.da + m * g.N + nw + 16 * p);
          block_regs(piece, da, p);
        }
      }
      f32x16 r0, r1;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float gate = acc[i][0][e], up = acc[i][1][e];
        const float sig = __builtin_amdgcn_rcpf(1.f + exp2f_fast(-gate * kLog2e));
        if constexpr (E == kGated) {
          r0[e] = gate * sig * up;
        } else {
          r0[e] = da[e] * up * sig * fmaf(gate, 1.f - sig, 1.f);
          r1[e] = da[e] * gate * sig;
        }
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const u32x4 v0 = row_piece(r0, p);
        const bool in_range = m < g.M && nw + 16 * p < g.N;
        const int64_t at = m * g.N + nw + 16 * p;
        if (in_range) *reinterpret_cast<u32x4 *>(g.out[0] + at) = v0;
        if constexpr (E == kGatedGrad) {
          const u32x4 v1 = row_piece(r1, p);
          if (in_range) *reinterpret_cast<u32x4 *>(g.out[1] + at) = v1;
        }
      }
    }
  }
}

template <bool XTR, bool WTR, Epilogue E>
hipError_t launch_gemm(GemmArgs g, hipStream_t stream) {
  constexpr int TM = 128, TN = 256;
  g.tiles_m = (int)((g.M + TM - 1) / TM);
  g.tiles_n = (int)((g.N + (E == kStore ? TN : TN / 2) - 1) / (E == kStore ? TN : TN / 2));
  gemm_kernel<TM, TN, 1, 4, 32, XTR, WTR, E>
      <<<dim3(g.z * g.tiles_m * g.tiles_n), dim3(256), 0, stream>>>(g);
  return hipGetLastError();
}

const bf16 *in(const void *p) { return static_cast<const bf16 *>(p); }

}  // namespace

hipError_t launch_swiglu_fwd(const void *x, const void *w_gate, const void *w_up, void *a, int M, int K,
                             int N, hipStream_t stream) {
  GemmArgs g{{in(x), in(x)}, {in(w_gate), in(w_up)}, K, K, M, N, K, 1, 1, 0, 0, nullptr, {(bf16 *)a, nullptr}};
  return launch_gemm<false, false, kGated>(g, stream);
}

hipError_t launch_swiglu_bwd(const void *da, const void *x, const void *w_gate, const void *w_up, void *dx,
                             void *dw_gate, void *dw_up, void *workspace, int M, int K, int N,
                             hipStream_t stream) {
  bf16 *dg = static_cast<bf16 *>(workspace), *du = dg + (int64_t)M * N;
  GemmArgs g{{in(x), in(x)}, {in(w_gate), in(w_up)}, K, K, M, N, K, 1, 1, 0, 0, in(da), {dg, du}};
  hipError_t e = launch_gemm<false, false, kGatedGrad>(g, stream);
  if (e == hipSuccess && dx) {
    GemmArgs d{{dg, du}, {in(w_gate), in(w_up)}, N, K, M, K, N, 2, 1, 0, 0, nullptr, {(bf16 *)dx, nullptr}};
    e = launch_gemm<false, true, kStore>(d, stream);
  }
  if (e == hipSuccess && dw_gate) {
    GemmArgs d{{dg, du}, {in(x), in(x)}, N, K, N, K, M, 1, 2, 0, 0, nullptr, {(bf16 *)dw_gate, (bf16 *)dw_up}};
    e = launch_gemm<true, true, kStore>(d, stream);
  }
  return e;
}

}  // namespace ttfa
