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
#include "fa_kernels.h"
#include "gemm.h"

namespace ttfa {

namespace {

// Few rows: bound by reading the weights once.  A workgroup takes 16 NB rows of Wg and the same ones of Wu;
// its eight waves take every eighth 128 k's, with all loads of those on their way at once, and multiply
// them with up to 16 MB rows of x (v_mfma_f32_16x16x32_bf16, W as first operand: D[n][m]).  A lane takes
// eight k's of every 32, so that a load instruction reads 64 consecutive bytes of each of 16 rows (with 32
// consecutive k's a lane, four pieces of 16 bytes of each: 50 MB of weights 16.5 us, 13.3 so).  The waves'
// sums are joined through LDS.  200 MB of weights and one row: 36 us, 5.6 TB/s; 7 MB 3.9 us, of which a
// launch and the latency of one round of loads are most.  More rows take longer by reading x again for
// every 16 NB columns (32 rows: 16.8 us at 50 MB).
struct K32 {
  u32x4 c[4];
  __device__ __forceinline__ void load(const bf16 *row, int k, int K) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c[j] = k + 32 * j < K ? *reinterpret_cast<const u32x4 *>(row + k + 32 * j) : u32x4{};
  }
  __device__ __forceinline__ bf16x8 values(int j) const { return __builtin_bit_cast(bf16x8, c[j]); }
};

constexpr int kRowWaves = 8;

template <int MB, int NB>
__global__ __launch_bounds__(64 * kRowWaves) void swiglu_rows_kernel(const bf16 *__restrict__ x,
                                                                     const bf16 *__restrict__ w_gate,
                                                                     const bf16 *__restrict__ w_up,
                                                                     bf16 *__restrict__ a, int M, int K, int N) {
  __shared__ f32x4 part[kRowWaves][2 * NB * MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, quarter = lane >> 4;
  const int n0 = blockIdx.x * 16 * NB;
  int64_t wrow[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c) wrow[c] = (int64_t)min(n0 + 16 * c + row, N - 1) * K;  // rows past the end: the last one's, not stored
  f32x4 acc[2][NB][MB] = {};
  for (int k0 = 128 * wave; k0 < K; k0 += 128 * kRowWaves) {
    const int k = k0 + 8 * quarter;
    K32 wg[NB], wu[NB], v[MB];
#pragma unroll
    for (int c = 0; c < NB; ++c) {
      wg[c].load(w_gate + wrow[c], k, K);
      wu[c].load(w_up + wrow[c], k, K);
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) v[b].load(x + (int64_t)min(16 * b + row, M - 1) * K, k, K);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          acc[0][c][b] = mfma16(wg[c].values(j), v[b].values(j), acc[0][c][b]);
          acc[1][c][b] = mfma16(wu[c].values(j), v[b].values(j), acc[1][c][b]);
        }
  }
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      part[wave][c * MB + b][lane] = acc[0][c][b];
      part[wave][(NB + c) * MB + b][lane] = acc[1][c][b];
    }
  __syncthreads();
  if (wave >= MB * NB) return;
  f32x4 g{}, u{};
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    g += part[w][wave][lane];
    u += part[w][MB * NB + wave][lane];
  }
  f32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = g[e] * sigmoid(g[e]) * u[e];
  const int m = 16 * (wave % MB) + row, n = n0 + 16 * (wave / MB) + 4 * quarter;
  if (m < M && n < N) *reinterpret_cast<bf16x4 *>(a + (int64_t)m * N + n) = pack4(r[0], r[1], r[2], r[3]);
}

// Rows of x up to which the kernel above is faster than a tile of 128 x 64 (K 768, N 2304, M 64: 6.8 us, tiles
// 11.6; K 2048, N 6144: 21.0, 32.6), but for many columns (K 4096, N 12288: 74, 68; M 48: 62, 66).
bool few_rows(int M, int N) { return M <= (N <= 8192 ? 64 : 48); }

const bf16 *in(const void *p) { return static_cast<const bf16 *>(p); }

}  // namespace

hipError_t launch_swiglu_fwd(const void *x, const void *w_gate, const void *w_up, void *a, int M, int K,
                             int N, hipStream_t stream) {
  if (few_rows(M, N)) {
    auto go = [&](auto kernel, int columns) {
      kernel<<<dim3((N + columns - 1) / columns), dim3(64 * kRowWaves), 0, stream>>>(
          in(x), in(w_gate), in(w_up), (bf16 *)a, M, K, N);
      return hipGetLastError();
    };
    // 32 columns a workgroup where 16 would give some CUs two workgroups and others one.
    if (N > 16 * 256 && N <= 32 * 256)
      return M <= 16   ? go(swiglu_rows_kernel<1, 2>, 32)
             : M <= 32 ? go(swiglu_rows_kernel<2, 2>, 32)
             : M <= 48 ? go(swiglu_rows_kernel<3, 2>, 32)
                       : go(swiglu_rows_kernel<4, 2>, 32);
    return M <= 16   ? go(swiglu_rows_kernel<1, 1>, 16)
           : M <= 32 ? go(swiglu_rows_kernel<2, 1>, 16)
           : M <= 48 ? go(swiglu_rows_kernel<3, 1>, 16)
                     : go(swiglu_rows_kernel<4, 1>, 16);
  }
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
