// Gated feed-forward input, gfx950: a = silu(x Wg^T) * (x Wu^T) in one kernel, and its backward.
// (model.py:111-125: act(gate_proj(x)) * up_proj(x); the down projection stays a product of its own.)
//
//   g = x Wg^T, u = x Wu^T, a = g u / (1 + e^-g)
//   du = da silu(g), dg = da u sig(g) (1 + g (1 - sig(g)))
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
// a is formed from both sums in fp32 registers: a workgroup's W tile holds rows of Wg and the same rows of
// Wu, so a wave has both sums of an element.  For the backward they are written as well, in 20 bits each: 12
// significant bits, an error of 2^-13 against the 2^-9 that every gradient has from its own rounding and
// from that of dg and du, as bf16 operands of the last two products (in bf16 they would add as much
// again).  That is 5 bytes an element; to form them again instead of reading them was 713 us at
// 16384 x 2048 x 6144, against 227 of the kernel that reads them (swiglu_grad_kernel).
#include "fa_kernels.h"
#include "gemm.h"

namespace ttfa {

namespace {

// Few rows: bound by reading the weights once.  A workgroup takes 16 NB rows of Wg and the same ones of Wu;
// its eight waves take every eighth 128 k's, with all loads of those on their way at once, and multiply
// them with up to 16 MB rows of x (v_mfma_f32_16x16x32_bf16, W as first operand: D[n][m]).  A lane takes
// eight k's of every 32, so that a load instruction reads 64 consecutive bytes of each of 16 rows (with 32
// consecutive k's a lane, four pieces of 16 bytes of each: 50 MB of weights 16.5 us, 13.3 so).  The waves'
// sums are joined through LDS.  200 MB of weights and one row: 36.7 us, 5.5 TB/s; 7 MB 4.1 us, of which a
// launch and the latency of one round of loads are most.  More rows take longer by reading x again for
// every 16 NB columns (32 rows: 15.6 us at 50 MB).
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
                                                                     bf16 *__restrict__ a,
                                                                     uint8_t *__restrict__ saved, int M, int K,
                                                                     int N) {
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
  if (m >= M || n >= N) return;
  const int64_t at = (int64_t)m * N + n;
  *reinterpret_cast<bf16x4 *>(a + at) = pack4(r[0], r[1], r[2], r[3]);
  if (!saved) return;
  const SavedSums s(saved, (int64_t)M * N);
  uint32_t gh[2], uh[2], low;
  saved_four({g[0], g[1], g[2], g[3]}, {u[0], u[1], u[2], u[3]}, gh, uh, low);
  *reinterpret_cast<u32x2 *>(s.high[0] + at) = u32x2{gh[0], gh[1]};
  *reinterpret_cast<u32x2 *>(s.high[1] + at) = u32x2{uh[0], uh[1]};
  *reinterpret_cast<uint32_t *>(s.low + at) = low;
}

// dg and du from da and the saved sums, eight elements a lane.  Bound by memory: 11 bytes an element.
__global__ __launch_bounds__(256) void swiglu_grad_kernel(const bf16 *__restrict__ da, const uint8_t *saved_at,
                                                          bf16 *__restrict__ dg, bf16 *__restrict__ du,
                                                          int64_t lanes) {
  const SavedSums s(const_cast<uint8_t *>(saved_at), 8 * lanes);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < lanes; i += (int64_t)gridDim.x * 256) {
    const bf16x8 d = reinterpret_cast<const bf16x8 *>(da)[i];
    const u32x4 gh = reinterpret_cast<const u32x4 *>(s.high[0])[i], uh = reinterpret_cast<const u32x4 *>(s.high[1])[i];
    const u32x2 low = reinterpret_cast<const u32x2 *>(s.low)[i];
    bf16x8 x, y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t l = low[e / 4] >> (8 * (e % 4));
      const float g = __uint_as_float((e % 2 ? gh[e / 2] & 0xffff0000u : gh[e / 2] << 16) | (l & 15) << 12);
      const float u = __uint_as_float((e % 2 ? uh[e / 2] & 0xffff0000u : uh[e / 2] << 16) | (l >> 4 & 15) << 12);
      const float sig = sigmoid(g), t = (float)d[e] * sig;
      x[e] = (bf16)(t * u * fmaf(g, 1.f - sig, 1.f));
      y[e] = (bf16)(t * g);
    }
    reinterpret_cast<bf16x8 *>(dg)[i] = x;
    reinterpret_cast<bf16x8 *>(du)[i] = y;
  }
}

const bf16 *in(const void *p) { return static_cast<const bf16 *>(p); }

}  // namespace

int64_t swiglu_saved_bytes(int M, int N) { return 5ll * M * N; }

hipError_t launch_swiglu_fwd(const void *x, const void *w_gate, const void *w_up, void *a, void *saved, int M,
                             int K, int N, hipStream_t stream) {
  if (swiglu_few_rows(M, N)) {
    auto go = [&](auto kernel, int columns) {
      kernel<<<dim3((N + columns - 1) / columns), dim3(64 * kRowWaves), 0, stream>>>(
          in(x), in(w_gate), in(w_up), (bf16 *)a, (uint8_t *)saved, M, K, N);
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
  GemmArgs g{{in(x), in(x)}, {in(w_gate), in(w_up)}, K, K, M, N, K, 1, 1, {(bf16 *)a, nullptr}, nullptr,
             (uint8_t *)saved, {}};
  const Cut c = cut_of(M, N, K, 1, 1, true);
  return saved ? launch_gemm<false, false, kGatedSave>(g, c, stream) : launch_gemm<false, false, kGated>(g, c, stream);
}

int64_t swiglu_bwd_workspace(int M, int K, int N) {
  const int64_t dx = part_bytes(cut_of(M, K, N, 2, 1, false), M, K, 1);
  const int64_t dw = part_bytes(cut_of(N, K, M, 1, 2, false), N, K, 2);
  return 4ll * M * N + std::max(dx, dw);
}

hipError_t launch_swiglu_bwd(const void *da, const void *saved, const void *x, const void *w_gate,
                             const void *w_up, void *dx, void *dw_gate, void *dw_up, void *workspace, int M,
                             int K, int N, hipStream_t stream) {
  bf16 *dg = static_cast<bf16 *>(workspace), *du = dg + (int64_t)M * N;
  float *part = reinterpret_cast<float *>(du + (int64_t)M * N);
  const int64_t lanes = (int64_t)M * N / 8;
  swiglu_grad_kernel<<<dim3((unsigned)std::min<int64_t>((lanes + 255) / 256, 1 << 20)), dim3(256), 0, stream>>>(
      in(da), static_cast<const uint8_t *>(saved), dg, du, lanes);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && dx) {
    GemmArgs d{{dg, du}, {in(w_gate), in(w_up)}, N, K, M, K, N, 2, 1, {(bf16 *)dx, nullptr}, part, nullptr, {}};
    e = launch_gemm<false, true, kStore>(d, cut_of(M, K, N, 2, 1, false), stream);
  }
  if (e == hipSuccess && dw_gate) {
    GemmArgs d{{dg, du}, {in(x), in(x)}, N, K, N, K, M, 1, 2, {(bf16 *)dw_gate, (bf16 *)dw_up}, part, nullptr, {}};
    e = launch_gemm<true, true, kStore>(d, cut_of(N, K, M, 1, 2, false), stream);
  }
  return e;
}

}  // namespace ttfa
