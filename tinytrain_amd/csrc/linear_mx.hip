// Products with a quantised weight, gfx950: y[m][n] = sum_k x[m][k] W[n][k], W in 4 or 8 bits with a
// power of two per 32 elements (kv_cache_mx.hip describes the format), x in bf16 or in 8 bits as the
// norm's kernel gives it.  The reference has no counterpart (its linear layers are bf16 products).
//
// Every value of either format is a bf16 as it stands, and so the products are bf16 ones with fp32
// sums: exact products, one rounding of y at the end.
//
// Few rows (up to kFewRows): bound by reading W once.  A workgroup takes 16 rows of W, its four waves
// every fourth 128 columns; a lane loads 32 consecutive elements of its row with their scale, converts
// them in registers, and multiplies them with the same 32 elements of 16 rows of x at a time
// (v_mfma_f32_16x16x32_bf16, W as first operand: D[n][m]).  The waves' sums are joined through LDS.
#include <type_traits>

#include "fa_common.h"
#include "fa_kernels.h"
#include "mx.h"
#include "ttfa.h"

namespace ttfa {

namespace {

// 32 consecutive elements of a row with their scale, as loaded; a lane past the row's end holds zeros.
template <int BITS>
struct Mx32 {
  u32x4 c[BITS / 4];
  uint32_t byte;
  __device__ __forceinline__ void load(const uint8_t *codes, const uint8_t *scales, int64_t group, bool ok) {
    byte = 0;
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) c[i] = u32x4{};
    if (ok) {
      byte = scales[group];
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i)
        c[i] = reinterpret_cast<const u32x4 *>(codes + group * (4 * BITS))[i];
    }
  }
  // elements 8 j .. 8 j + 7
  __device__ __forceinline__ bf16x8 values(int j) const {
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

template <int BITS, bool XMX, int MB>
__global__ __launch_bounds__(256) void linear_mx_rows_kernel(
    const void *__restrict__ x, const uint8_t *__restrict__ x_scales, const uint8_t *__restrict__ codes,
    const uint8_t *__restrict__ scales, bf16 *__restrict__ y, int M, int K, int N) {
  __shared__ f32x4 part[4][MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, quarter = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB;
  const int64_t groups = K / 32, wrow = (int64_t)min(n0 + row, N - 1) * groups;
  int64_t xrow[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) xrow[b] = (int64_t)min(m0 + 16 * b + row, M - 1) * groups;
  f32x4 acc[MB] = {};
  for (int k = 4 * wave + quarter; k - quarter < groups; k += 16) {
    const bool ok = k < groups;
    Mx32<BITS> w;
    w.load(codes, scales, wrow + k, ok);
    typename std::conditional<XMX, Mx32<8>, Rows32>::type v[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      if constexpr (XMX) v[b].load((const uint8_t *)x, x_scales, xrow[b] + k, ok);
      else v[b].load((const bf16 *)x, xrow[b] + k, ok);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8 wv = w.values(j);
#pragma unroll
      for (int b = 0; b < MB; ++b)
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, v[b].values(j), acc[b], 0, 0, 0);
    }
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) part[wave][b][lane] = acc[b];
  __syncthreads();
  for (int b = wave; b < MB; b += 4) {
    const f32x4 t = (part[0][b][lane] + part[1][b][lane]) + (part[2][b][lane] + part[3][b][lane]);
    const int m = m0 + 16 * b + row, n = n0 + 4 * quarter;
    if (m < M && n < N) *reinterpret_cast<bf16x4 *>(y + (int64_t)m * N + n) = pack4(t[0], t[1], t[2], t[3]);
  }
}

}  // namespace

hipError_t launch_linear_mx(const void *x, const void *x_scales, const void *codes, const void *scales,
                            void *y, int M, int K, int N, int bits, hipStream_t stream) {
  auto go = [&](auto bits_, auto xmx, auto mb) {
    constexpr int MB = decltype(mb)::value;
    linear_mx_rows_kernel<decltype(bits_)::value, decltype(xmx)::value, MB>
        <<<dim3((N + 15) / 16, (M + 16 * MB - 1) / (16 * MB)), dim3(256), 0, stream>>>(
            x, (const uint8_t *)x_scales, (const uint8_t *)codes, (const uint8_t *)scales, (bf16 *)y, M, K, N);
  };
  using std::integral_constant;
  auto by_rows = [&](auto b, auto xmx) {
    if (M <= 16) go(b, xmx, integral_constant<int, 1>{});
    else if (M <= 32) go(b, xmx, integral_constant<int, 2>{});
    else go(b, xmx, integral_constant<int, 4>{});
  };
  auto by_x = [&](auto b) {
    if (x_scales) by_rows(b, std::true_type{});
    else by_rows(b, std::false_type{});
  };
  if (bits == 4) by_x(integral_constant<int, 4>{});
  else by_x(integral_constant<int, 8>{});
  return hipGetLastError();
}

}  // namespace ttfa
