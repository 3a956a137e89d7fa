// Quantised KV cache: rows are rounded as they are written (kv_append_mx_kernel) and read back
// (kv_read_mx_kernel), gfx950.  The reference has no KV cache (generate.py:7-20 recomputes the
// prefix; README.md:158 plans one).
//
// Format (OCP Microscaling): 32 consecutive elements of a row share a power of two 2^e, held as
// the byte e + 127; the elements are e2m1 (4 bits, two to a byte, the lower one in the low
// nibble) or e4m3 (8 bits).  For a group of largest magnitude a, e is the smallest integer with
// a <= M 2^e, M the type's largest value plus half of its last step (6 + 1, 448 + 16): the
// largest element then rounds down by no more than half a step, and on normal data the 4-bit
// error is 3% below that of M = 6.  An element is x 2^-e rounded to nearest even, which the
// hardware conversions do in one step (checked against the definition for every bf16 value and
// a million fp32 values next to the rounding borders).  x 2^-e is exact, so the cache is defined
// to the bit.  e is clamped so that every value is a finite normal bf16; a group with a NaN or an
// infinity gets the byte 255, which the conversions read back as NaN.
#include "fa_common.h"
#include "fa_kernels.h"
#include "mx.h"

namespace ttfa {

namespace {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Largest of the group's 32 magnitudes: over the four lanes that hold it.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));  // lane ^ 1
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));  // lane ^ 2
}

// Eight elements of a row, as a lane holds them.
template <class T>
struct Eight;

template <>
struct Eight<bf16> {
  u32x4 w;
  __device__ void load(const bf16 *p) { w = *reinterpret_cast<const u32x4 *>(p); }
  // fp32 bits of the largest magnitude (order of magnitudes = order of their bits, NaN last)
  __device__ uint32_t top() const {
    u16x2 m{};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    return (uint32_t)max(m[0], m[1]) << 16;
  }
  template <int BITS>
  __device__ u32x2 codes(float scale) const {
    u32x2 c{};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = mx_pack<BITS>(c, i, bits_bf16(w[i]), scale);
    return c;
  }

 private:
  static __device__ bf16x2 bits_bf16(uint32_t x) { return __builtin_bit_cast(bf16x2, x); }
};

template <>
struct Eight<float> {
  f32x4 a, b;
  __device__ void load(const float *p) {
    a = reinterpret_cast<const f32x4 *>(p)[0];
    b = reinterpret_cast<const f32x4 *>(p)[1];
  }
  __device__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = max(max(m, __float_as_uint(a[i]) & 0x7fffffffu), __float_as_uint(b[i]) & 0x7fffffffu);
    return m;
  }
  template <int BITS>
  __device__ u32x2 codes(float scale) const {
    u32x2 c = mx_pack<BITS>(u32x2{}, 0, f32x2{a[0], a[1]}, scale);
    c = mx_pack<BITS>(c, 1, f32x2{a[2], a[3]}, scale);
    c = mx_pack<BITS>(c, 2, f32x2{b[0], b[1]}, scale);
    return mx_pack<BITS>(c, 3, f32x2{b[2], b[3]}, scale);
  }
};

}  // namespace

// A lane takes eight elements, D / 8 lanes a row; blockIdx.y picks K or V.  Row t of T goes to
// position cache_seqlens[b] - T + t; one outside the cache is not written.
template <int D, int BITS, class T>
__global__ __launch_bounds__(256) void kv_append_mx_kernel(KvRows<T> in, KvCache cache,
                                                           const int *__restrict__ cache_seqlens,
                                                           int rows, int Hkv, int n_rows, int Lmax) {
  constexpr int LPR = D / 8, CODE = D * BITS / 8;
  const int which = blockIdx.y;
  const int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, ln = threadIdx.x % LPR;
  if (row >= rows) return;  // whole rows, so whole groups of lanes
  const int bh = row / n_rows, t = row - bh * n_rows;
  const int b = bh / Hkv, h = bh - b * Hkv;
  const int64_t pos = (int64_t)cache_seqlens[b] - n_rows + t;
  if (pos < 0 || pos >= Lmax) return;
  const int64_t *st = in.stride[which];
  Eight<T> x;
  x.load(in.x[which] + b * st[0] + h * st[1] + t * st[2] + 8 * ln);
  const uint32_t byte = mx_scale_byte<BITS>(quad_max(x.top()));
  u32x2 c = x.template codes<BITS>(__uint_as_float(byte << 23));
  if (byte == 255) c = u32x2{};
  const int64_t at = (int64_t)bh * Lmax + pos;
  uint8_t *out = cache.codes[which] + at * CODE;
  if constexpr (BITS == 4) reinterpret_cast<uint32_t *>(out)[ln] = c[0];
  else reinterpret_cast<u32x2 *>(out)[ln] = c;
  if (ln % 4 == 0) cache.scales[which][at * (D / 32) + ln / 4] = (uint8_t)byte;
}

// The inverse: row t of n_rows comes from position cache_seqlens[b] - n_rows + t, zeros where that
// lies outside the cache.
template <int D, int BITS, class T>
__global__ __launch_bounds__(256) void kv_read_mx_kernel(KvCache cache,
                                                         const int *__restrict__ cache_seqlens,
                                                         T *__restrict__ k, T *__restrict__ v, int rows,
                                                         int Hkv, int n_rows, int Lmax) {
  constexpr int LPR = D / 8, CODE = D * BITS / 8;
  const int which = blockIdx.y;
  const int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, ln = threadIdx.x % LPR;
  if (row >= rows) return;
  const int bh = row / n_rows, t = row - bh * n_rows;
  const int64_t pos = (int64_t)cache_seqlens[bh / Hkv] - n_rows + t;
  u32x2 c{};
  uint32_t byte = 0;
  if (pos >= 0 && pos < Lmax) {
    const int64_t at = (int64_t)bh * Lmax + pos;
    const uint8_t *src = cache.codes[which] + at * CODE;
    if constexpr (BITS == 4) c[0] = reinterpret_cast<const uint32_t *>(src)[ln];
    else c = reinterpret_cast<const u32x2 *>(src)[ln];
    byte = cache.scales[which][at * (D / 32) + ln / 4];
  }
  const float scale = __uint_as_float(byte << 23);
  T *out = (which ? v : k) + (int64_t)row * D + 8 * ln;
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<bf16x8 *>(out) = mx_values8<BITS>(c, scale);
  } else {
    reinterpret_cast<f32x4 *>(out)[0] = mx_values4_f32<BITS>(c, 0, scale);
    reinterpret_cast<f32x4 *>(out)[1] = mx_values4_f32<BITS>(c, 1, scale);
  }
}

namespace {

// f(kernel tag): the instantiation of (D, bits, dtype)
template <class F>
hipError_t kv_dispatch(int D, int bits, bool f32, F f) {
  auto by_type = [&](auto d, auto b) {
    return f32 ? f(d, b, float{}) : f(d, b, bf16{});
  };
  using std::integral_constant;
  auto by_bits = [&](auto d) {
    return bits == 4 ? by_type(d, integral_constant<int, 4>{}) : by_type(d, integral_constant<int, 8>{});
  };
  return D == 64 ? by_bits(integral_constant<int, 64>{}) : by_bits(integral_constant<int, 128>{});
}

}  // namespace

hipError_t launch_kv_append(const void *k, const void *v, const int64_t (&stride)[2][3],
                            const KvCache &cache, const int *cache_seqlens, int B, int Hkv,
                            int n_rows, int Lmax, int D, int bits, bool f32, hipStream_t stream) {
  const int rows = B * Hkv * n_rows;
  return kv_dispatch(D, bits, f32, [&](auto d, auto b, auto t) {
    using T = decltype(t);
    constexpr int kD = decltype(d)::value, kBits = decltype(b)::value;
    KvRows<T> in{{(const T *)k, (const T *)v}, {}};
    for (int i = 0; i < 6; ++i) in.stride[i / 3][i % 3] = stride[i / 3][i % 3];
    const dim3 grid((unsigned)(((int64_t)rows * (kD / 8) + 255) / 256), 2);
    kv_append_mx_kernel<kD, kBits, T><<<grid, dim3(256), 0, stream>>>(in, cache, cache_seqlens, rows,
                                                                     Hkv, n_rows, Lmax);
    return hipGetLastError();
  });
}

hipError_t launch_kv_read(const KvCache &cache, const int *cache_seqlens, void *k, void *v, int B,
                          int Hkv, int n_rows, int Lmax, int D, int bits, bool f32,
                          hipStream_t stream) {
  const int rows = B * Hkv * n_rows;
  return kv_dispatch(D, bits, f32, [&](auto d, auto b, auto t) {
    using T = decltype(t);
    constexpr int kD = decltype(d)::value, kBits = decltype(b)::value;
    const dim3 grid((unsigned)(((int64_t)rows * (kD / 8) + 255) / 256), 2);
    kv_read_mx_kernel<kD, kBits, T><<<grid, dim3(256), 0, stream>>>(cache, cache_seqlens, (T *)k, (T *)v,
                                                                   rows, Hkv, n_rows, Lmax);
    return hipGetLastError();
  });
}

}  // namespace ttfa
