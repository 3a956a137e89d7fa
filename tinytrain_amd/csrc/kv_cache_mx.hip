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
// hardware conversions do in one step (tested against the definition with every bf16 value, and
// with every rounding border and its fp32 neighbours under every e).  x 2^-e is exact, so the cache is defined
// to the bit.  e is clamped so that every value is a finite normal bf16; a group with a NaN or an
// infinity gets the byte 255, which the conversions read back as NaN.
#include "fa_common.h"
#include "fa_kernels.h"
#include "mx.h"

namespace ttfa {

namespace {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

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

// Rows moved by a call are numbered (b, h, t).
//
// A lane takes eight elements, D / 8 lanes a row, U rows of a lane at once; blockIdx.y picks K or V.
// Row t of T goes to position cache_seqlens[b] - T + t; one outside the cache is not written.
// Bound by memory: 16 x 8 rows of up to 4000, D 128, bf16 to 4 bits 47 us (copy rate: 45).
template <int D, int BITS, class T, int U>
__global__ __launch_bounds__(256) void kv_append_mx_kernel(KvRows<T> in, KvCache cache,
                                                           const int *__restrict__ cache_seqlens,
                                                           int rows, Divisor heads, Divisor per_head,
                                                           int Lmax) {
  constexpr int LPR = D / 8, CODE = D * BITS / 8, STEP = 256 / LPR;
  const int which = blockIdx.y;
  const int row0 = blockIdx.x * (STEP * U) + threadIdx.x / LPR, ln = threadIdx.x % LPR;
  const int64_t *st = in.stride[which];
  Eight<T> x[U];
  int64_t at[U];  // position in the cache, over all heads; -1: not written
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t row = row0 + u * STEP;
    at[u] = -1;
    if (row < (uint32_t)rows) {  // whole rows, so whole groups of lanes
      const uint32_t bh = per_head.quotient(row), t = row - bh * per_head.n;
      const uint32_t b = heads.quotient(bh), h = bh - b * heads.n;
      const int64_t pos = (int64_t)cache_seqlens[b] - per_head.n + t;
      if (pos >= 0 && pos < Lmax) {
        at[u] = (int64_t)bh * Lmax + pos;
        x[u].load(in.x[which] + b * st[0] + h * st[1] + t * st[2] + 8 * ln);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] < 0) continue;
    const uint32_t byte = mx_scale_byte<BITS>(quad_max(x[u].top()));
    u32x2 c = x[u].template codes<BITS>(__uint_as_float(byte << 23));
    if (byte == 255) c = u32x2{};
    uint8_t *out = cache.codes[which] + at[u] * CODE;
    if constexpr (BITS == 4) reinterpret_cast<uint32_t *>(out)[ln] = c[0];
    else reinterpret_cast<u32x2 *>(out)[ln] = c;
    if (ln % 4 == 0) cache.scales[which][at[u] * (D / 32) + ln / 4] = (uint8_t)byte;
  }
}

// The inverse: row t of n_rows comes from position cache_seqlens[b] - n_rows + t, zeros where that
// lies outside the cache.  A lane writes 16 bytes, so that every store instruction writes whole lines, past
// the L2 (the rows are read by another kernel, mostly after more of them than it holds).  Bound by memory:
// 16 x 8 x 4000 rows of D 128 in 4 bits 60 us, through the L2 76 (copy rate: 63).  With a kernel behind it that
// reads the rows at once, in us, first past the L2: 8 MB of rows 8.4, 8.4; 34 MB 22.4, 21.2; 67 MB 39.0, 36.8;
// 134 MB 69.5, 70.3; as fp32 67 MB 39.4, 37.6; 537 MB 272, 294.
template <int D, int BITS, class T, int U>
__global__ __launch_bounds__(256) void kv_read_mx_kernel(KvCache cache,
                                                         const int *__restrict__ cache_seqlens,
                                                         T *__restrict__ k, T *__restrict__ v, int rows,
                                                         Divisor heads, Divisor per_head, int Lmax) {
  constexpr int E = 16 / sizeof(T), LPR = D / E, CODE = D * BITS / 8, STEP = 256 / LPR;
  constexpr int BYTES = E * BITS / 8;  // of a lane's codes: 2, 4 or 8
  const int which = blockIdx.y;
  const int row0 = blockIdx.x * (STEP * U) + threadIdx.x / LPR, ln = threadIdx.x % LPR;
  u32x2 c[U];
  uint32_t byte[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t row = row0 + u * STEP;
    c[u] = u32x2{};
    byte[u] = 0;
    if (row < (uint32_t)rows) {
      const uint32_t bh = per_head.quotient(row), t = row - bh * per_head.n;
      const int64_t pos = (int64_t)cache_seqlens[heads.quotient(bh)] - per_head.n + t;
      if (pos >= 0 && pos < Lmax) {
        const int64_t at = (int64_t)bh * Lmax + pos;
        const uint8_t *src = cache.codes[which] + at * CODE;
        if constexpr (BYTES == 2) c[u][0] = reinterpret_cast<const uint16_t *>(src)[ln];
        else if constexpr (BYTES == 4) c[u][0] = reinterpret_cast<const uint32_t *>(src)[ln];
        else c[u] = reinterpret_cast<const u32x2 *>(src)[ln];
        byte[u] = cache.scales[which][at * (D / 32) + ln * E / 32];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = row0 + u * STEP;
    if (row >= rows) continue;
    const float scale = __uint_as_float(byte[u] << 23);
    T *out = (which ? v : k) + (int64_t)row * D + E * ln;
    if constexpr (sizeof(T) == 2)
      __builtin_nontemporal_store(mx_values8<BITS>(c[u], scale), reinterpret_cast<bf16x8 *>(out));
    else
      __builtin_nontemporal_store(mx_values4_f32<BITS>(c[u][0], scale), reinterpret_cast<f32x4 *>(out));
  }
}

// Plain rows into the format (weights, activations): a lane takes eight elements, one after the other over
// all rows, whose length is a multiple of a group.  Bound by memory: 12288 x 4096 bf16 into 4 bits 23 us (5.5 TB/s), into
// 8 bits 27 (5.7); fp32 38 (6.1) and 40 (6.4).
template <int BITS, class T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *__restrict__ x, uint8_t *__restrict__ codes,
                                                          uint8_t *__restrict__ scales, int64_t lanes) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= lanes) return;  // whole groups of lanes
  Eight<T> v;
  v.load(x + 8 * i);
  const uint32_t byte = mx_scale_byte<BITS>(quad_max(v.top()));
  u32x2 c = v.template codes<BITS>(__uint_as_float(byte << 23));
  if (byte == 255) c = u32x2{};
  if constexpr (BITS == 4) reinterpret_cast<uint32_t *>(codes)[i] = c[0];
  else reinterpret_cast<u32x2 *>(codes)[i] = c;
  if (i % 4 == 0) scales[i / 4] = (uint8_t)byte;
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

// f(rows of a lane at once, grid) for `rows` rows of `lanes` lanes each.  Two rows at once keep more
// loads on the way, which pays for some moves (TWO) of 2^21 lanes, of eight elements there, or more: appends
// of bf16 81.7 -> 74.0 us at 16 x 8 x 4000 rows of D 128 in 8 bits, reads of 8 bits as bf16 74.4 -> 66.1, and
// 22.4 -> 20.4 at 2^21 lanes; small calls, which leave CUs idle, lose (2.5 -> 2.8 at 32 x 8 rows).  The others
// lose: appends of fp32 28.2 -> 29.5 at 2 x 8 x 8192, reads of 4 bits 19.6 -> 21.3 at 8 x 16384, reads of 8
// bits as fp32, of four elements a lane, 15.7 -> 16.1 at 2^21 lanes and 67.0 -> 68.5 at 2^23.
template <bool TWO, class F>
hipError_t kv_launch(int rows, int lanes, F f) {
  auto go = [&](auto u) {
    const int64_t per = 256 / lanes * decltype(u)::value;
    f(u, dim3((unsigned)((rows + per - 1) / per), 2));
    return hipGetLastError();
  };
  if constexpr (TWO)
    if ((int64_t)rows * lanes >= 1 << 21) return go(std::integral_constant<int, 2>{});
  return go(std::integral_constant<int, 1>{});
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
    return kv_launch<sizeof(T) == 2>(rows, kD / 8, [&](auto u, dim3 grid) {
      kv_append_mx_kernel<kD, kBits, T, decltype(u)::value><<<grid, dim3(256), 0, stream>>>(
          in, cache, cache_seqlens, rows, Divisor(Hkv), Divisor(n_rows), Lmax);
    });
  });
}

hipError_t launch_kv_read(const KvCache &cache, const int *cache_seqlens, void *k, void *v, int B,
                          int Hkv, int n_rows, int Lmax, int D, int bits, bool f32,
                          hipStream_t stream) {
  const int rows = B * Hkv * n_rows;
  return kv_dispatch(D, bits, f32, [&](auto d, auto b, auto t) {
    using T = decltype(t);
    constexpr int kD = decltype(d)::value, kBits = decltype(b)::value;
    return kv_launch<kBits == 8 && sizeof(T) == 2>(rows, kD * (int)sizeof(T) / 16, [&](auto u, dim3 grid) {
      kv_read_mx_kernel<kD, kBits, T, decltype(u)::value><<<grid, dim3(256), 0, stream>>>(
          cache, cache_seqlens, (T *)k, (T *)v, rows, Divisor(Hkv), Divisor(n_rows), Lmax);
    });
  });
}

hipError_t launch_mx_quantize(const void *x, void *codes, void *scales, int64_t elements, int bits,
                              bool f32, hipStream_t stream) {
  const int64_t lanes = elements / 8;
  auto go = [&](auto b, auto t) {
    using T = decltype(t);
    mx_quantize_kernel<decltype(b)::value, T><<<dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, stream>>>(
        (const T *)x, (uint8_t *)codes, (uint8_t *)scales, lanes);
    return hipGetLastError();
  };
  using std::integral_constant;
  if (bits == 4) return f32 ? go(integral_constant<int, 4>{}, float{}) : go(integral_constant<int, 4>{}, bf16{});
  return f32 ? go(integral_constant<int, 8>{}, float{}) : go(integral_constant<int, 8>{}, bf16{});
}

}  // namespace ttfa
