// Device-side conversions of the quantised element types of the KV cache and of weights (kv_cache_mx.hip
// describes the format): e2m1 (BITS 4) and e4m3 (BITS 8) with a shared power of two per 32 elements.
#pragma once

#include <type_traits>

#include "fa_common.h"

namespace ttfa {

typedef short s16x2 __attribute__((ext_vector_type(2)));

// Division of numbers below 2^31 by a number that the launch knows: a multiplication with its
// reciprocal, rounded up at 2^(31 + bits of the divisor), which is exact for them.
struct Divisor {
  uint32_t n, mul, shift;
  explicit Divisor(int d) : n((uint32_t)d), shift(0) {
    while ((1u << shift) < n) ++shift;
    mul = (uint32_t)((((uint64_t)1 << (31 + shift)) + n - 1) / n);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
    return (uint32_t)(((uint64_t)x * mul) >> 31) >> shift;
  }
};

// New rows of K (0) and V (1): [B, H, T, D] with the strides of the first three in elements.
template <class T>
struct KvRows {
  const T *x[2];
  int64_t stride[2][3];
};

// Largest of the group's 32 magnitudes: over the four lanes that hold it.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));  // lane ^ 1
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));  // lane ^ 2
}

// Byte e + 127 of a group whose largest magnitude has the fp32 bits `top`: the smallest e with
// top <= M 2^e, M = 7 = 1.75 * 2^2 or 464 = 1.8125 * 2^8 (the exponent goes up by one where the
// fraction is above M's), clamped; 255 for an infinity or NaN.
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  constexpr uint32_t frac = BITS == 4 ? 0x600000 : 0x680000;
  constexpr int shift = BITS == 4 ? 2 : 8, lo = BITS == 4 ? 2 : 10, hi = BITS == 4 ? 252 : 246;
  const int e = (int)((top + (0x7fffff - frac)) >> 23) - shift;
  return top >= 0x7f800000u ? 255u : (uint32_t)min(max(e, lo), hi);
}

// Elements 2i, 2i + 1 of eight, divided by `scale` (a power of two) and rounded to nearest even,
// into their place among the codes c.  The e2m1 conversion saturates; the e4m3 one gives NaN past
// 464, which only a clamped scale (magnitudes of 2^127 and more) can leave: hence the clamp to the
// largest value.
constexpr float kMx8Top = 448.0f * 0x1p119f;

template <int BITS>
__device__ __forceinline__ u32x2 mx_pack(u32x2 c, int i, f32x2 x, float scale) {
  if constexpr (BITS == 4) {
    uint32_t w = c[0];
    switch (i) {
      case 0: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0); break;
      case 1: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 1); break;
      case 2: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 2); break;
      default: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 3); break;
    }
    c[0] = w;
  } else {
    const float a = __builtin_amdgcn_fmed3f(x[0], -kMx8Top, kMx8Top);
    const float b = __builtin_amdgcn_fmed3f(x[1], -kMx8Top, kMx8Top);
    const uint32_t old = c[i >> 1];  // a copy: __builtin_bit_cast of a vector's element reads element 0
    s16x2 w = __builtin_bit_cast(s16x2, old);
    w = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, 1)
              : __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, 0);
    c[i >> 1] = __builtin_bit_cast(uint32_t, w);
  }
  return c;
}

template <int BITS>
__device__ __forceinline__ u32x2 mx_pack(u32x2 c, int i, bf16x2 x, float scale) {
  if constexpr (BITS == 4) {
    uint32_t w = c[0];
    switch (i) {
      case 0: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, x, scale, 0); break;
      case 1: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, x, scale, 1); break;
      case 2: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, x, scale, 2); break;
      default: w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, x, scale, 3); break;
    }
    c[0] = w;
    return c;
  } else {
    return mx_pack<BITS>(c, i, f32x2{(float)x[0], (float)x[1]}, scale);
  }
}

// Two bf16 values: elements 2i, 2i + 1 of the codes w (BITS 4: i = 0..3; BITS 8: i = 0..1).
// Only the exponent bits of `scale` count; all ones there give NaN.
template <int BITS, int I>
__device__ __forceinline__ bf16x2 mx_values2(uint32_t w, float scale) {
  if constexpr (BITS == 4) return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I);
  else return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, I);
}

// Eight bf16 values of the codes c (BITS 4: in c[0]).
template <int BITS>
__device__ __forceinline__ bf16x8 mx_values8(u32x2 c, float scale) {
  bf16x2 x[4];
  if constexpr (BITS == 4) {
    x[0] = mx_values2<4, 0>(c[0], scale);
    x[1] = mx_values2<4, 1>(c[0], scale);
    x[2] = mx_values2<4, 2>(c[0], scale);
    x[3] = mx_values2<4, 3>(c[0], scale);
  } else {
    x[0] = mx_values2<8, 0>(c[0], scale);
    x[1] = mx_values2<8, 1>(c[0], scale);
    x[2] = mx_values2<8, 0>(c[1], scale);
    x[3] = mx_values2<8, 1>(c[1], scale);
  }
  return bf16x8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
}

// Four fp32 values of the codes w (BITS 4: in its low half).
template <int BITS>
__device__ __forceinline__ f32x4 mx_values4_f32(uint32_t w, float scale) {
  f32x2 x, y;
  if constexpr (BITS == 4) {
    x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
    y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  } else {
    x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, 0);
    y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, 1);
  }
  return f32x4{x[0], x[1], y[0], y[1]};
}

}  // namespace ttfa
