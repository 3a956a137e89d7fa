// RMSNorm over rows of C elements, with the residual's addition before it, gfx950: the two lines
// h = x + branch; y = norm(h) of the reference's block (model.py:128-139, norm :24-35) in one pass,
// its backward in one more, and the forward with an output in 8 bits.
//
//   h = x + r, rounded to r's type;  s = 1 / sqrt(mean(h^2) + eps);  y = h s w
//   d = dh + s (w dy) - h s^3 mean(h w dy);  dx = dr = d;  dw = sum over rows of dy h s
//
// y is computed from the rounded h, so the backward, which reads h again, differentiates what the
// forward computed; s is computed again there from the same h, which costs no bytes.
//
// A row belongs to L lanes (8 to 64 of a wave, or the 256 or 512 of a workgroup), 8 elements at a time:
// lane l holds chunks l, l + L, ... in registers, so every tensor is read and written once.  Sums
// are fp32 over the lanes (fp64 for the 8-bit output, whose codes are defined to the bit).
#include <type_traits>

#include "fa_common.h"
#include "fa_kernels.h"
#include "mx.h"
#include "ttfa.h"

namespace ttfa {

namespace {

struct F8 {
  float v[8];
};

__device__ __forceinline__ bf16x8 raw8(const bf16 *p) { return *reinterpret_cast<const bf16x8 *>(p); }

__device__ __forceinline__ F8 raw8(const float *p) {
  const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
  return F8{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}

// Eight elements as they lie in memory.
__device__ __forceinline__ F8 floats(const bf16x8 &b) {
  F8 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f.v[i] = (float)b[i];
  return f;
}
__device__ __forceinline__ F8 floats(const F8 &f) { return f; }

template <class T>
__device__ __forceinline__ F8 load8(const T *p) {
  return floats(raw8(p));
}

template <class T>
using Raw8 = typename std::conditional<std::is_same<T, float>::value, F8, bf16x8>::type;

__device__ __forceinline__ void store8(bf16 *p, const F8 &f) {
  bf16x8 b;
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = (bf16)f.v[i];
  *reinterpret_cast<bf16x8 *>(p) = b;
}

__device__ __forceinline__ void store8(float *p, const F8 &f) {
  reinterpret_cast<f32x4 *>(p)[0] = f32x4{f.v[0], f.v[1], f.v[2], f.v[3]};
  reinterpret_cast<f32x4 *>(p)[1] = f32x4{f.v[4], f.v[5], f.v[6], f.v[7]};
}

template <class T>
__device__ __forceinline__ float rounded(float x) {
  return (float)(T)x;
}

// The lanes of a row: L = 2^log2 of a wave, or all WT threads of the workgroup.
template <int WT>
struct Lanes {
  static constexpr int THREADS = WT ? WT : 256;
  int log2;
  __device__ __forceinline__ int count() const { return WT ? WT : 1 << log2; }
  __device__ __forceinline__ int lane() const { return WT ? threadIdx.x : threadIdx.x & ((1 << log2) - 1); }
  __device__ __forceinline__ int group() const { return WT ? 0 : threadIdx.x >> log2; }
  __device__ __forceinline__ int groups() const { return WT ? 1 : 256 >> log2; }
};

// Sum over the row's lanes; every lane gets it, from the same order of additions.  `shared` holds a
// value per wave of a workgroup's row and is free again at the next call's barrier pair.
template <int WT, class T>
__device__ __forceinline__ T row_sum(T x, const Lanes<WT> &ln, T *shared) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1)
    if (WT || m < (1 << ln.log2)) x += __shfl_xor(x, m);
  if constexpr (WT != 0) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (shared[0] + shared[1]) + (shared[2] + shared[3]);
    if constexpr (WT == 512) x += (shared[4] + shared[5]) + (shared[6] + shared[7]);
  }
  return x;
}

// h of one row in v, stored where there is a residual.
template <class TX, class TR, bool RES, int CH>
__device__ __forceinline__ void load_h(F8 (&v)[CH], const TX *x, const TR *r, TR *h, int64_t at,
                                       int ln, int L, int nch) {
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = ln + i * L;
    if (c < nch) {
      v[i] = load8(x + at + 8 * c);
      if constexpr (RES) {
        const F8 b = load8(r + at + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i].v[e] = rounded<TR>(v[i].v[e] + b.v[e]);
        store8(h + at + 8 * c, v[i]);
      }
    } else {
      v[i] = F8{};
    }
  }
}

template <class TX, class TR, class TY, bool RES, int CH, int WT>
__global__ __launch_bounds__(Lanes<WT>::THREADS) void rms_norm_fwd_kernel(const TX *__restrict__ x,
                                                           const TR *__restrict__ r,
                                                           const float *__restrict__ w,
                                                           TY *__restrict__ y, TR *__restrict__ h,
                                                           int64_t M, int nch, Lanes<WT> lanes,
                                                           float inv_c, float eps) {
  __shared__ float shared[8];
  const int ln = lanes.lane(), L = lanes.count();
  const int64_t step = (int64_t)gridDim.x * lanes.groups();
  for (int64_t row = (int64_t)blockIdx.x * lanes.groups() + lanes.group(); row < M; row += step) {
    const int64_t at = row * nch * 8;
    F8 v[CH];
    load_h<TX, TR, RES>(v, x, r, h, at, ln, L, nch);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(v[i].v[e], v[i].v[e], sum);
    const float s = 1.f / sqrtf(row_sum(sum, lanes, shared) * inv_c + eps);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = ln + i * L;
      if (c < nch) {
        const F8 k = load8(w + 8 * c);
        F8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = v[i].v[e] * s * k.v[e];
        store8(y + at + 8 * c, o);
      }
    }
  }
}

// d rounded to fp32 towards zero, the last bit set if anything was lost: rounding that to fewer bits
// gives what rounding d itself gives.
__device__ __forceinline__ float sticky(double d) {
  const float f = (float)d;
  uint32_t b = __float_as_uint(f);
  if ((double)f != d) {
    if (fabs((double)f) > fabs(d)) b -= 1;
    b |= 1;
  }
  return __uint_as_float(b);
}

// The forward with y in 8 bits: 32 elements (four lanes) share a power of two, as in the quantised
// KV cache.  Norm and product in fp64, then one rounding: in fp32 a value within 2^-20 of the middle
// between two codes could go to either, by how the sum is split over lanes.
template <class TX, class TR, bool RES, int CH, int WT>
__global__ __launch_bounds__(Lanes<WT>::THREADS) void rms_norm_mx_kernel(const TX *__restrict__ x,
                                                          const TR *__restrict__ r,
                                                          const float *__restrict__ w,
                                                          uint8_t *__restrict__ codes,
                                                          uint8_t *__restrict__ scales,
                                                          TR *__restrict__ h, int64_t M, int nch,
                                                          Lanes<WT> lanes, double eps) {
  __shared__ double shared[8];
  const int ln = lanes.lane(), L = lanes.count();
  const int64_t step = (int64_t)gridDim.x * lanes.groups();
  for (int64_t row = (int64_t)blockIdx.x * lanes.groups() + lanes.group(); row < M; row += step) {
    const int64_t at = row * nch * 8;
    F8 v[CH];
    load_h<TX, TR, RES>(v, x, r, h, at, ln, L, nch);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fma((double)v[i].v[e], (double)v[i].v[e], sum);
    const double s = 1.0 / sqrt(row_sum(sum, lanes, shared) / (double)(8 * nch) + eps);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = ln + i * L;
      if (c < nch) {  // nch is a multiple of four: whole groups of lanes
        const F8 k = load8(w + 8 * c);
        uint32_t top = 0;
        F8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          o.v[e] = sticky((double)v[i].v[e] * s * (double)k.v[e]);
          top = max(top, __float_as_uint(o.v[e]) & 0x7fffffffu);
        }
        const uint32_t byte = mx_scale_byte<8>(quad_max(top));
        const float scale = __uint_as_float(byte << 23);
        u32x2 q{};
#pragma unroll
        for (int e = 0; e < 4; ++e) q = mx_pack<8>(q, e, f32x2{o.v[2 * e], o.v[2 * e + 1]}, scale);
        if (byte == 255) q = u32x2{};
        *reinterpret_cast<u32x2 *>(codes + at + 8 * c) = q;
        if (c % 4 == 0) scales[(at + 8 * c) / 32] = (uint8_t)byte;
      }
    }
  }
}

// Backward.  Workgroups walk the rows and keep dw of their rows in registers: lane groups are added
// through LDS, the workgroup's sum goes to part[blockIdx.x] (to dw itself where it is the only one).
// TX is the type of dx where that is another than TR (dx null: d is the gradient of both).
template <class TX, class TR, class TY, int CH, int WT>
__global__ __launch_bounds__(Lanes<WT>::THREADS) void rms_norm_bwd_kernel(
    const TY *__restrict__ dy, const TR *__restrict__ dh, const TR *__restrict__ h,
    const float *__restrict__ w, TX *__restrict__ dx, TR *__restrict__ dr, float *__restrict__ part,
    int64_t M, int nch, Lanes<WT> lanes, float inv_c, float eps) {
  extern __shared__ float acc_lds[];
  __shared__ float shared[8];
  const int ln = lanes.lane(), L = lanes.count();
  const int64_t step = (int64_t)gridDim.x * lanes.groups();
  F8 acc[CH], k[CH];
  auto load_w = [&] {
#pragma unroll
    for (int i = 0; i < CH; ++i) k[i] = ln + i * L < nch ? load8(w + 8 * (ln + i * L)) : F8{};
  };
#pragma unroll
  for (int i = 0; i < CH; ++i) acc[i] = F8{};
  // The widest rows leave no registers for w, nor for the next row on its way during a row.
  constexpr bool AHEAD = WT != 512;
  if (AHEAD) load_w();
  Raw8<TR> nh[CH], nd[CH];
  Raw8<TY> ng[CH];
  auto load = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = ln + i * L;
      const bool ok = row < M && c < nch;
      const int64_t at = row * nch * 8 + 8 * c;
      nh[i] = ok ? raw8(h + at) : Raw8<TR>{};
      ng[i] = ok ? raw8(dy + at) : Raw8<TY>{};
      nd[i] = ok && dh ? raw8(dh + at) : Raw8<TR>{};
    }
  };
  int64_t row = (int64_t)blockIdx.x * lanes.groups() + lanes.group();
  if (AHEAD) load(row);
  for (; row < M; row += step) {
    if (!AHEAD) load(row);
    const int64_t at = row * nch * 8;
    F8 v[CH], g[CH], d[CH];
    float sq = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = floats(nh[i]), g[i] = floats(ng[i]), d[i] = floats(nd[i]);
    if (AHEAD) load(row + step);
    else load_w();
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sq = fmaf(v[i].v[e], v[i].v[e], sq);
        dot = fmaf(v[i].v[e], g[i].v[e] * k[i].v[e], dot);
      }
    const float s = 1.f / sqrtf(row_sum(sq, lanes, shared) * inv_c + eps);
    const float b = row_sum(dot, lanes, shared) * inv_c * s * s;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = ln + i * L;
      if (c < nch) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          d[i].v[e] += s * (g[i].v[e] * k[i].v[e] - v[i].v[e] * b);
          acc[i].v[e] = fmaf(g[i].v[e], v[i].v[e] * s, acc[i].v[e]);
        }
        store8(dr + at + 8 * c, d[i]);
        if constexpr (!std::is_same<TX, TR>::value)
          if (dx) store8(dx + at + 8 * c, d[i]);
      }
    }
  }
  float *out = part + (int64_t)blockIdx.x * nch * 8;
  if constexpr (WT != 0) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (ln + i * L < nch) store8(out + 8 * (ln + i * L), acc[i]);
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (ln + i * L < nch) store8(acc_lds + (int64_t)(lanes.group() * nch + ln + i * L) * 8, acc[i]);
    __syncthreads();
    for (int c = threadIdx.x; c < nch * 2; c += 256) {
      f32x4 t{};
      for (int q = 0; q < lanes.groups(); ++q)
        t += reinterpret_cast<const f32x4 *>(acc_lds)[q * nch * 2 + c];
      reinterpret_cast<f32x4 *>(out)[c] = t;
    }
  }
}

// dw = sum of n partials [n][C], in a fixed order: a workgroup takes 16 columns, 64 partials at once.  (512 partials
// of 768 columns: 4.0 us.  With 64 columns a workgroup, 12 of them, 1024 partials took 20.7.)
__global__ __launch_bounds__(256) void rms_norm_dw_kernel(const float *__restrict__ part,
                                                          float *__restrict__ dw, int n, int nq) {
  __shared__ f32x4 shared[64][4];
  const int col = blockIdx.x * 4 + (threadIdx.x & 3), row = threadIdx.x >> 2;
  f32x4 t{};
  if (col < nq)
#pragma unroll 8
    for (int i = row; i < n; i += 64) t += reinterpret_cast<const f32x4 *>(part)[(int64_t)i * nq + col];
  shared[row][threadIdx.x & 3] = t;
  __syncthreads();
  if (row < 8) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += shared[row + 8 * i][threadIdx.x & 3];
    shared[row][threadIdx.x & 3] = t;
  }
  __syncthreads();
  if (row == 0 && col < nq) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += shared[i][threadIdx.x];
    reinterpret_cast<f32x4 *>(dw)[col] = t;
  }
}

// How a row of nch chunks is spread: lanes (log2; 8, 9: the workgroup's), chunks a lane.
struct Spread {
  int log2, ch;
  int threads() const { return log2 == 9 ? 512 : 256; }
};

// Up to three chunks a lane, fewer where the rows would not give 512 workgroups (rows past a wave's: the workgroup's).
Spread spread_of(int nch, int64_t M) {
  for (int l = 3; l <= 6; ++l)
    if (nch <= 3 << l) {
      while (l < 6 && nch > 1 << l && M >> (8 - l) < 512) ++l;
      return {l, (nch + (1 << l) - 1) >> l};
    }
  return nch <= 256 ? Spread{8, 1} : nch <= 512 ? Spread{8, 2} : nch <= 1024 ? Spread{8, 4} : Spread{9, 4};
}

// f(chunks a lane, threads of a workgroup's row or 0) as compile-time values
template <class F>
void by_spread(const Spread &s, F f) {
  using std::integral_constant;
  using One = integral_constant<int, 1>;
  using Two = integral_constant<int, 2>;
  using Three = integral_constant<int, 3>;
  using Four = integral_constant<int, 4>;
  if (s.log2 == 9) return f(Four{}, integral_constant<int, 512>{});
  if (s.log2 == 8 && s.ch == 1) return f(One{}, integral_constant<int, 256>{});
  if (s.log2 == 8) return s.ch == 2 ? f(Two{}, integral_constant<int, 256>{}) : f(Four{}, integral_constant<int, 256>{});
  using InWave = integral_constant<int, 0>;
  if (s.ch == 1) return f(One{}, InWave{});
  if (s.ch == 2) return f(Two{}, InWave{});
  return f(Three{}, InWave{});
}

int64_t rows_of_workgroup(const Spread &s) { return s.log2 >= 8 ? 1 : 256 >> s.log2; }

// f(value of the type that dt names)
template <class F>
void by_type(int dt, F f) {
  if (dt == TTFA_F32) f(float{});
  else f(bf16{});
}

// Workgroups of a forward: one pass over the rows up to 2^20 workgroups, then each takes several.
unsigned fwd_grid(int64_t M, const Spread &s) {
  const int64_t per = rows_of_workgroup(s), n = (M + per - 1) / per;
  return (unsigned)(n < 1 << 20 ? n : 1 << 20);
}

}  // namespace

constexpr int kMostParts = 512;  // workgroups of a backward: what is resident at once, two a CU

int rms_norm_bwd_parts(int64_t M, int C) {
  const Spread s = spread_of(C / 8, M);
  const int64_t per = rows_of_workgroup(s), n = (M + per - 1) / per;
  return (int)(n < kMostParts ? n : kMostParts);
}

hipError_t launch_rms_norm_fwd(const void *x, const void *r, const float *w, void *y, void *h,
                               int64_t M, int C, int x_dtype, int r_dtype, int y_dtype, double eps,
                               hipStream_t stream) {
  const int nch = C / 8;
  const Spread sp = spread_of(nch, M);
  const dim3 grid(fwd_grid(M, sp));
  by_spread(sp, [&](auto ch, auto wide) {
    by_type(x_dtype, [&](auto tx) {
      by_type(y_dtype, [&](auto ty) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        constexpr int CH = decltype(ch)::value;
        constexpr int W = decltype(wide)::value;
        if (r)
          by_type(r_dtype, [&](auto tr) {
            using TR = decltype(tr);
            rms_norm_fwd_kernel<TX, TR, TY, true, CH, W><<<grid, dim3(sp.threads()), 0, stream>>>(
                (const TX *)x, (const TR *)r, w, (TY *)y, (TR *)h, M, nch, Lanes<W>{sp.log2}, 1.f / C,
                (float)eps);
          });
        else
          rms_norm_fwd_kernel<TX, TX, TY, false, CH, W><<<grid, dim3(sp.threads()), 0, stream>>>(
              (const TX *)x, nullptr, w, (TY *)y, nullptr, M, nch, Lanes<W>{sp.log2}, 1.f / C, (float)eps);
      });
    });
  });
  return hipGetLastError();
}

hipError_t launch_rms_norm_mx(const void *x, const void *r, const float *w, void *codes, void *scales,
                              void *h, int64_t M, int C, int x_dtype, int r_dtype, double eps,
                              hipStream_t stream) {
  const int nch = C / 8;
  const Spread sp = spread_of(nch, M);
  const dim3 grid(fwd_grid(M, sp));
  by_spread(sp, [&](auto ch, auto wide) {
    by_type(x_dtype, [&](auto tx) {
      using TX = decltype(tx);
      constexpr int CH = decltype(ch)::value;
      constexpr int W = decltype(wide)::value;
      if (r)
        by_type(r_dtype, [&](auto tr) {
          using TR = decltype(tr);
          rms_norm_mx_kernel<TX, TR, true, CH, W><<<grid, dim3(sp.threads()), 0, stream>>>(
              (const TX *)x, (const TR *)r, w, (uint8_t *)codes, (uint8_t *)scales, (TR *)h, M, nch,
              Lanes<W>{sp.log2}, eps);
        });
      else
        rms_norm_mx_kernel<TX, TX, false, CH, W><<<grid, dim3(sp.threads()), 0, stream>>>(
            (const TX *)x, nullptr, w, (uint8_t *)codes, (uint8_t *)scales, nullptr, M, nch,
            Lanes<W>{sp.log2}, eps);
    });
  });
  return hipGetLastError();
}

hipError_t launch_rms_norm_bwd(const void *dy, const void *dh, const void *h, const float *w, void *dx,
                               void *dr, float *dw, float *part, int64_t M, int C, int r_dtype,
                               int y_dtype, double eps, hipStream_t stream) {
  const int nch = C / 8, parts = rms_norm_bwd_parts(M, C);
  const Spread sp = spread_of(nch, M);
  float *out = parts == 1 ? dw : part;
  by_spread(sp, [&](auto ch, auto wide) {
    by_type(r_dtype, [&](auto tr) {
      by_type(y_dtype, [&](auto ty) {
        using TR = decltype(tr);
        using TY = decltype(ty);
        using TX = typename std::conditional<std::is_same<TR, float>::value, bf16, float>::type;
        constexpr int W = decltype(wide)::value;
        const size_t lds = W != 0 ? 0 : (size_t)(256 >> sp.log2) * C * sizeof(float);
        rms_norm_bwd_kernel<TX, TR, TY, decltype(ch)::value, W><<<dim3(parts), dim3(sp.threads()), lds, stream>>>(
            (const TY *)dy, (const TR *)dh, (const TR *)h, w, (TX *)dx, (TR *)dr, out, M, nch,
            Lanes<W>{sp.log2}, 1.f / C, (float)eps);
      });
    });
  });
  if (parts > 1)
    rms_norm_dw_kernel<<<dim3((C / 4 + 3) / 4), dim3(256), 0, stream>>>(part, dw, parts, C / 4);
  return hipGetLastError();
}

}  // namespace ttfa
