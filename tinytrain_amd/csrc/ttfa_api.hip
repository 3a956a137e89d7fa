// C ABI of libttfa.so: argument validation and dispatch (declarations in include/ttfa.h).
//
// Validation runs before any HIP call, so every argument error is reported without a
// GPU (and without touching the HIP runtime).  Launch failures come back as the
// positive hipError_t of hipGetLastError().
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "ttfa.h"
#include "fa_kernels.h"

// Delta rows of ttfa_bwd_static: a file-scope device array, one copy per GPU the library
// runs on, held until the process ends.  Host code never passes `scratch` itself to a
// kernel (in host code the name is a stand-in, not a device address): it passes the
// per-device address hipGetSymbolAddress returns (static_scratch_ptr below).
static __device__ __align__(256) float scratch[TTFA_BWD_STATIC_MAX_ROWS];

namespace {

int check_common(int B, int Hq, int Hkv, int T, int D, int dtype, float scale) {
  if (dtype != TTFA_BF16 && dtype != TTFA_F32) return TTFA_E_DTYPE;
  if (D != 64 && D != 128) return TTFA_E_HEAD_DIM;
  if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0) return TTFA_E_GROUP;
  if (B < 1 || T < 1) return TTFA_E_SEQ;
  // Per-head byte extents must fit the 32-bit buffer descriptors used by the kernels,
  // and total element counts must fit int64 with margin.
  const int64_t esz = dtype == TTFA_BF16 ? 2 : 4;
  if ((int64_t)T * D * esz > (int64_t)0x7fffffff) return TTFA_E_SEQ;
  if ((int64_t)B * Hq > (int64_t)0x7fffffff / 4) return TTFA_E_SEQ;
  if ((int64_t)B * Hq * ((T + 127) / 128) > (int64_t)0x7fffffff) return TTFA_E_SEQ;
  // fp32 grids: one workgroup per 16-row block of every query and KV head.
  if (dtype == TTFA_F32 && (int64_t)B * (Hq + Hkv) * ((T + 15) / 16) > (int64_t)0x7fffffff)
    return TTFA_E_SEQ;
  if (!(scale > 0.f) || !isfinite(scale)) return TTFA_E_SCALE;
  return TTFA_OK;
}

// Packed variable-length sequences: bf16 only; n_seq, total, max_seqlen >= 1; per-
// sequence byte extents within the 32-bit buffer descriptors; grids within int range.
int check_varlen(int n_seq, int total, int max_seqlen, int Hq, int Hkv, int D, int dtype,
                 float scale) {
  if (dtype != TTFA_BF16) return TTFA_E_DTYPE;
  if (D != 64 && D != 128) return TTFA_E_HEAD_DIM;
  if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0) return TTFA_E_GROUP;
  if (n_seq < 1 || total < 1 || max_seqlen < 1) return TTFA_E_SEQ;
  if ((int64_t)max_seqlen * D * 2 > (int64_t)0x7fffffff) return TTFA_E_SEQ;
  if ((int64_t)((max_seqlen + 127) / 128) * n_seq * Hq > (int64_t)0x7fffffff) return TTFA_E_SEQ;
  if ((int64_t)Hq * total > (int64_t)0x7fffffff) return TTFA_E_SEQ;
  if (!(scale > 0.f) || !isfinite(scale)) return TTFA_E_SCALE;
  return TTFA_OK;
}

// KV-cache decode: bf16; G * Tq query columns fit one 32-wide MFMA tile; cache byte
// extents within the 32-bit buffer descriptors.
int check_decode(int B, int Hq, int Hkv, int Tq, int Lmax, int D, int dtype, float scale) {
  if (dtype != TTFA_BF16) return TTFA_E_DTYPE;
  if (D != 64 && D != 128) return TTFA_E_HEAD_DIM;
  if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0) return TTFA_E_GROUP;
  if (B < 1 || Tq < 1 || Lmax < 1) return TTFA_E_SEQ;
  if ((int64_t)(Hq / Hkv) * Tq > 32) return TTFA_E_QROWS;
  if ((int64_t)Lmax * D * 2 > (int64_t)0x7fffffff) return TTFA_E_SEQ;
  if ((int64_t)B * Hq * Tq > (int64_t)0x7fffffff / 4) return TTFA_E_SEQ;
  if (!(scale > 0.f) || !isfinite(scale)) return TTFA_E_SCALE;
  return TTFA_OK;
}

// Quantised KV cache of rows of D elements: extents of one head within 32-bit byte offsets.
int check_kv(int B, int Hkv, int max_seqlen, int D, int bits) {
  if (bits != 4 && bits != 8) return TTFA_E_BITS;
  if (D != 64 && D != 128) return TTFA_E_HEAD_DIM;
  if (Hkv < 1) return TTFA_E_GROUP;
  if (B < 1 || max_seqlen < 1) return TTFA_E_SEQ;
  if ((int64_t)max_seqlen * D > (int64_t)0x7fffffff) return TTFA_E_SEQ;
  if ((int64_t)B * Hkv > (int64_t)0x7fffffff / 4) return TTFA_E_SEQ;
  return TTFA_OK;
}

// Rows moved in or out of it: a launch has fewer than 2^32 threads, of four elements at least each,
// and a last workgroup that may be part empty.
int check_kv_rows(int B, int Hkv, int rows, int max_seqlen, int D, int bits, int dtype) {
  if (dtype != TTFA_BF16 && dtype != TTFA_F32) return TTFA_E_DTYPE;
  const int rc = check_kv(B, Hkv, max_seqlen, D, bits);
  if (rc) return rc;
  const int64_t most = (((int64_t)1 << 34) - (1 << 13)) / D;
  return rows < 1 || (int64_t)rows > most / ((int64_t)B * Hkv) ? TTFA_E_SEQ : TTFA_OK;
}

int check_decode_mx(int B, int Hq, int Hkv, int Tq, int max_seqlen, int D, int bits, int dtype,
                    float scale) {
  int rc = check_kv(B, Hkv, max_seqlen, D, bits);
  if (!rc && (int64_t)B * Hkv >= 1 << 24) rc = TTFA_E_SEQ;  // workgroups of 256 threads, 2^32 in all
  // a length of 1 in place of max_seqlen, which check_kv holds to bytes of fewer bits
  return rc ? rc : check_decode(B, Hq, Hkv, Tq, 1, D, dtype, scale);
}

int check_seqlens(const int *cache_seqlens) {
  if (cache_seqlens == nullptr) return TTFA_E_NULL;
  return reinterpret_cast<uintptr_t>(cache_seqlens) & 3u ? TTFA_E_ALIGN : TTFA_OK;
}

ttfa::KvCache kv_cache(const void *k_codes, const void *k_scales, const void *v_codes,
                       const void *v_scales) {
  auto p = [](const void *x) { return const_cast<uint8_t *>(static_cast<const uint8_t *>(x)); };
  return {{p(k_codes), p(v_codes)}, {p(k_scales), p(v_scales)}};
}

// Device address of `scratch` on the current device, resolved once per device (the first
// ttfa_bwd_static call on it) and cached; *out stays null on failure.
hipError_t static_scratch_ptr(float **out) {
  static std::atomic<uintptr_t> addr[64];  // by device ordinal, 0 = not resolved yet
  *out = nullptr;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
  uintptr_t a = addr[dev].load(std::memory_order_acquire);
  if (a == 0) {
    void *ptr = nullptr;
    e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return e;
    if (ptr == nullptr) return hipErrorInvalidSymbol;
    a = reinterpret_cast<uintptr_t>(ptr);
    addr[dev].store(a, std::memory_order_release);
  }
  *out = reinterpret_cast<float *>(a);
  return hipSuccess;
}

int check_ptrs(const void *const *ptrs, int n) {
  for (int i = 0; i < n; ++i)
    if (ptrs[i] == nullptr) return TTFA_E_NULL;
  for (int i = 0; i < n; ++i)
    if (reinterpret_cast<uintptr_t>(ptrs[i]) & 15u) return TTFA_E_ALIGN;
  return TTFA_OK;
}

bool is_dtype(int dtype) { return dtype == TTFA_BF16 || dtype == TTFA_F32; }

// M rows of C elements, C a multiple of `unit` up to `most`; total elements within int64 with margin.
int check_rows(int64_t M, int C, int unit, int most) {
  if (C < unit || C % unit || C > most) return TTFA_E_COLS;
  return M < 1 || M > ((int64_t)1 << 40) / C ? TTFA_E_SEQ : TTFA_OK;
}

int check_norm(int64_t M, int C, int unit, int x_dtype, int r_dtype, int y_dtype, double eps) {
  if (!is_dtype(x_dtype) || !is_dtype(r_dtype) || !is_dtype(y_dtype)) return TTFA_E_DTYPE;
  if (!(eps >= 0.0) || !(eps < 1.0)) return TTFA_E_EPS;
  return check_rows(M, C, unit, 16384);
}

// The residual and its sum, which come together or not at all, after the other pointers.
int check_residual(const void *const *ptrs, int n, const void *residual, const void *h) {
  const int rc = check_ptrs(ptrs, n);
  if (rc || (!residual && !h)) return rc;
  const void *pair[] = {residual, h};
  return check_ptrs(pair, 2);
}

constexpr int kMostCols = 1 << 20;  // of a product: a tile's byte offsets stay within 31 bits

// Tiles of tm x tn of a result: their number fits an int with room for its parts.
int check_tiles(int64_t M, int64_t N, int tm, int tn) {
  return (M + tm - 1) / tm * ((N + tn - 1) / tn) < 1 << 23 ? TTFA_OK : TTFA_E_SEQ;
}

int check_swiglu(int M, int K, int N) {
  int rc = check_rows(M, K, 8, kMostCols);
  if (rc || (rc = check_rows(M, N, 8, kMostCols))) return rc;
  if ((rc = check_tiles(M, N, 128, 128)) || (rc = check_tiles(M, K, 128, 128))) return rc;
  return check_tiles(2ll * N, K, 128, 128);
}

int check_linear_mx(int M, int K, int N, int bits) {
  if (bits != 4 && bits != 8) return TTFA_E_BITS;
  int rc = check_rows(M, K, 32, kMostCols);
  if (rc || (rc = check_rows(M, N, 8, kMostCols))) return rc;
  return check_tiles(M, N, 128, 128);
}

// The workspace of ttfa_bwd_ws: Delta rows, padded to 16 bytes, then the dK/dV partials.
int64_t delta_floats(int B, int Hq, int T) { return ((int64_t)B * Hq * T + 3) / 4 * 4; }

ttfa::DkdvSplit split_of(int B, int Hq, int Hkv, int T, int D, int dtype) {
  return dtype == TTFA_BF16 ? ttfa::dkdv_split(B, Hq, Hkv, T, D)
                            : ttfa::dkdv_split_f32(B, Hq, Hkv, T, D);
}

}  // namespace

extern "C" {

int ttfa_abi_version(void) { return TTFA_ABI_VERSION; }

int ttfa_d128_wide(int B, int Hq, int T, int *fwd_wide, int *dq_wide) {
  if (!fwd_wide || !dq_wide) return TTFA_E_NULL;
  if (B < 1 || Hq < 1 || T < 1) return TTFA_E_SEQ;
  *fwd_wide = ttfa::fwd128_uses_wide(B, Hq, T) ? 1 : 0;
  *dq_wide = ttfa::dq128_uses_wide(B, Hq, T) ? 1 : 0;
  return TTFA_OK;
}

const char *ttfa_strerror(int code) {
  switch (code) {
    case TTFA_OK: return "success";
    case TTFA_E_NULL: return "ttfa: a required pointer is NULL";
    case TTFA_E_HEAD_DIM: return "ttfa: head dim D must be 64 or 128";
    case TTFA_E_GROUP: return "ttfa: Hq must be a positive multiple of Hkv";
    case TTFA_E_SEQ: return "ttfa: B and T must be >= 1 and sizes must fit the kernels' index range";
    case TTFA_E_ALIGN: return "ttfa: every pointer must be 16-byte aligned";
    case TTFA_E_DTYPE: return "ttfa: dtype must be TTFA_BF16 or TTFA_F32";
    case TTFA_E_SCALE: return "ttfa: scale must be finite and > 0";
    case TTFA_E_EPS: return "ttfa: eps must be in [0, 1)";
    case TTFA_E_QROWS: return "ttfa: decode needs (Hq / Hkv) * Tq <= 32 query rows per KV head";
    case TTFA_E_BITS: return "ttfa: a quantised cache or weight holds elements of 4 or 8 bits";
    case TTFA_E_STRIDE: return "ttfa: strides must be multiples of 16 bytes and not negative";
    case TTFA_E_COLS:
      return "ttfa: row lengths must be multiples of 8 (32 where rows are quantised) and in range";
    case TTFA_E_SCRATCH:
      return "ttfa: ttfa_bwd_static needs B * Hq * T <= TTFA_BWD_STATIC_MAX_ROWS (1048576)";
    default: break;
  }
  if (code > 0) return hipGetErrorString(static_cast<hipError_t>(code));
  return "ttfa: unknown status code";
}

int ttfa_fwd(const void *q, const void *k, const void *v, void *o, float *lse, int B, int Hq,
             int Hkv, int T, int D, int dtype, float scale, void *hip_stream) {
  int rc = check_common(B, Hq, Hkv, T, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k, v, o, lse};
  if ((rc = check_ptrs(ptrs, 5))) return rc;
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  hipError_t e = dtype == TTFA_BF16
                     ? ttfa::launch_fwd_bf16(q, k, v, o, lse, B, Hq, Hkv, T, D, scale, s)
                     : ttfa::launch_fwd_f32(q, k, v, o, lse, B, Hq, Hkv, T, D, scale, s);
  return static_cast<int>(e);
}

int ttfa_bwd_dq(const void *q, const void *k, const void *v, const void *o, const void *dout,
                const float *lse, float *delta_ws, void *dq, int B, int Hq, int Hkv, int T,
                int D, int dtype, float scale, void *hip_stream) {
  int rc = check_common(B, Hq, Hkv, T, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k, v, o, dout, lse, delta_ws, dq};
  if ((rc = check_ptrs(ptrs, 8))) return rc;
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  hipError_t e =
      dtype == TTFA_BF16
          ? ttfa::launch_bwd_dq_bf16(q, k, v, o, dout, lse, delta_ws, dq, B, Hq, Hkv, T, D, scale, s)
          : ttfa::launch_bwd_dq_f32(q, k, v, o, dout, lse, delta_ws, dq, B, Hq, Hkv, T, D, scale, s);
  return static_cast<int>(e);
}

int ttfa_bwd_dkdv(const void *q, const void *k, const void *v, const void *dout,
                  const float *lse, const float *delta_ws, void *dk, void *dv, int B, int Hq,
                  int Hkv, int T, int D, int dtype, float scale, void *hip_stream) {
  int rc = check_common(B, Hq, Hkv, T, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k, v, dout, lse, delta_ws, dk, dv};
  if ((rc = check_ptrs(ptrs, 8))) return rc;
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  hipError_t e =
      dtype == TTFA_BF16
          ? ttfa::launch_bwd_dkdv_bf16(q, k, v, dout, lse, delta_ws, dk, dv, B, Hq, Hkv, T, D, scale, s)
          : ttfa::launch_bwd_dkdv_f32(q, k, v, dout, lse, delta_ws, dk, dv, B, Hq, Hkv, T, D, scale, s);
  return static_cast<int>(e);
}

int ttfa_varlen_fwd(const void *q, const void *k, const void *v, void *o, float *lse,
                    const int *cu_seqlens, int n_seq, int total, int max_seqlen, int Hq, int Hkv,
                    int D, int dtype, float scale, void *hip_stream) {
  int rc = check_varlen(n_seq, total, max_seqlen, Hq, Hkv, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k, v, o, lse};
  if ((rc = check_ptrs(ptrs, 5))) return rc;
  if (cu_seqlens == nullptr) return TTFA_E_NULL;
  if (reinterpret_cast<uintptr_t>(cu_seqlens) & 3u) return TTFA_E_ALIGN;
  return static_cast<int>(ttfa::launch_fwd_varlen_bf16(q, k, v, o, lse, cu_seqlens, n_seq, total,
                                                       max_seqlen, Hq, Hkv, D, scale,
                                                       static_cast<hipStream_t>(hip_stream)));
}

int ttfa_varlen_bwd(const void *q, const void *k, const void *v, const void *o,
                    const void *dout, const float *lse, float *delta_ws, void *dq, void *dk,
                    void *dv, const int *cu_seqlens, int n_seq, int total, int max_seqlen,
                    int Hq, int Hkv, int D, int dtype, float scale, void *hip_stream) {
  int rc = check_varlen(n_seq, total, max_seqlen, Hq, Hkv, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k, v, o, dout, lse, delta_ws, dq, dk, dv};
  if ((rc = check_ptrs(ptrs, 10))) return rc;
  if (cu_seqlens == nullptr) return TTFA_E_NULL;
  if (reinterpret_cast<uintptr_t>(cu_seqlens) & 3u) return TTFA_E_ALIGN;
  return static_cast<int>(ttfa::launch_bwd_varlen_bf16(
      q, k, v, o, dout, lse, delta_ws, dq, dk, dv, cu_seqlens, n_seq, total, max_seqlen, Hq, Hkv,
      D, scale, static_cast<hipStream_t>(hip_stream)));
}

long long ttfa_decode_workspace_bytes(int B, int Hq, int Hkv, int Tq, int max_seqlen, int D) {
  if (check_decode(B, Hq, Hkv, Tq, max_seqlen, D, TTFA_BF16, 1.f)) return -1;
  const ttfa::DecodeSplit sp = ttfa::decode_split(B, Hkv, max_seqlen, D);
  return (long long)B * Hq * Tq * sp.n_chunks * (D + 2) * (long long)sizeof(float);
}

int ttfa_decode_fwd(const void *q, const void *k_cache, const void *v_cache,
                    const int *cache_seqlens, void *o, float *lse, float *workspace, int B,
                    int Hq, int Hkv, int Tq, int max_seqlen, int D, int dtype, float scale,
                    void *hip_stream) {
  int rc = check_decode(B, Hq, Hkv, Tq, max_seqlen, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k_cache, v_cache, o, lse, workspace};
  if ((rc = check_ptrs(ptrs, 6))) return rc;
  if (cache_seqlens == nullptr) return TTFA_E_NULL;
  if (reinterpret_cast<uintptr_t>(cache_seqlens) & 3u) return TTFA_E_ALIGN;
  return static_cast<int>(ttfa::launch_decode_bf16(q, k_cache, v_cache, cache_seqlens, o, lse,
                                                   workspace, B, Hq, Hkv, Tq, max_seqlen, D,
                                                   scale, static_cast<hipStream_t>(hip_stream)));
}

int ttfa_kv_append(const void *k, const void *v, void *k_codes, void *k_scales, void *v_codes,
                   void *v_scales, const int *cache_seqlens, const long long *strides, int B, int Hkv,
                   int rows, int max_seqlen, int D, int bits, int dtype, void *hip_stream) {
  int rc = check_kv_rows(B, Hkv, rows, max_seqlen, D, bits, dtype);
  if (rc) return rc;
  const void *ptrs[] = {k, v, k_codes, k_scales, v_codes, v_scales};
  if ((rc = check_ptrs(ptrs, 6)) || (rc = check_seqlens(cache_seqlens))) return rc;
  const int64_t most = (int64_t)1 << 40, unit = dtype == TTFA_BF16 ? 8 : 4;
  int64_t st[2][3];
  const int64_t dense[3] = {(int64_t)Hkv * rows * D, (int64_t)rows * D, D};
  for (int i = 0; i < 6; ++i) {
    const int64_t x = strides ? strides[i] : dense[i % 3];
    if (x < 0 || x % unit || x > most) return TTFA_E_STRIDE;
    st[i / 3][i % 3] = x;
  }
  return static_cast<int>(ttfa::launch_kv_append(
      k, v, st, kv_cache(k_codes, k_scales, v_codes, v_scales), cache_seqlens, B, Hkv, rows,
      max_seqlen, D, bits, dtype == TTFA_F32, static_cast<hipStream_t>(hip_stream)));
}

int ttfa_kv_read(const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales,
                 const int *cache_seqlens, void *k, void *v, int B, int Hkv, int rows, int max_seqlen,
                 int D, int bits, int dtype, void *hip_stream) {
  int rc = check_kv_rows(B, Hkv, rows, max_seqlen, D, bits, dtype);
  if (rc) return rc;
  const void *ptrs[] = {k_codes, k_scales, v_codes, v_scales, k, v};
  if ((rc = check_ptrs(ptrs, 6)) || (rc = check_seqlens(cache_seqlens))) return rc;
  return static_cast<int>(ttfa::launch_kv_read(
      kv_cache(k_codes, k_scales, v_codes, v_scales), cache_seqlens, k, v, B, Hkv, rows, max_seqlen, D,
      bits, dtype == TTFA_F32, static_cast<hipStream_t>(hip_stream)));
}

long long ttfa_decode_mx_workspace_bytes(int B, int Hq, int Hkv, int Tq, int max_seqlen, int D,
                                         int bits) {
  if (check_decode_mx(B, Hq, Hkv, Tq, max_seqlen, D, bits, TTFA_BF16, 1.f)) return -1;
  const ttfa::DecodeSplit sp = ttfa::decode_mx_split(B, Hkv, max_seqlen, D);
  if (sp.n_chunks == 1) return 0;
  return (long long)B * Hq * Tq * sp.n_chunks * (D + 2) * (long long)sizeof(float);
}

int ttfa_decode_mx_fwd(const void *q, const void *k_codes, const void *k_scales, const void *v_codes,
                       const void *v_scales, const int *cache_seqlens, void *o, float *lse,
                       float *workspace, int B, int Hq, int Hkv, int Tq, int max_seqlen, int D,
                       int bits, int dtype, float scale, void *hip_stream) {
  int rc = check_decode_mx(B, Hq, Hkv, Tq, max_seqlen, D, bits, dtype, scale);
  if (rc) return rc;
  const bool one = ttfa::decode_mx_split(B, Hkv, max_seqlen, D).n_chunks == 1;
  const void *ptrs[] = {q, k_codes, k_scales, v_codes, v_scales, o, lse, workspace};
  if ((rc = check_ptrs(ptrs, one ? 7 : 8)) || (rc = check_seqlens(cache_seqlens))) return rc;
  return static_cast<int>(ttfa::launch_decode_mx(
      q, kv_cache(k_codes, k_scales, v_codes, v_scales), cache_seqlens, o, lse, workspace, B, Hq, Hkv,
      Tq, max_seqlen, D, bits, scale, static_cast<hipStream_t>(hip_stream)));
}

int ttfa_bwd(const void *q, const void *k, const void *v, const void *o, const void *dout,
             const float *lse, float *delta_ws, void *dq, void *dk, void *dv, int B, int Hq,
             int Hkv, int T, int D, int dtype, float scale, void *hip_stream) {
  int rc = check_common(B, Hq, Hkv, T, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k, v, o, dout, lse, delta_ws, dq, dk, dv};
  if ((rc = check_ptrs(ptrs, 10))) return rc;
  if (dtype == TTFA_F32)
    return static_cast<int>(ttfa::launch_bwd_f32(q, k, v, o, dout, lse, delta_ws, dq, dk, dv,
                                                 nullptr, ttfa::DkdvSplit{0, 0, 0}, B, Hq, Hkv, T,
                                                 D, scale,
                                                 static_cast<hipStream_t>(hip_stream)));
  rc = ttfa_bwd_dq(q, k, v, o, dout, lse, delta_ws, dq, B, Hq, Hkv, T, D, dtype, scale, hip_stream);
  if (rc) return rc;
  return ttfa_bwd_dkdv(q, k, v, dout, lse, delta_ws, dk, dv, B, Hq, Hkv, T, D, dtype, scale,
                       hip_stream);
}

long long ttfa_bwd_workspace_bytes(int B, int Hq, int Hkv, int T, int D, int dtype) {
  if (check_common(B, Hq, Hkv, T, D, dtype, 1.f)) return -1;
  const ttfa::DkdvSplit sp = split_of(B, Hq, Hkv, T, D, dtype);
  return 4ll * (delta_floats(B, Hq, T) + (dtype == TTFA_BF16
                                              ? ttfa::dkdv_part_floats(sp, B, Hkv, D)
                                              : ttfa::dkdv_part_floats_f32(sp, B, Hkv, D)));
}

int ttfa_bwd_ws(const void *q, const void *k, const void *v, const void *o, const void *dout,
                const float *lse, float *workspace, void *dq, void *dk, void *dv, int B, int Hq,
                int Hkv, int T, int D, int dtype, float scale, void *hip_stream) {
  int rc = check_common(B, Hq, Hkv, T, D, dtype, scale);
  if (rc) return rc;
  const void *ptrs[] = {q, k, v, o, dout, lse, workspace, dq, dk, dv};
  if ((rc = check_ptrs(ptrs, 10))) return rc;
  const ttfa::DkdvSplit sp = split_of(B, Hq, Hkv, T, D, dtype);
  if (sp.stages == 0)
    return ttfa_bwd(q, k, v, o, dout, lse, workspace, dq, dk, dv, B, Hq, Hkv, T, D, dtype, scale,
                    hip_stream);
  float *part = workspace + delta_floats(B, Hq, T);
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  if (dtype == TTFA_F32)
    return static_cast<int>(ttfa::launch_bwd_f32(q, k, v, o, dout, lse, workspace, dq, dk, dv, part,
                                                 sp, B, Hq, Hkv, T, D, scale, s));
  rc = ttfa_bwd_dq(q, k, v, o, dout, lse, workspace, dq, B, Hq, Hkv, T, D, dtype, scale, hip_stream);
  if (rc) return rc;
  return static_cast<int>(ttfa::launch_bwd_dkdv_split_bf16(q, k, v, dout, lse, workspace, dk, dv,
                                                           part, sp, B, Hq, Hkv, T, D, scale, s));
}

int ttfa_bwd_static(const void *q, const void *k, const void *v, const void *o,
                    const void *dout, const float *lse, void *dq, void *dk, void *dv, int B,
                    int Hq, int Hkv, int T, int D, int dtype, float scale, void *hip_stream) {
  int rc = check_common(B, Hq, Hkv, T, D, dtype, scale);
  if (rc) return rc;
  if ((int64_t)B * Hq * T > TTFA_BWD_STATIC_MAX_ROWS) return TTFA_E_SCRATCH;
  const void *ptrs[] = {q, k, v, o, dout, lse, dq, dk, dv};
  if ((rc = check_ptrs(ptrs, 9))) return rc;
  float *delta = nullptr;
  hipError_t e = static_scratch_ptr(&delta);
  if (e != hipSuccess) return static_cast<int>(e);
  // Every call writes all B * Hq * T rows of Delta (dQ pass) before the dK/dV pass reads
  // them, so nothing left by an earlier call is ever read and nothing needs clearing.
  return ttfa_bwd(q, k, v, o, dout, lse, delta, dq, dk, dv, B, Hq, Hkv, T, D, dtype, scale,
                  hip_stream);
}

int ttfa_rms_norm_fwd(const void *x, const void *residual, const float *w, void *y, void *h,
                      long long M, int C, int x_dtype, int r_dtype, int y_dtype, double eps,
                      void *hip_stream) {
  int rc = check_norm(M, C, 8, x_dtype, residual ? r_dtype : x_dtype, y_dtype, eps);
  if (rc) return rc;
  const void *ptrs[] = {x, w, y};
  if ((rc = check_residual(ptrs, 3, residual, h))) return rc;
  return static_cast<int>(ttfa::launch_rms_norm_fwd(x, residual, w, y, h, M, C, x_dtype, r_dtype, y_dtype,
                                                    eps, static_cast<hipStream_t>(hip_stream)));
}

int ttfa_rms_norm_mx(const void *x, const void *residual, const float *w, void *codes, void *scales,
                     void *h, long long M, int C, int x_dtype, int r_dtype, double eps,
                     void *hip_stream) {
  int rc = check_norm(M, C, 32, x_dtype, residual ? r_dtype : x_dtype, TTFA_BF16, eps);
  if (rc) return rc;
  const void *ptrs[] = {x, w, codes, scales};
  if ((rc = check_residual(ptrs, 4, residual, h))) return rc;
  return static_cast<int>(ttfa::launch_rms_norm_mx(x, residual, w, codes, scales, h, M, C, x_dtype, r_dtype,
                                                   eps, static_cast<hipStream_t>(hip_stream)));
}

long long ttfa_rms_norm_workspace_bytes(long long M, int C) {
  if (check_rows(M, C, 8, 16384)) return -1;
  const int parts = ttfa::rms_norm_bwd_parts(M, C);
  return parts == 1 ? 0 : (long long)parts * C * (long long)sizeof(float);
}

int ttfa_rms_norm_bwd(const void *dy, const void *dh, const void *h, const float *w, void *dx, void *dr,
                      float *dw, float *workspace, long long M, int C, int r_dtype, int y_dtype,
                      double eps, void *hip_stream) {
  int rc = check_norm(M, C, 8, r_dtype, r_dtype, y_dtype, eps);
  if (rc) return rc;
  const bool one = ttfa::rms_norm_bwd_parts(M, C) == 1;
  const void *ptrs[] = {dy, h, w, dr, dw, dh ? dh : dr, dx ? dx : dr, workspace};
  if ((rc = check_ptrs(ptrs, one ? 7 : 8))) return rc;
  return static_cast<int>(ttfa::launch_rms_norm_bwd(dy, dh, h, w, dx, dr, dw, workspace, M, C, r_dtype,
                                                    y_dtype, eps, static_cast<hipStream_t>(hip_stream)));
}

long long ttfa_swiglu_saved_bytes(int M, int N) {
  return check_swiglu(M, 8, N) ? -1 : ttfa::swiglu_saved_bytes(M, N);
}

int ttfa_swiglu_fwd(const void *x, const void *w_gate, const void *w_up, void *a, void *saved, int M, int K,
                    int N, void *hip_stream) {
  int rc = check_swiglu(M, K, N);
  if (rc) return rc;
  const void *ptrs[] = {x, w_gate, w_up, a, saved ? saved : a};
  if ((rc = check_ptrs(ptrs, 5))) return rc;
  return static_cast<int>(
      ttfa::launch_swiglu_fwd(x, w_gate, w_up, a, saved, M, K, N, static_cast<hipStream_t>(hip_stream)));
}

long long ttfa_swiglu_workspace_bytes(int M, int K, int N) {
  return check_swiglu(M, K, N) ? -1 : ttfa::swiglu_bwd_workspace(M, K, N);
}

int ttfa_swiglu_bwd(const void *da, const void *saved, const void *x, const void *w_gate, const void *w_up,
                    void *dx, void *dw_gate, void *dw_up, void *workspace, int M, int K, int N,
                    void *hip_stream) {
  int rc = check_swiglu(M, K, N);
  if (rc) return rc;
  if (!dx && !dw_gate) return TTFA_E_NULL;
  if (!dw_gate != !dw_up) return TTFA_E_NULL;
  const void *ptrs[] = {da, saved, x, w_gate, w_up, workspace, dx ? dx : x, dw_gate ? dw_gate : x, dw_up ? dw_up : x};
  if ((rc = check_ptrs(ptrs, 9))) return rc;
  return static_cast<int>(ttfa::launch_swiglu_bwd(da, saved, x, w_gate, w_up, dx, dw_gate, dw_up, workspace, M,
                                                  K, N, static_cast<hipStream_t>(hip_stream)));
}

int ttfa_mx_quantize(const void *x, void *codes, void *scales, long long M, int K, int bits, int dtype,
                     void *hip_stream) {
  if (!is_dtype(dtype)) return TTFA_E_DTYPE;
  if (bits != 4 && bits != 8) return TTFA_E_BITS;
  int rc = check_rows(M, K, 32, kMostCols);
  if (rc) return rc;
  if (M > (((int64_t)1 << 34) - (1 << 13)) / K) return TTFA_E_SEQ;  // launches of fewer than 2^32 threads
  const void *ptrs[] = {x, codes, scales};
  if ((rc = check_ptrs(ptrs, 3))) return rc;
  return static_cast<int>(ttfa::launch_mx_quantize(x, codes, scales, M * K, bits, dtype == TTFA_F32,
                                                   static_cast<hipStream_t>(hip_stream)));
}

long long ttfa_linear_mx_workspace_bytes(int M, int K, int N, int bits, int x_quantised) {
  return check_linear_mx(M, K, N, bits) ? -1 : ttfa::linear_mx_workspace(M, K, N, x_quantised != 0);
}

int ttfa_linear_mx(const void *x, const void *x_scales, const void *codes, const void *scales, void *y,
                   void *workspace, int M, int K, int N, int bits, void *hip_stream) {
  int rc = check_linear_mx(M, K, N, bits);
  if (rc) return rc;
  const void *ptrs[] = {x, codes, scales, y, x_scales ? x_scales : x, workspace};
  if ((rc = check_ptrs(ptrs, ttfa_linear_mx_workspace_bytes(M, K, N, bits, x_scales != nullptr) ? 6 : 5)))
    return rc;
  return static_cast<int>(ttfa::launch_linear_mx(x, x_scales, codes, scales, y, workspace, M, K, N, bits,
                                                 static_cast<hipStream_t>(hip_stream)));
}

}  // extern "C"
