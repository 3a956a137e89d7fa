"""A KV cache held in 4 or 8 bits, backed by libttfa.so (inference; no backward).

The cache of ``flash_attn_decode`` at 4.25 or 8.25 bits per element instead of 16 (the reference
regenerates the whole prefix per token, generate.py:7-20; a KV cache is on its roadmap, README.md:158):

* ``mx_cache(B, Hkv, max_seqlen, D, bits)`` allocates one;
* ``kv_cache_append(k, v, *cache, cache_seqlens)`` rounds new rows into it;
* ``flash_attn_decode_mx(q, *cache, cache_seqlens)`` attends over it;
* ``kv_cache_read(*cache, cache_seqlens, rows, dtype)`` gives rows back as plain K and V.

Format (OCP Microscaling): 32 consecutive elements of a row share a power of two 2^e, held as the byte
e + 127; the elements are e2m1 (bits 4, two to a byte, the lower one in the low nibble) or e4m3
(bits 8).  codes are uint8 [B, Hkv, max_seqlen, D * bits / 8], scales uint8 [B, Hkv, max_seqlen, D / 32];
the operators tell ``bits`` and D from these shapes.  e is the smallest integer for which the
group's largest magnitude is at most 7 * 2^e (bits 4) or 464 * 2^e (bits 8), an element x / 2^e
rounded to nearest even.  A group with a NaN or an infinity reads back as NaN.

``cache_seqlens`` [B] int32 counts the new rows already, in every one of these calls: row t of T new (or
wanted) ones of sequence b sits at position cache_seqlens[b] - T + t.  A length past max_seqlen
shifts none of them: a query attends to the keys up to its own position that the cache holds.  Rows at positions outside
0 .. max_seqlen - 1 are not written by ``kv_cache_append`` and are zeros from ``kv_cache_read``, so appending a batch
of prompts padded on the left to T rows needs no mask, and ``cache_seqlens`` filled with n makes
``kv_cache_read(..., rows=n)`` the first n rows.  (Zero rows are keys of score 0 to ``flash_attn``, which has no mask:
attention over padded prompts takes the real rows, as ``flash_attn_varlen`` does.)  A step of generation:

    cache_seqlens += 1
    kv_cache_append(k, v, *cache, cache_seqlens)          # k, v [B, Hkv, 1, D]
    o, lse = flash_attn_decode_mx(q, *cache, cache_seqlens)

Supported: D in {64, 128}; rows in bf16 or fp32 with any strides that are multiples of 16 bytes and
a dense last dimension; q in bf16, with the limits of ``flash_attn_decode``; tensors that start at a
multiple of 16 bytes; max_seqlen * D below 2^31.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from .. import _lib
from .flash_attn import FlashAttnInputError

__all__ = ["MXCache", "mx_cache", "kv_cache_append", "kv_cache_read", "flash_attn_decode_mx"]

GROUP = 32  # elements that share a scale
_DTYPES = {torch.bfloat16: _lib.TTFA_BF16, torch.float32: _lib.TTFA_F32}


class MXCache(NamedTuple):
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor


def mx_cache(B: int, Hkv: int, max_seqlen: int, D: int, bits: int = 4, device="cuda") -> MXCache:
    """An empty cache (all rows read as zeros)."""
    if bits not in (4, 8):
        raise FlashAttnInputError(f"a quantised cache holds 4 or 8 bits, not {bits}")
    if D not in (64, 128):
        raise FlashAttnInputError(f"head dim D={D} is not supported (64 or 128)")
    sizes = (D * bits // 8, D // GROUP) * 2
    return MXCache(*(torch.zeros(B, Hkv, max_seqlen, n, dtype=torch.uint8, device=device) for n in sizes))


def _check_cache(k_codes, k_scales, v_codes, v_scales, cache_seqlens):
    """(B, Hkv, max_seqlen, D, bits) of a cache and its lengths."""
    cache = (("k_codes", k_codes), ("k_scales", k_scales), ("v_codes", v_codes), ("v_scales", v_scales))
    for name, t in cache:
        if t.dim() != 4 or t.dtype != torch.uint8 or not t.is_contiguous():
            raise FlashAttnInputError(f"{name} must be a contiguous 4-D uint8 tensor")
    if k_codes.shape != v_codes.shape or k_scales.shape != v_scales.shape \
            or k_codes.shape[:3] != k_scales.shape[:3]:
        raise FlashAttnInputError(
            f"codes {tuple(k_codes.shape)}, {tuple(v_codes.shape)} and scales {tuple(k_scales.shape)}, "
            f"{tuple(v_scales.shape)} do not make one cache")
    B, Hkv, L, n = k_codes.shape
    if max(B, Hkv, L) > 0x7fffffff:
        raise FlashAttnInputError(f"a cache of {B} x {Hkv} x {L} rows is too large")
    D = GROUP * k_scales.shape[3]
    if D not in (64, 128):
        raise FlashAttnInputError(f"head dim D={D} is not supported (64 or 128)")
    if n not in (D // 2, D):
        raise FlashAttnInputError(f"codes of D={D} have {D // 2} (4 bits) or {D} (8 bits) bytes a row, not {n}")
    if cache_seqlens.shape != (B,) or cache_seqlens.dtype != torch.int32:
        raise FlashAttnInputError("cache_seqlens must be an int32 tensor [B]")
    return B, Hkv, L, D, 8 * n // D


def _check_rows(n):
    if n > 0x7fffffff:  # the C ABI's int
        raise FlashAttnInputError(f"{n} rows are too many for one call")


def _check_device(*tensors):
    for t in tensors:
        if t.device.type != "cuda" or t.device != tensors[0].device:
            raise FlashAttnInputError("all tensors must be on one ROCm GPU device")


def _strides(t: torch.Tensor) -> list[int]:
    """Element strides of the batch, head and row dimensions (0 where there is one index)."""
    s = [t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)]
    if (t.shape[3] > 1 and t.stride(3) != 1) or any(x * t.element_size() % 16 for x in s):
        raise FlashAttnInputError(
            f"rows of strides {t.stride()} need a dense last dimension and strides of multiples of "
            "16 bytes: call contiguous()")
    return s


@torch.library.custom_op("tinytrain::kv_cache_append",
                         mutates_args=("k_codes", "k_scales", "v_codes", "v_scales"))
def kv_cache_append(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                    v_codes: torch.Tensor, v_scales: torch.Tensor, cache_seqlens: torch.Tensor) -> None:
    B, Hkv, L, D, bits = _check_cache(k_codes, k_scales, v_codes, v_scales, cache_seqlens)
    if k.dim() != 4 or k.shape != v.shape or k.shape[:2] != (B, Hkv) or k.shape[3] != D:
        raise FlashAttnInputError(f"k and v must be [{B}, {Hkv}, T, {D}] for this cache; got "
                                  f"{tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise FlashAttnInputError("k and v must both be bfloat16 or float32")
    _check_rows(k.shape[2])
    strides = (ctypes.c_longlong * 6)(*_strides(k), *_strides(v))
    _check_device(k_codes, k_scales, v_codes, v_scales, cache_seqlens, k, v)
    if len({t.data_ptr() for t in (k_codes, k_scales, v_codes, v_scales)}) != 4:
        raise FlashAttnInputError("codes and scales of K and V must be four tensors")
    seqlens = cache_seqlens.contiguous()  # held until the launch is enqueued
    with torch.cuda.device(k_codes.device):
        _lib.check(_lib.load().ttfa_kv_append(
            k.data_ptr(), v.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
            v_scales.data_ptr(), seqlens.data_ptr(), strides, B, Hkv, k.shape[2], L, D, bits,
            _DTYPES[k.dtype], torch.cuda.current_stream(k_codes.device).cuda_stream))


@kv_cache_append.register_fake
def _(k, v, k_codes, k_scales, v_codes, v_scales, cache_seqlens):
    return None


@torch.library.custom_op("tinytrain::kv_cache_read", mutates_args=())
def kv_cache_read(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                  v_scales: torch.Tensor, cache_seqlens: torch.Tensor, rows: int,
                  dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    B, Hkv, L, D, bits = _check_cache(k_codes, k_scales, v_codes, v_scales, cache_seqlens)
    if rows < 1:
        raise FlashAttnInputError(f"rows must be positive, not {rows}")
    _check_rows(rows)
    if dtype not in _DTYPES:
        raise FlashAttnInputError("rows are read as bfloat16 or float32")
    _check_device(k_codes, k_scales, v_codes, v_scales, cache_seqlens)
    k, v = (torch.empty((B, Hkv, rows, D), device=k_codes.device, dtype=dtype) for _ in range(2))
    seqlens = cache_seqlens.contiguous()
    with torch.cuda.device(k_codes.device):
        _lib.check(_lib.load().ttfa_kv_read(
            k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
            seqlens.data_ptr(), k.data_ptr(), v.data_ptr(), B, Hkv, rows, L, D, bits, _DTYPES[dtype],
            torch.cuda.current_stream(k_codes.device).cuda_stream))
    return k, v


@kv_cache_read.register_fake
def _(k_codes, k_scales, v_codes, v_scales, cache_seqlens, rows, dtype=torch.bfloat16):
    shape = (*k_codes.shape[:2], rows, GROUP * k_scales.shape[3])
    return k_codes.new_empty(shape, dtype=dtype), k_codes.new_empty(shape, dtype=dtype)


@torch.library.custom_op("tinytrain::flash_attn_decode_mx", mutates_args=())
def flash_attn_decode_mx(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                         v_codes: torch.Tensor, v_scales: torch.Tensor,
                         cache_seqlens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    B, Hkv, L, D, bits = _check_cache(k_codes, k_scales, v_codes, v_scales, cache_seqlens)
    if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D:
        raise FlashAttnInputError(f"q must be [{B}, Hq, Tq, {D}] for this cache; got {tuple(q.shape)}")
    Hq, Tq = q.shape[1:3]
    if Hkv < 1 or Hq % Hkv:
        raise FlashAttnInputError(f"Hq={Hq} must be a multiple of Hkv={Hkv}")
    if (Hq // Hkv) * Tq > 32:
        raise FlashAttnInputError(f"(Hq / Hkv) * Tq = {(Hq // Hkv) * Tq} exceeds 32 query rows")
    if q.dtype != torch.bfloat16 or not q.is_contiguous():
        raise FlashAttnInputError("q must be contiguous bfloat16")
    _check_device(k_codes, k_scales, v_codes, v_scales, cache_seqlens, q)
    lib = _lib.load()
    nbytes = lib.ttfa_decode_mx_workspace_bytes(B, Hq, Hkv, Tq, L, D, bits)
    if nbytes < 0:
        _lib.check(_lib.E_SEQ)
    ws = torch.empty((nbytes // 4,), device=q.device, dtype=torch.float32) if nbytes else None
    o = torch.empty_like(q)
    lse = torch.empty((B, Hq, Tq), device=q.device, dtype=torch.float32)
    seqlens = cache_seqlens.contiguous()
    with torch.cuda.device(q.device):
        _lib.check(lib.ttfa_decode_mx_fwd(
            q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
            v_scales.data_ptr(), seqlens.data_ptr(), o.data_ptr(), lse.data_ptr(),
            ws.data_ptr() if nbytes else None, B, Hq,
            Hkv, Tq, L, D, bits, _lib.TTFA_BF16, 1.0 / math.sqrt(D),
            torch.cuda.current_stream(q.device).cuda_stream))
    return o, lse


@flash_attn_decode_mx.register_fake
def _(q, k_codes, k_scales, v_codes, v_scales, cache_seqlens):
    B, Hq, Tq, D = q.shape
    return torch.empty_like(q), q.new_empty((B, Hq, Tq), dtype=torch.float32)


# Each custom op, with plain eager calls taken by the native path (csrc/torch_native.cpp; None: the
# op's).  torch.compile and the torch.library tools see the op itself.

class _AppendNativeFirst(type(kv_cache_append)):
    def __call__(self, k, v, k_codes, k_scales, v_codes, v_scales, cache_seqlens):
        if not torch.compiler.is_compiling() and _lib.plain_cuda(k):
            if _lib.native().kv_cache_append(k, v, k_codes, k_scales, v_codes, v_scales, cache_seqlens):
                return None
        return super().__call__(k, v, k_codes, k_scales, v_codes, v_scales, cache_seqlens)


class _ReadNativeFirst(type(kv_cache_read)):
    def __call__(self, k_codes, k_scales, v_codes, v_scales, cache_seqlens, rows, dtype=torch.bfloat16):
        if not torch.compiler.is_compiling() and _lib.plain_cuda(k_codes) and dtype in _DTYPES:
            out = _lib.native().kv_cache_read(k_codes, k_scales, v_codes, v_scales, cache_seqlens, rows,
                                              _DTYPES[dtype])
            if out is not None:
                return out
        return super().__call__(k_codes, k_scales, v_codes, v_scales, cache_seqlens, rows, dtype)


class _DecodeNativeFirst(type(flash_attn_decode_mx)):
    def __call__(self, q, k_codes, k_scales, v_codes, v_scales, cache_seqlens):
        if not torch.compiler.is_compiling() and _lib.plain_cuda(q):
            out = _lib.native().flash_attn_decode_mx(q, k_codes, k_scales, v_codes, v_scales, cache_seqlens)
            if out is not None:
                return out
        return super().__call__(q, k_codes, k_scales, v_codes, v_scales, cache_seqlens)


kv_cache_append.__class__ = _AppendNativeFirst
kv_cache_read.__class__ = _ReadNativeFirst
flash_attn_decode_mx.__class__ = _DecodeNativeFirst
