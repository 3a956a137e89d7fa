"""Products with weights held in 4 or 8 bits, backed by libttfa.so (inference; no backward).

* ``mx_quantize(w, bits)`` -> (codes, scales): rounds rows [..., K] (bf16 or fp32), a weight once and for all
* ``linear_mx(x, codes, scales)`` -> x W^T in bf16, x [..., K] bf16
* ``linear_mx(x_codes, codes, scales, x_scales)``: x in 8 bits, as ``add_rms_norm_mx`` or
  ``mx_quantize(x, 8)`` gives it

W [N, K] is held as codes uint8 [N, K * bits / 8] and scales uint8 [N, K / 32], in the format of the quantised
KV cache (``kv_cache``): 32 consecutive elements of a row share a power of two; ``bits`` and K are told
from the shapes.  Sums are fp32 and y is rounded once.  With x in bf16 the products of the held values are
exact; with x in 8 bits both go to the matrix unit as they lie, which drops of every eight consecutive
products the bits below 2^-13 of the largest (on random values 2^-19 of sum |x w|, far below y's rounding).
A step of generation beside that cache:

    codes, scales, h = add_rms_norm_mx(x, h, norm_weight)
    q = linear_mx(codes, *w_q, scales)

Supported: K a multiple of 32 and N of 8, both up to 2^20; any number of rows M, none among them, for which y has
fewer than 2^23 tiles of 128 x 128 (M < 2^30, and less from N of 256 on: 2^17 - 128 at 2^20) and, in
``mx_quantize``, x no more than 2^34 - 2^13 elements; contiguous tensors that start at a multiple of 16 bytes.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .rms_norm import GROUP, BlockInputError, _check_device, _check_rows, _ptr, _stream

__all__ = ["mx_quantize", "linear_mx"]

MAX_COLS = 1 << 20
_DTYPES = {torch.bfloat16: _lib.TTFA_BF16, torch.float32: _lib.TTFA_F32}


@torch.library.custom_op("tinytrain::mx_quantize", mutates_args=())
def mx_quantize(x: torch.Tensor, bits: int = 4) -> tuple[torch.Tensor, torch.Tensor]:
    if bits not in (4, 8):
        raise BlockInputError(f"rows are held in 4 or 8 bits, not {bits}")
    if x.dtype not in _DTYPES:
        raise BlockInputError(f"x must be bfloat16 or float32, not {x.dtype}")
    _check_rows("x", x, GROUP, MAX_COLS)
    _check_device(x)
    K = x.shape[-1]
    codes = x.new_empty((*x.shape[:-1], K * bits // 8), dtype=torch.uint8)
    scales = x.new_empty((*x.shape[:-1], K // GROUP), dtype=torch.uint8)
    if x.numel():
        with torch.cuda.device(x.device):
            _lib.check(_lib.load().ttfa_mx_quantize(
                x.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.numel() // K, K, bits, _DTYPES[x.dtype],
                _stream(x.device)))
    return codes, scales


@mx_quantize.register_fake
def _(x, bits=4):
    K = x.shape[-1]
    return (x.new_empty((*x.shape[:-1], K * bits // 8), dtype=torch.uint8),
            x.new_empty((*x.shape[:-1], K // GROUP), dtype=torch.uint8))


@torch.library.custom_op("tinytrain::linear_mx", mutates_args=())
def _linear_mx(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
               x_scales: Optional[torch.Tensor]) -> torch.Tensor:
    for name, t in (("codes", codes), ("scales", scales)):
        if t.dim() != 2 or t.dtype != torch.uint8 or not t.is_contiguous():
            raise BlockInputError(f"{name} must be a contiguous 2-D uint8 tensor")
    N, K = scales.shape[0], GROUP * scales.shape[1]
    if codes.shape[0] != N or codes.shape[1] not in (K // 2, K) or not 0 < K <= MAX_COLS:
        raise BlockInputError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not make one "
                              "weight of 4 or 8 bits")
    if N < 8 or N % 8 or N > MAX_COLS:
        raise BlockInputError(f"N={N} must be a multiple of 8 up to {MAX_COLS}")
    if x.dim() < 1 or x.shape[-1] != K or not x.is_contiguous():
        raise BlockInputError(f"x must be contiguous [..., {K}] for this weight, got {tuple(x.shape)}")
    if x.dtype != (torch.bfloat16 if x_scales is None else torch.uint8):
        raise BlockInputError(f"x must be bfloat16, or uint8 codes with x_scales; got {x.dtype}")
    if x_scales is not None and (x_scales.shape != (*x.shape[:-1], K // GROUP) or x_scales.dtype != torch.uint8
                                 or not x_scales.is_contiguous()):
        raise BlockInputError(f"x_scales must be contiguous uint8 {(*x.shape[:-1], K // GROUP)}")
    _check_device(x, codes, scales, *(() if x_scales is None else (x_scales,)))
    M, bits = x.numel() // K, 8 * codes.shape[1] // K
    if M > 0x7fffffff:  # the C ABI's int
        raise BlockInputError(f"{M} rows are too many for one call")
    y = x.new_empty((*x.shape[:-1], N), dtype=torch.bfloat16)
    if M:
        lib = _lib.load()
        nbytes = lib.ttfa_linear_mx_workspace_bytes(M, K, N, bits, int(x_scales is not None))
        if nbytes < 0:
            _lib.check(_lib.E_SEQ)
        ws = torch.empty((nbytes,), device=x.device, dtype=torch.uint8) if nbytes else None
        with torch.cuda.device(x.device):
            _lib.check(lib.ttfa_linear_mx(x.data_ptr(), _ptr(x_scales), codes.data_ptr(), scales.data_ptr(),
                                          y.data_ptr(), _ptr(ws), M, K, N, bits, _stream(x.device)))
    return y


@_linear_mx.register_fake
def _(x, codes, scales, x_scales):
    return x.new_empty((*x.shape[:-1], codes.shape[0]), dtype=torch.bfloat16)


def linear_mx(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
              x_scales: torch.Tensor | None = None) -> torch.Tensor:
    """x W^T for the quantised weight (codes, scales); see module doc."""
    if not torch.compiler.is_compiling() and _lib.plain_cuda(x):
        # the native path (csrc/torch_native.cpp) for plain eager calls; None: the custom op's
        y = _lib.native().linear_mx(x, codes, scales, x_scales)
        if y is not None:
            return y
    return _linear_mx(x, codes, scales, x_scales)
