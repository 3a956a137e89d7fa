"""RMSNorm with the residual's addition before it, backed by libttfa.so.

What a block of the reference does between its attention and its feed-forward, and between two blocks
(model.py:128-139, norm :24-35):

    h = residual + x                 # x: a branch's output
    y = norm(h)

* ``add_rms_norm(x, residual, weight, eps)`` -> (y, h)
* ``rms_norm(x, weight, eps)`` -> y, the norm alone
* ``add_rms_norm_mx(x, residual, weight, eps)`` -> (codes, scales, h): y in 8 bits, what ``linear_mx`` takes
  (inference; residual may be None, h is x then)

x and residual [..., C], each bf16 or fp32, contiguous; weight [C].  h has residual's type: the sum is
formed in fp32 and rounded to it, and y is computed from that h in fp32 and rounded to ``dtype`` (x's if
not given), so a residual stream in fp32 with branches in bf16, as under autocast, is one call.

Gradients flow to x, residual and weight, through y and h; they may come in any strides.  They are those of the formula at the h that
was returned; dx and dresidual are one tensor where their types are.  The weight's is summed in a fixed
order.  (codes, scales) is the format of the quantised KV cache: 32 elements share a power of two, e4m3
elements rounded once from a 64-bit y; a group with a NaN or an infinity reads as NaN.

Supported: C a multiple of 8 (32 for ``add_rms_norm_mx``) up to 16384; any number of rows, none among
them, up to 2^40 elements; tensors that start at a multiple of 16 bytes, gradients anywhere; eps in [0, 1).
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib

__all__ = ["add_rms_norm", "rms_norm", "add_rms_norm_mx", "BlockInputError"]

GROUP = 32
MAX_COLS = 16384
_DTYPES = {torch.bfloat16: _lib.TTFA_BF16, torch.float32: _lib.TTFA_F32}


class BlockInputError(ValueError):
    """Inputs outside the contract of the block's operators."""


def _check_device(*tensors):
    for t in tensors:
        if t.device.type != "cuda" or t.device != tensors[0].device:
            raise BlockInputError("all tensors must be on one ROCm GPU device (the HIP library is the only "
                                  "implementation)")


def _check_rows(name: str, t: torch.Tensor, unit: int, most: int) -> None:
    if t.dim() < 1 or t.shape[-1] < unit or t.shape[-1] % unit or t.shape[-1] > most:
        raise BlockInputError(f"{name} must have rows of a multiple of {unit} elements up to {most}, got "
                              f"{tuple(t.shape)}")
    if not t.is_contiguous():
        raise BlockInputError(f"{name} must be contiguous")


def _check(x, residual, weight, unit):
    _check_rows("x", x, unit, MAX_COLS)
    if x.dtype not in _DTYPES:
        raise BlockInputError(f"x must be bfloat16 or float32, not {x.dtype}")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype not in _DTYPES:
            raise BlockInputError(f"residual must be bfloat16 or float32 {tuple(x.shape)}, got "
                                  f"{residual.dtype} {tuple(residual.shape)}")
        if not residual.is_contiguous():
            raise BlockInputError("residual must be contiguous")
    if weight.shape != x.shape[-1:] or not weight.is_floating_point():
        raise BlockInputError(f"weight must be [{x.shape[-1]}], got {weight.dtype} {tuple(weight.shape)}")
    _check_device(x, weight, *(() if residual is None else (residual,)))


def _laid_out(g: torch.Tensor) -> torch.Tensor:
    """A gradient as the library takes it: contiguous, and from a multiple of 16 bytes on, which a piece of a
    longer tensor's gradient need not be."""
    g = g.contiguous()
    return g.clone() if g.data_ptr() % 16 else g


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


@torch.library.custom_op("tinytrain::rms_norm_fwd", mutates_args=())
def rms_norm_fwd(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float,
                 dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h); h is empty without a residual."""
    _check(x, residual, weight, 8)
    if dtype not in _DTYPES:
        raise BlockInputError(f"y is bfloat16 or float32, not {dtype}")
    y = torch.empty_like(x, dtype=dtype)
    h = x.new_empty(0) if residual is None else torch.empty_like(residual)
    if x.numel():
        w = weight.float().contiguous()
        with torch.cuda.device(x.device):
            _lib.check(_lib.load().ttfa_rms_norm_fwd(
                x.data_ptr(), _ptr(residual), w.data_ptr(), y.data_ptr(),
                None if residual is None else h.data_ptr(), x.numel() // x.shape[-1], x.shape[-1],
                _DTYPES[x.dtype], _DTYPES[(x if residual is None else residual).dtype], _DTYPES[dtype],
                float(eps), _stream(x.device)))
    return y, h


@rms_norm_fwd.register_fake
def _(x, residual, weight, eps, dtype):
    return (torch.empty_like(x, dtype=dtype),
            x.new_empty(0) if residual is None else torch.empty_like(residual))


@torch.library.custom_op("tinytrain::rms_norm_bwd", mutates_args=())
def rms_norm_bwd(dy: torch.Tensor, dh: Optional[torch.Tensor], h: torch.Tensor, weight: torch.Tensor,
                 eps: float, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(gradient in h's type, the same in ``dtype`` or empty where that is h's, dweight)."""
    _check(h, None, weight, 8)
    if dy.shape != h.shape or dy.dtype not in _DTYPES or dtype not in _DTYPES:
        raise BlockInputError("dy must have h's shape, and it and dx be bfloat16 or float32")
    if dh is not None and (dh.shape != h.shape or dh.dtype != h.dtype):
        raise BlockInputError("dh must match h in shape and dtype")
    _check_device(h, dy, *(() if dh is None else (dh,)))
    dr = torch.empty_like(h)
    dx = h.new_empty(0, dtype=dtype) if dtype == h.dtype else torch.empty_like(h, dtype=dtype)
    dw = torch.zeros_like(weight, dtype=torch.float32) if h.numel() == 0 \
        else torch.empty(weight.shape, dtype=torch.float32, device=h.device)
    if h.numel():
        dy, dh = _laid_out(dy), None if dh is None else _laid_out(dh)
        w, M, C, lib = weight.float().contiguous(), h.numel() // h.shape[-1], h.shape[-1], _lib.load()
        nbytes = lib.ttfa_rms_norm_workspace_bytes(M, C)
        if nbytes < 0:
            _lib.check(_lib.E_SEQ)
        ws = torch.empty((nbytes // 4,), device=h.device, dtype=torch.float32) if nbytes else None
        with torch.cuda.device(h.device):
            _lib.check(lib.ttfa_rms_norm_bwd(
                dy.data_ptr(), _ptr(dh), h.data_ptr(), w.data_ptr(),
                None if dtype == h.dtype else dx.data_ptr(), dr.data_ptr(), dw.data_ptr(), _ptr(ws), M, C,
                _DTYPES[h.dtype], _DTYPES[dy.dtype], float(eps), _stream(h.device)))
    return dr, dx, dw.to(weight.dtype)


@rms_norm_bwd.register_fake
def _(dy, dh, h, weight, eps, dtype):
    return (torch.empty_like(h), h.new_empty(0, dtype=dtype) if dtype == h.dtype
            else torch.empty_like(h, dtype=dtype), torch.empty_like(weight))


def _setup_context(ctx, inputs, output):
    x, residual, weight, eps, _ = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x if residual is None else output[1], weight)
    ctx.eps, ctx.x_dtype, ctx.added = eps, x.dtype, residual is not None


def _backward_fn(ctx, dy, dh):
    h, weight = ctx.saved_tensors
    if dy is None:  # h alone was read: the sum's gradient (zeros through the norm would make NaN rows' NaN)
        dh = dh if ctx.added else None
        return None if dh is None else dh.to(ctx.x_dtype), dh, None, None, None
    dr, dx, dw = rms_norm_bwd(dy, dh if ctx.added else None, h, weight, ctx.eps, ctx.x_dtype)
    return dr if ctx.x_dtype == h.dtype else dx, dr if ctx.added else None, dw, None, None


rms_norm_fwd.register_autograd(_backward_fn, setup_context=_setup_context)


@torch.library.custom_op("tinytrain::rms_norm_mx", mutates_args=())
def rms_norm_mx(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, h); h is empty without a residual."""
    _check(x, residual, weight, GROUP)
    codes = torch.empty_like(x, dtype=torch.uint8)
    scales = x.new_empty((*x.shape[:-1], x.shape[-1] // GROUP), dtype=torch.uint8)
    h = x.new_empty(0) if residual is None else torch.empty_like(residual)
    if x.numel():
        w = weight.float().contiguous()
        with torch.cuda.device(x.device):
            _lib.check(_lib.load().ttfa_rms_norm_mx(
                x.data_ptr(), _ptr(residual), w.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                None if residual is None else h.data_ptr(), x.numel() // x.shape[-1], x.shape[-1],
                _DTYPES[x.dtype], _DTYPES[(x if residual is None else residual).dtype], float(eps),
                _stream(x.device)))
    return codes, scales, h


@rms_norm_mx.register_fake
def _(x, residual, weight, eps):
    return (torch.empty_like(x, dtype=torch.uint8),
            x.new_empty((*x.shape[:-1], x.shape[-1] // GROUP), dtype=torch.uint8),
            x.new_empty(0) if residual is None else torch.empty_like(residual))


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                 dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = residual + x, y its norm; see module doc."""
    if residual is not None and not torch.compiler.is_compiling() and _lib.plain_cuda(x) \
            and (dtype is None or dtype in _DTYPES):
        # the native path (csrc/torch_native.cpp) for plain eager calls; None: the custom op's
        out = _lib.native().add_rms_norm(x, residual, weight, float(eps),
                                         -1 if dtype is None else _DTYPES[dtype])
        if out is not None:
            return out
    if residual is None:
        raise BlockInputError("residual is missing: rms_norm is the norm alone")
    return rms_norm_fwd(x, residual, weight, float(eps), x.dtype if dtype is None else dtype)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             dtype: torch.dtype | None = None) -> torch.Tensor:
    """The norm of x; see module doc."""
    if not torch.compiler.is_compiling() and _lib.plain_cuda(x) and (dtype is None or dtype in _DTYPES):
        out = _lib.native().add_rms_norm(x, None, weight, float(eps), -1 if dtype is None else _DTYPES[dtype])
        if out is not None:
            return out
    return rms_norm_fwd(x, None, weight, float(eps), x.dtype if dtype is None else dtype)[0]


def add_rms_norm_mx(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                    eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, h): ``add_rms_norm`` with y in 8 bits; see module doc."""
    if not torch.compiler.is_compiling() and _lib.plain_cuda(x):
        out = _lib.native().add_rms_norm_mx(x, residual, weight, float(eps))
        if out is not None:
            return out
    codes, scales, h = rms_norm_mx(x, residual, weight, float(eps))
    return codes, scales, x if residual is None else h
