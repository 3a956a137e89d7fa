"""Gated feed-forward input, backed by libttfa.so: both projections, the activation and their product.

    a = silu(x @ w_gate.T) * (x @ w_up.T)

what the reference's MLP (model.py:111-125) does before its down projection, as one kernel: the two
products stay in fp32 registers, and a is rounded to bf16 once.

``swiglu(x, w_gate, w_up)``: x [..., K], w_gate and w_up [N, K], bf16, contiguous; a [..., N].  Gradients
flow to all three.  Where one is needed, the forward keeps both products for it, in 20 bits each (12
significant: 5 bytes an element of a); the backward rounds the gradients of both to bf16 once, as operands
of the products that give dx and the weights' gradients.
Where x or both weights need no gradient, theirs is not computed.  Sums have a fixed order: results are
bitwise reproducible.

Supported: K and N multiples of 8 up to 2^20; any number of rows M, none among them, for which each of a, dx and
the two weights' gradients together has fewer than 2^23 tiles of 128 x 128 (M < 2^30, and less from N or K of
256 on: 2^17 - 128 at 2^20); tensors that start at a multiple of 16 bytes, gradients anywhere.
"""

from __future__ import annotations

import torch

from .. import _lib
from .rms_norm import BlockInputError, _check_device, _check_rows, _laid_out, _stream

__all__ = ["swiglu", "swiglu_fwd", "swiglu_bwd"]

MAX_COLS = 1 << 20


def _check(x, w_gate, w_up):
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up)):
        if t.dtype != torch.bfloat16:
            raise BlockInputError(f"{name} must be bfloat16, not {t.dtype}")
        _check_rows(name, t, 8, MAX_COLS)
    if w_gate.dim() != 2 or w_gate.shape != w_up.shape or w_gate.shape[1] != x.shape[-1]:
        raise BlockInputError(f"w_gate and w_up must be [N, {x.shape[-1]}], got {tuple(w_gate.shape)} and "
                              f"{tuple(w_up.shape)}")
    N = w_gate.shape[0]
    if N < 8 or N % 8 or N > MAX_COLS:
        raise BlockInputError(f"N={N} must be a multiple of 8 up to {MAX_COLS}")
    _check_device(x, w_gate, w_up)
    M = x.numel() // x.shape[-1]
    if M > 0x7fffffff:  # the C ABI's int
        raise BlockInputError(f"{M} rows are too many for one call")
    return M, x.shape[-1], N


def _bytes(n, device):
    if n < 0:
        _lib.check(_lib.E_SEQ)
    return torch.empty((n,), device=device, dtype=torch.uint8)


@torch.library.custom_op("tinytrain::swiglu_fwd", mutates_args=())
def swiglu_fwd(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, save: bool
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """(a, what the backward needs, or empty)."""
    M, K, N = _check(x, w_gate, w_up)
    a = x.new_empty((*x.shape[:-1], N))
    lib = _lib.load()
    saved = _bytes(lib.ttfa_swiglu_saved_bytes(M, N) if save and M else 0, x.device)
    if M:
        with torch.cuda.device(x.device):
            _lib.check(lib.ttfa_swiglu_fwd(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), a.data_ptr(),
                                           saved.data_ptr() if save else None, M, K, N, _stream(x.device)))
    return a, saved


@swiglu_fwd.register_fake
def _(x, w_gate, w_up, save):
    M, N = x.numel() // x.shape[-1], w_gate.shape[0]
    return x.new_empty((*x.shape[:-1], N)), x.new_empty(5 * M * N if save else 0, dtype=torch.uint8)


@torch.library.custom_op("tinytrain::swiglu_bwd", mutates_args=())
def swiglu_bwd(da: torch.Tensor, saved: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
               need_dx: bool, need_dw: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw_gate, dw_up); what is not needed is empty."""
    M, K, N = _check(x, w_gate, w_up)
    if da.shape != (*x.shape[:-1], N) or da.dtype != x.dtype or da.device != x.device:
        raise BlockInputError(f"da must be bfloat16 {(*x.shape[:-1], N)} beside x")
    if saved.numel() == 0 and M:  # a forward that kept nothing
        saved = swiglu_fwd(x, w_gate, w_up, True)[1]
    if saved.shape != (5 * M * N,) or saved.dtype != torch.uint8 or saved.device != x.device:
        raise BlockInputError(f"saved must be the forward's {5 * M * N} bytes beside x")
    dx = torch.empty_like(x) if need_dx else x.new_empty(0)
    make = torch.empty_like if M else torch.zeros_like
    dwg, dwu = (make(w_gate), make(w_up)) if need_dw else (x.new_empty(0), x.new_empty(0))
    if M and (need_dx or need_dw):
        da, saved, lib = _laid_out(da), _laid_out(saved), _lib.load()
        ws = _bytes(lib.ttfa_swiglu_workspace_bytes(M, K, N), x.device)
        with torch.cuda.device(x.device):
            _lib.check(lib.ttfa_swiglu_bwd(
                da.data_ptr(), saved.data_ptr(), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
                dx.data_ptr() if need_dx else None, dwg.data_ptr() if need_dw else None,
                dwu.data_ptr() if need_dw else None, ws.data_ptr(), M, K, N, _stream(x.device)))
    return dx, dwg, dwu


@swiglu_bwd.register_fake
def _(da, saved, x, w_gate, w_up, need_dx, need_dw):
    none = x.new_empty(0)
    return (torch.empty_like(x) if need_dx else none,
            torch.empty_like(w_gate) if need_dw else x.new_empty(0),
            torch.empty_like(w_up) if need_dw else x.new_empty(0))


def _setup_context(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:3], output[1])
    ctx.mark_non_differentiable(output[1])


def _backward_fn(ctx, da, _):
    x, w_gate, w_up, saved = ctx.saved_tensors
    need_x, need_g, need_u, _ = ctx.needs_input_grad
    dx, dwg, dwu = swiglu_bwd(da, saved, x, w_gate, w_up, need_x, need_g or need_u)
    return dx if need_x else None, dwg if need_g else None, dwu if need_u else None, None


swiglu_fwd.register_autograd(_backward_fn, setup_context=_setup_context)


def swiglu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    """silu(x @ w_gate.T) * (x @ w_up.T); see module doc."""
    if not torch.compiler.is_compiling() and _lib.plain_cuda(x):
        # the native path (csrc/torch_native.cpp) for plain eager calls; None: the custom op's
        a = _lib.native().swiglu(x, w_gate, w_up)
        if a is not None:
            return a
    save = torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad)
    return swiglu_fwd(x, w_gate, w_up, save)[0]
