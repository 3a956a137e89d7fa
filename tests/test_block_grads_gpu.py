"""Gradients as autograd hands them on: an output that nothing reads, and gradients that do not start at a multiple of
16 bytes."""

import math

import pytest
import torch

from helpers import announce
from tinytrain_amd.kernels.rms_norm import add_rms_norm, rms_norm, rms_norm_fwd
from tinytrain_amd.kernels.swiglu import swiglu, swiglu_fwd
from test_block_gpu import BF, F32, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", [add_rms_norm, lambda x, r, w, eps: rms_norm_fwd(x, r, w, eps, x.dtype)],
                         ids=["native", "op"])
@pytest.mark.parametrize("xt, rt", [(BF, BF), (BF, F32), (F32, BF)])
def test_norm_that_nothing_reads(xt, rt, call):
    """Through h alone the gradient is that of the sum, also in rows that the norm makes NaN."""
    announce(f"add_rms_norm, h alone, {xt} {rt}")
    x, r, w = _rand(6, 96, seed=1, dtype=xt), _rand(6, 96, seed=2, dtype=rt), _rand(96, seed=3)
    x[1] = r[1] = 0                    # 0 / 0 with eps 0
    x[2, 5], r[4, 7] = math.nan, math.inf
    t = [v.requires_grad_() for v in (x, r, w)]
    dh = _rand(6, 96, seed=4, dtype=rt)
    dx, dr, dw = torch.autograd.grad(call(*t, 0.0)[1], t, dh, allow_unused=True)
    assert dx.dtype == xt and dr.dtype == rt
    assert torch.equal(dr, dh) and torch.equal(dx, dh.to(xt)) and (dw is None or not dw.any())


def test_norm_that_nothing_reads_compiled():
    announce("add_rms_norm, h alone, torch.compile")
    x, r, w = _rand(6, 96, seed=1, dtype=BF), _rand(6, 96, seed=2), _rand(96, seed=3)
    x[2, 5] = math.nan
    t = [v.requires_grad_() for v in (x, r, w)]
    torch._dynamo.reset()
    h = torch.compile(lambda *a: add_rms_norm(*a)[1], backend="aot_eager")(*t)
    dh = _rand(6, 96, seed=4)
    dx, dr, _ = torch.autograd.grad(h, t, dh, allow_unused=True)
    torch._dynamo.reset()
    assert torch.equal(dr, dh) and torch.equal(dx, dh.to(BF))


def _odd(t):
    """The same values, contiguous, three elements behind a multiple of 16 bytes."""
    buf = torch.empty(t.numel() + 3, device="cuda", dtype=t.dtype)
    assert buf.data_ptr() % 16 == 0
    buf[3:] = t.flatten()
    return buf[3:].view(t.shape)


@pytest.mark.parametrize("call", [lambda x, r, w: add_rms_norm(x, r, w), lambda x, r, w: rms_norm_fwd(x, r, w, 1e-6, BF),
                                  lambda x, r, w: (rms_norm(x, w), x + r)], ids=["native", "op", "alone"])
def test_norm_takes_gradients_anywhere(call):
    announce("norm, gradients off 16 bytes")
    t = [v.requires_grad_() for v in (_rand(9, 96, seed=1, dtype=BF), _rand(9, 96, seed=2), _rand(96, seed=3))]
    dy, dh = _rand(9, 96, seed=4, dtype=BF), _rand(9, 96, seed=5)
    want = torch.autograd.grad(call(*t), t, (dy, dh))
    for a, b in zip(want, torch.autograd.grad(call(*t), t, (_odd(dy), _odd(dh)))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("call", [swiglu, lambda *t: swiglu_fwd(*t, True)[0]], ids=["native", "op"])
@pytest.mark.parametrize("M", [5, 200])
def test_swiglu_takes_gradients_anywhere(M, call):
    announce(f"swiglu, gradients off 16 bytes, M={M}")
    t = [v.requires_grad_() for v in (_rand(M, 96, seed=1, dtype=BF), _rand(72, 96, seed=2, dtype=BF),
                                      _rand(72, 96, seed=3, dtype=BF))]
    da = _rand(M, 72, seed=4, dtype=BF)
    want = torch.autograd.grad(call(*t), t, da)
    for a, b in zip(want, torch.autograd.grad(call(*t), t, _odd(da))):
        assert torch.equal(a, b)


def test_gradient_of_a_concatenation():
    """Where such gradients come from: a piece of a longer row."""
    x, w, wg, wu = (v.requires_grad_() for v in (_rand(9, 96, seed=1, dtype=BF), _rand(96, seed=3),
                                                 _rand(72, 96, seed=4, dtype=BF), _rand(72, 96, seed=5, dtype=BF)))
    head, by = _rand(3, seed=6, dtype=BF), _rand(3 + 9 * 96 + 9 * 72, seed=7, dtype=BF)
    y, a = rms_norm(x, w), swiglu(x, wg, wu)
    got = torch.autograd.grad(torch.cat([head, y.flatten(), a.flatten()]), (x, w, wg, wu), by)
    y, a = rms_norm(x, w), swiglu(x, wg, wu)
    want = torch.autograd.grad((y, a), (x, w, wg, wu), (by[3:867].clone().view(9, 96), by[867:].clone().view(9, 72)))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
