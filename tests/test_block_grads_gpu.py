"""Gradients as autograd hands them on: an output that nothing reads."""

import math

import pytest
import torch

from helpers import announce
from tinytrain_amd.kernels.rms_norm import add_rms_norm, rms_norm_fwd
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
