"""The tiles of swiglu and its backward at sizes where they are wide, cut into parts, or several to a workgroup, every
element against 64 bits, and the forward that keeps nothing.

CASES names for each size the tiles of the forward, of dx and of the weights' gradients (test_product_cut_host.py holds
them to the rule): ``two`` and ``deep`` are 128 x 128 tiles with two and four stages, ``wide`` ones are 256 x 256 (the
forward's hold half as many columns of each weight); ``/n`` is a contraction in n parts, the number is that of all
pieces of work.  A workgroup takes more than one where that passes 512 (``two``) or 256.

Tolerances: those of test_block_gpu.py, which has the reasons.
"""

import math

import pytest
import torch

from helpers import announce
from oracle import block
from tinytrain_amd.kernels.swiglu import swiglu, swiglu_fwd
from test_block_gpu import BF, U, _check_swiglu, _rand, _within

pytestmark = pytest.mark.gpu

CASES = {
    (12000, 2056, 2056): (("wide", 799), ("wide", 423), ("wide/3", 486)),
    (14130, 520, 3416): (("wide", 1512), ("wide/3", 504), ("wide/3", 252)),
    (66, 1808, 6536): (("deep", 103), ("deep/16", 240), ("wide", 416)),
    (67, 1296, 5576): (("deep", 88), ("deep/22", 242), ("two", 968)),
    (6194, 8, 8456): (("wide", 1675), ("two/10", 490), ("two/7", 938)),
    (16507, 792, 8): (("deep", 129), ("two", 903), ("deep/18", 252)),
    (16466, 8, 400): (("two", 903), ("deep", 129), ("deep/29", 232)),
    (129, 200, 264): (("deep", 10), ("deep/10", 40), ("deep", 12)),
}


@pytest.mark.parametrize("M, K, N", CASES)
def test_every_element(M, K, N):
    announce(f"swiglu M={M} K={K} N={N} {CASES[M, K, N]}")
    a, grads = _check_swiglu(M, K, N)
    again, grads2 = _check_swiglu(M, K, N)
    assert torch.equal(a, again) and all(torch.equal(p, q) for p, q in zip(grads, grads2))


def _inputs(M, K, N):
    return (_rand(M, K, seed=1, dtype=BF),
            *(_rand(N, K, seed=s, dtype=BF, scale=1 / math.sqrt(K)) for s in (2, 3)))


@pytest.mark.parametrize("M, K, N", [*CASES, (1, 64, 72), (33, 768, 328), (64, 40, 8192)])
def test_forward_that_keeps_nothing(M, K, N):
    """Without gradients: against 64 bits, and the bits of the forward that keeps its products."""
    announce(f"swiglu without gradients M={M} K={K} N={N}")
    x, wg, wu = _inputs(M, K, N)
    a = swiglu(x, wg, wu)
    want, unit = block.swiglu(x, wg, wu)
    _within("a", a, want, 2 * K * U * unit + 2.0**-20 * want.abs())
    kept, saved = swiglu_fwd(x, wg, wu, True)
    assert saved.numel() == 5 * M * N and torch.equal(a, kept)


@pytest.mark.parametrize("M, K, N", [(12000, 264, 1032), (66, 1808, 6536), (6194, 8, 8456)])
def test_nan_stays_in_place(M, K, N):
    """NaN in rows of x: those rows of a and dx, and all of the weights' gradients; in a row of w_up: that column of a."""
    announce(f"swiglu with NaN M={M} K={K} N={N}")
    x, wg, wu = _inputs(M, K, N)
    da = _rand(M, N, seed=4, dtype=BF)

    def run(x, wu):
        t = [v.clone().requires_grad_() for v in (x, wg, wu)]
        a = swiglu(*t)
        return a.detach(), *torch.autograd.grad(a, t, da)
    a0, dx0, _, _ = run(x, wu)
    rows, cols = [3, 63, M - 1], [5, 127, N - 1]
    bad = x.clone()
    bad[rows, K - 1] = math.nan
    a, dx, dwg, dwu = run(bad, wu)
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[rows] = False
    assert torch.isnan(a[rows]).all() and torch.equal(a[keep], a0[keep])
    assert torch.isnan(dx[rows]).all() and torch.equal(dx[keep], dx0[keep])
    assert torch.isnan(dwg).all() and torch.isnan(dwu).all()
    bad = wu.clone()
    bad[cols, 0] = math.nan
    a = run(x, bad)[0]
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    keep[cols] = False
    assert torch.isnan(a[:, cols]).all() and torch.equal(a[:, keep], a0[:, keep])


STREAMS = [(1000, 136, 1032), (1300, 136, 1032)]  # both products of the backward in parts


def test_two_streams_with_parts():
    """Backward passes on two streams at the same time, each with parts of both products in its workspace: bitwise what
    each gives alone."""
    announce(f"swiglu on two streams {STREAMS}")
    wg, wu = (t.requires_grad_() for t in _inputs(*STREAMS[0])[1:])

    def step(M, K, N):
        x, da = _rand(M, K, seed=M, dtype=BF).requires_grad_(), _rand(M, N, seed=M + 1, dtype=BF)
        torch.cuda.current_stream().synchronize()
        out = []
        for _ in range(10):
            a = swiglu(x, wg, wu)
            out.append((a.detach(), *torch.autograd.grad(a, (x, wg, wu), da)))
        return out
    want = [step(*size)[-1] for size in STREAMS]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in STREAMS], []
    for s, size in zip(streams, STREAMS):
        with torch.cuda.stream(s):
            got.append(step(*size))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for g in runs:
            assert all(torch.equal(p, q) for p, q in zip(w, g))
