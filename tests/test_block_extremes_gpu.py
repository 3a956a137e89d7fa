"""The block's operators at the ends of what they take: the longest rows and most columns, more rows than a launch has
workgroups for, more than 2^31 elements, and NaN of every kind.

Long sums are made of small whole numbers, which fp32 adds exactly, so nothing but the result's rounding is allowed for;
many rows are one run of them over and over, whose every repetition gives the bits of a call of that run alone.
"""

import pytest
import torch

from helpers import announce
from oracle import mx_cache
from tinytrain_amd.kernels.linear_mx import linear_mx, mx_quantize
from tinytrain_amd.kernels.rms_norm import add_rms_norm, add_rms_norm_mx
from tinytrain_amd.kernels.swiglu import swiglu
from test_block_gpu import BF, U, _rand, _within

pytestmark = pytest.mark.gpu
MOST = 1 << 20


def _signs(*shape, seed=0):
    """-1, 0 and 1."""
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=g, device="cuda").to(BF)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("M, K, N", [(1, MOST, 8), (20, MOST, 72), (70, MOST, 40), (300, MOST - 96, 264), (1, 32, MOST),
                                     (5, 96, MOST), (17, 96, MOST), (300, 32, MOST)])
def test_linear_mx_longest(M, K, N, x8, bits):
    announce(f"linear_mx M={M} K={K} N={N} bits={bits} x8={x8}")
    x, w = _signs(M, K, seed=1), _signs(N, K, seed=2)
    want = (x.float() @ w.float().t()).to(BF)  # whole numbers below 2^24
    codes, scales = mx_quantize(w, bits)
    xs = None
    if x8:
        x, xs = mx_quantize(x, 8)
    assert torch.equal(linear_mx(x, codes, scales, xs), want)


@pytest.mark.parametrize("M, K, N", [(1, MOST, 8), (70, MOST, 8), (1, 8, MOST), (17, 8, MOST), (300, 16, MOST - 8)])
def test_swiglu_longest(M, K, N):
    """The products' sums are exact; 64 columns have a gradient, so that dx's sums have 128 terms that are not zero."""
    announce(f"swiglu M={M} K={K} N={N}")
    x, wg, wu = _signs(M, K, seed=1), _signs(N, K, seed=2), _signs(N, K, seed=3)
    da = torch.zeros(M, N, device="cuda", dtype=BF)
    cols = torch.arange(N - 1, -1, -max(N // 64, 1), device="cuda")[:64]
    da[:, cols] = _rand(M, len(cols), seed=4, dtype=BF)
    t = [v.requires_grad_() for v in (x, wg, wu)]
    a = swiglu(*t)
    xd, gd, ud, d = (v.detach().double() for v in (*t, da))
    g, u = xd @ gd.t(), xd @ ud.t()
    p = torch.sigmoid(g)
    # sig = 1 / (1 + 2^(-g log2 e)): the rounding of the exponent is 2^-23 |g|, and past 130 sig is 0 or 1.  Below
    # 2^-126 fp32 has no normal numbers, and below 2^-128 the denominator is infinite: sig is 0 there, off by < 2^-126.
    sig, least = 2.0**-20 + 2.0**-22 * g.abs().clamp(max=130), 2.0**-126
    _within("a", a.detach(), g * p * u, (g * p * u).abs() * sig + least * (g * u).abs())
    slope = p * (1 + g * (1 - p))     # whole g: not near its zero
    dg, du = d * u * slope, d * g * p
    # one rounding to bf16, and g and u read with 12 bits: |silu'| < 1.1, |silu''| <= 1/2
    eg = dg.abs() * (2.0**-8 + sig) + (d * u).abs() * (2.0**-13 * (slope.abs() + 0.5 * g.abs()) + least * (1 + g.abs()))
    eu = du.abs() * (2.0**-8 + sig) + (d * g).abs() * (2.0**-13 * 1.1 + least)
    dx, dwg, dwu = torch.autograd.grad(a, t, da)
    _within("dx", dx, dg @ gd + du @ ud, (eg + 256 * U * dg.abs()) @ gd.abs() + (eu + 256 * U * du.abs()) @ ud.abs())
    _within("dw_gate", dwg, dg.t() @ xd, (eg + 2 * M * U * dg.abs()).t() @ xd.abs())
    _within("dw_up", dwu, du.t() @ xd, (eu + 2 * M * U * du.abs()).t() @ xd.abs())


def _repeated(run, M):
    return run.repeat(-(-M // run.shape[0]), 1)[:M]


def _repeats(t, run):
    n = run.shape[0]
    whole = t[:t.shape[0] // n * n].view(-1, n, *run.shape[1:])
    return (whole == run).all() and torch.equal(t[len(whole) * n:], run[:t.shape[0] % n])


def test_norms_of_more_rows_than_workgroups():
    M = (1 << 25) + 70  # 32 rows a workgroup, 2^20 workgroups
    announce(f"add_rms_norm {M} x 8, add_rms_norm_mx {M} x 32")
    w = _rand(32, seed=3)
    x, r = _rand(1000, 8, seed=1, dtype=BF), _rand(1000, 8, seed=2)
    for got, want in zip(add_rms_norm(_repeated(x, M), _repeated(r, M), w[:8]), add_rms_norm(x, r, w[:8])):
        assert _repeats(got, want)
    x, r = _rand(1000, 32, seed=1, dtype=BF), _rand(1000, 32, seed=2, dtype=BF)
    for got, want in zip(add_rms_norm_mx(_repeated(x, M), _repeated(r, M), w), add_rms_norm_mx(x, r, w)):
        assert _repeats(got, want)


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_to_quantise_past_2_31(bits):
    M, K = 2**31 // 4096 + 300, 4096
    announce(f"mx_quantize {M} x {K} into {bits} bits")
    x = _rand(1000, K, seed=1, dtype=BF)
    got, want = mx_quantize(_repeated(x, M), bits), mx_quantize(x, bits)
    c, s = mx_cache.quantise(x.cpu(), bits)
    assert torch.equal(want[0].cpu(), c) and torch.equal(want[1].cpu(), s)
    assert all(_repeats(a, b) for a, b in zip(got, want))


def test_scales_laid_out_for_more_rows_than_workgroups():
    """K no multiple of 128 and 2^28 rows and more of scales, a dword each."""
    M, K, N = (1 << 28) + 1000, 32, 8
    announce(f"linear_mx M={M} K={K} N={N}")
    x, xs = mx_quantize(_rand(1000, K, seed=1, dtype=BF), 8)
    w = mx_quantize(_rand(N, K, seed=2), 4)
    want = linear_mx(x, *w, xs)
    assert _repeats(linear_mx(_repeated(x, M), *w, _repeated(xs, M)), want)


@pytest.mark.parametrize("bits", [0x7f81, 0x7fc0, 0x7fff, -0x7f, -0x40, -0x1])  # bf16 NaN of both signs
@pytest.mark.parametrize("M", [3, 200])
def test_swiglu_nan_of_every_kind(M, bits):
    """Through what the forward keeps a NaN stays one."""
    announce(f"swiglu NaN {bits & 0xffff:#x} M={M}")
    x, wg, wu = _rand(M, 104, seed=1, dtype=BF), _rand(136, 104, seed=2, dtype=BF), _rand(136, 104, seed=3, dtype=BF)
    nan = torch.tensor(bits, dtype=torch.int16, device="cuda").view(BF)
    assert torch.isnan(nan)
    x[1, 7] = nan
    t = [v.requires_grad_() for v in (x, wg, wu)]
    a = swiglu(*t)
    dx, dwg, dwu = torch.autograd.grad(a, t, _rand(M, 136, seed=4, dtype=BF))
    assert torch.isnan(a[1]).all() and torch.isnan(dx[1]).all() and torch.isnan(dwg).all() and torch.isnan(dwu).all()
    rest = [m for m in range(M) if m != 1]
    assert torch.isfinite(a[rest]).all() and torch.isfinite(dx[rest]).all()
