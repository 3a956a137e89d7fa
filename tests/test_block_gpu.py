"""GPU tests of the block's operators (RMSNorm with the residual, gated feed-forward, products with quantised
weights) against the 64-bit oracle.

Tolerances count roundings.  u = 2^-24 for fp32, and half a step of the result's type at the end
(bf16 2^-8, fp32 2^-24 of the value).
* Norm: a lane adds at most 64 squares and the rows' lanes are joined in at most 8 steps, so the mean is off
  by at most 72 u, its root by half of that, and five more roundings follow: 48 u with room.  Gradients:
  two such sums and ten roundings on the terms: 160 u of the terms' sizes.  dw adds at most 5 rows a lane
  (512 workgroups), 32 lane groups and 8 + 16 partials, each term off by 48 u: 170 u with the sizes of
  these tests.
* Products: n terms in fp32, each addition off by at most 2 u (the matrix unit may cut instead of round):
  2 n u of the sum of magnitudes.  The activation (an exponential and a reciprocal of one step each, the
  argument of the exponential rounded) adds 2^-20 with |g| < 8.  dg and du are rounded to bf16 before the
  last products: 2^-8 of their magnitudes.  The backward reads the sums rounded to 12 bits: 2^-13 of them.
* With both operands quantised the matrix unit drops, within every eight consecutive products, the bits below
  2^-13 of the largest: less than 8 * 2^-13 = 2^-10 of it.
"""

import math
import random

import pytest
import torch

from helpers import announce
from oracle import block, mx_cache
from tinytrain_amd import _lib
from tinytrain_amd.kernels.linear_mx import linear_mx, mx_quantize
from tinytrain_amd.kernels.rms_norm import add_rms_norm, add_rms_norm_mx, rms_norm, rms_norm_bwd, rms_norm_fwd
from tinytrain_amd.kernels.swiglu import swiglu, swiglu_bwd, swiglu_fwd

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0**-24


def _rand(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _within(name, got, want, tol):
    """|got - want| <= tol + half a step of got's type, everywhere; NaN where the oracle has NaN."""
    err = (got.double() - want).abs()
    tol = tol + want.abs() * _half(got.dtype) * (1 + 2.0**-7) + 1e-37
    bad = ~(err <= tol) & ~(torch.isnan(want) & torch.isnan(got.double())) & ~(got.double() == want)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {(err / tol).nan_to_num(0).max():.3g} of the tolerance"


# ----------------------------------------------------------------------------------- norm

NORM_SHAPES = [(1, 8), (3, 64), (37, 72), (5, 256), (130, 768), (33, 1000), (9, 2048), (7, 2056), (6, 4096), (5, 8200),
               (3, 16384), (5000, 96), (4100, 768)]


@pytest.mark.parametrize("M, C", NORM_SHAPES)
@pytest.mark.parametrize("xt, rt", [(BF, BF), (BF, F32), (F32, BF), (F32, F32)])
def test_add_rms_norm(M, C, xt, rt):
    announce(f"add_rms_norm M={M} C={C} {xt} {rt}")
    x, r = _rand(M, C, seed=1, dtype=xt), _rand(M, C, seed=2, dtype=rt, scale=3.0)
    w = 1 + 0.3 * _rand(C, seed=3)
    t = [v.requires_grad_() for v in (x, r, w)]
    yt = F32 if (M + C) % 3 == 0 else BF
    y, h = add_rms_norm(*t, 1e-6, yt)
    assert y.dtype == yt and h.dtype == rt
    want, stored = block.add_rms_norm(x.detach(), r.detach(), w.detach(), 1e-6)
    assert torch.equal(h, stored)
    _within("y", y.detach(), want, 48 * U * want.abs())
    dy, dh = _rand(M, C, seed=4, dtype=yt), _rand(M, C, seed=5, dtype=rt)
    dx, dr, dw = torch.autograd.grad((y, h), t, (dy, dh))
    assert (dx.dtype, dr.dtype, dw.dtype) == (xt, rt, F32)
    d, size, wantw, sizew = block.add_rms_norm_grads(dy, dh, stored, w.detach(), 1e-6)
    _within("dx", dx, d, 160 * U * size)
    _within("dr", dr, d, 160 * U * size)
    _within("dw", dw, wantw, 170 * U * sizew)


@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("shape", [(7, 64), (2, 3, 1000), (4096,)])
def test_rms_norm_alone(shape, xt):
    announce(f"rms_norm {shape} {xt}")
    x, w = _rand(*shape, seed=1, dtype=xt).requires_grad_(), (1 + 0.3 * _rand(shape[-1], seed=2)).to(BF).requires_grad_()
    y = rms_norm(x, w, 1e-5, BF)
    want, _ = block.add_rms_norm(x.detach(), None, w.detach(), 1e-5)
    _within("y", y.detach(), want, 48 * U * want.abs())
    dy = _rand(*shape, seed=3, dtype=BF)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    d, size, wantw, sizew = block.add_rms_norm_grads(dy, None, x.detach(), w.detach(), 1e-5)
    _within("dx", dx, d, 160 * U * size)
    assert dw.dtype == BF
    _within("dw", dw, wantw, 170 * U * sizew)


def test_norm_unused_outputs_and_strided_gradients():
    """A gradient through h alone or y alone, expanded and transposed gradients."""
    x, r, w = _rand(40, 72, seed=1, dtype=BF), _rand(40, 72, seed=2), _rand(72, seed=3)
    t = [v.requires_grad_() for v in (x, r, w)]
    g = _rand(72, 40, seed=4).t()
    y, h = add_rms_norm(*t)
    dx, dr, dw = torch.autograd.grad(h, t, g, allow_unused=True, retain_graph=True)
    assert torch.equal(dr, g) and torch.equal(dx, g.to(BF)) and (dw is None or not dw.any())
    gy = torch.ones(1, 1, device="cuda", dtype=BF).expand(40, 72)
    dx, dr, dw = torch.autograd.grad(y, t, gy)
    d, size, wantw, sizew = block.add_rms_norm_grads(gy, None, h.detach(), w.detach(), 1e-6)
    _within("dr", dr, d, 160 * U * size)
    _within("dx", dx, d, 160 * U * size)
    _within("dw", dw, wantw, 170 * U * sizew)


def test_norm_special_rows():
    """A row of zeros, rows with NaN and infinity, and their neighbours."""
    x, r, w = _rand(6, 96, seed=1, dtype=BF), _rand(6, 96, seed=2, dtype=BF), _rand(96, seed=3)
    x[1] = 0
    r[1] = 0
    x[2, 5] = math.nan
    r[4, 7] = math.inf
    want, stored = block.add_rms_norm(x, r, w, 1e-6)
    y, h = add_rms_norm(x, r, w)
    assert torch.equal(h.nan_to_num(-1), stored.nan_to_num(-1)) and not y[1].any()
    for row in (0, 1, 3, 5):
        _within("y", y[row], want[row], 48 * U * want[row].abs())
    assert torch.isnan(y[2]).all() and torch.isnan(y[4, 7])
    codes, scales, _ = add_rms_norm_mx(x, r, w)
    assert (scales[2] == 255).all() and not codes[2].any()
    assert not (codes[1] & 127).any()  # zeros, of the weights' signs
    assert (scales[[0, 1, 3, 5]] != 255).all()
    y0, _ = add_rms_norm(x * 0, r * 0, w, 0.0)   # 0 / 0, as the formula has it
    assert torch.isnan(y0).all()


@pytest.mark.parametrize("M, C", [(1, 32), (33, 96), (130, 768), (9, 2048), (7, 2080), (6, 4096), (3, 16384)])
@pytest.mark.parametrize("xt, rt", [(BF, BF), (F32, F32), (BF, F32), (F32, None)])
def test_add_rms_norm_mx(M, C, xt, rt):
    """Bytes equal to the definition's: y in 64 bits, rounded once."""
    announce(f"add_rms_norm_mx M={M} C={C} {xt} {rt}")
    x = _rand(M, C, seed=1, dtype=xt)
    r = None if rt is None else _rand(M, C, seed=2, dtype=rt, scale=3.0)
    w = 1 + 0.3 * _rand(C, seed=3)
    codes, scales, h = add_rms_norm_mx(x, r, w, 1e-6)
    want, stored = block.add_rms_norm(x, r, w, 1e-6)
    assert torch.equal(h, stored)
    c, s = mx_cache.quantise(want.cpu(), 8)
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu(), c)


def test_norm_empty_and_other_ranks():
    w = torch.ones(64, device="cuda", requires_grad=True)
    for shape in ((0, 64), (2, 0, 64)):
        x, r = torch.empty(shape, device="cuda", dtype=BF, requires_grad=True), torch.empty(shape, device="cuda")
        y, h = add_rms_norm(x, r, w)
        assert y.shape == h.shape == shape
        dx, dw = torch.autograd.grad((y.float() + h).sum(), (x, w))
        assert dx.shape == shape and not dw.any()
        codes, scales, _ = add_rms_norm_mx(x.detach(), r, w.detach())
        assert codes.shape == shape and scales.shape == (*shape[:-1], 2)


# --------------------------------------------------------------------------------- swiglu

SWIGLU_SHAPES = [(1, 8, 8), (1, 768, 2304), (5, 64, 72), (16, 104, 200), (33, 768, 328), (100, 40, 136), (128, 32, 128),
                 (129, 200, 264), (300, 1000, 520), (1000, 136, 1032), (2051, 72, 128),
                 (4100, 520, 2056), (8197, 264, 2056), (20000, 136, 264), (5000, 2056, 776),
                 (3, 136, 4104), (31, 72, 4360), (48, 1160, 4104), (64, 40, 8192), (65, 40, 8192), (16, 264, 8200),
                 (17, 264, 8200)]


def _check_swiglu(M, K, N):
    x = _rand(M, K, seed=1, dtype=BF).requires_grad_()
    wg, wu = (_rand(N, K, seed=s, dtype=BF, scale=1 / math.sqrt(K)).requires_grad_() for s in (2, 3))
    a = swiglu(x, wg, wu)
    want, unit = block.swiglu(*(t.detach() for t in (x, wg, wu)))
    _within("a", a.detach(), want, 2 * K * U * unit + 2.0**-20 * want.abs())
    da = _rand(M, N, seed=4, dtype=BF)
    grads = torch.autograd.grad(a, (x, wg, wu), da)
    oracle = block.swiglu_grads(da, *(t.detach() for t in (x, wg, wu)))
    for g, (name, (want, size, unit)) in zip(grads, oracle.items()):
        n = 2 * N if name == "dx" else M
        _within(name, g, want, (2.0**-8 + 2.0**-20 + 2 * n * U) * size + (2 * K * U * 1.01 + 2.0**-13) * unit)
    return a, grads


@pytest.mark.parametrize("M, K, N", SWIGLU_SHAPES)
def test_swiglu(M, K, N):
    announce(f"swiglu M={M} K={K} N={N}")
    a, grads = _check_swiglu(M, K, N)
    again, grads2 = _check_swiglu(M, K, N)
    assert torch.equal(a, again) and all(torch.equal(p, q) for p, q in zip(grads, grads2))


def test_swiglu_random_sizes():
    rng = random.Random(7)
    for _ in range(12):
        M, K, N = rng.randint(1, 700), 8 * rng.randint(1, 90), 8 * rng.randint(1, 120)
        announce(f"swiglu M={M} K={K} N={N}")
        _check_swiglu(M, K, N)


def test_swiglu_needs_and_strides():
    """Frozen inputs get no gradient, the others the same bits; gradients with other strides; 3-D rows."""
    x, wg, wu = _rand(6, 7, 64, seed=1, dtype=BF), _rand(48, 64, seed=2, dtype=BF), _rand(48, 64, seed=3, dtype=BF)
    da = _rand(6, 48, 7, seed=4, dtype=BF).transpose(1, 2)
    full = torch.autograd.grad(swiglu(*(t.requires_grad_() for t in (x, wg, wu))), (x, wg, wu), da)
    for need in ((1, 0, 0), (0, 1, 1), (0, 0, 1)):
        t = [v.detach().clone().requires_grad_(bool(n)) for v, n in zip((x, wg, wu), need)]
        got = torch.autograd.grad(swiglu(*t), [v for v, n in zip(t, need) if n], da)
        for g, w in zip(got, [f for f, n in zip(full, need) if n]):
            assert torch.equal(g, w)
    flat = torch.autograd.grad(swiglu(x.view(42, 64), wg, wu), x, da.contiguous().view(42, 48))
    assert torch.equal(flat[0], full[0])
    e = torch.empty(0, 64, device="cuda", dtype=BF, requires_grad=True)
    a = swiglu(e, wg, wu)
    ge, gg = torch.autograd.grad(a.sum(), (e, wg))
    assert a.shape == (0, 48) and ge.shape == e.shape and not gg.any()


@pytest.mark.parametrize("M", [3, 200])
def test_swiglu_keeps_nan_and_infinity_in_place(M):
    """A NaN in a row of x reaches that row of a and of dx and its columns of the weights' gradients; one in a
    row of a weight reaches that column of a."""
    K, N = 104, 136
    x, wg, wu = _rand(M, K, seed=1, dtype=BF), _rand(N, K, seed=2, dtype=BF), _rand(N, K, seed=3, dtype=BF)
    da = _rand(M, N, seed=4, dtype=BF)
    clean = swiglu(x, wg, wu)
    t = [v.clone().requires_grad_() for v in (x, wg, wu)]
    cgrads = torch.autograd.grad(swiglu(*t), t, da)
    bad = x.clone()
    bad[1, K - 1] = math.nan
    t = [bad.requires_grad_(), wg.clone().requires_grad_(), wu.clone().requires_grad_()]
    a = swiglu(*t)
    dx, dwg, _ = torch.autograd.grad(a, t, da)
    rows = [m for m in range(M) if m != 1]
    assert torch.isnan(a[1]).all() and torch.equal(a[rows], clean[rows])
    assert torch.isnan(dx[1]).all() and torch.equal(dx[rows], cgrads[0][rows]) and torch.isnan(dwg).all()
    bad = wu.clone()
    bad[N - 1, 0] = math.inf
    a = swiglu(x, wg, bad)
    assert torch.equal(a[:, :N - 1], clean[:, :N - 1]) and not torch.isfinite(a[:, N - 1]).any()


def test_swiglu_activation_at_its_ends():
    """Large gates of either sign: silu is g, or 0."""
    g = torch.tensor([0.0, 1.0, -1.0, 20.0, -20.0, 80.0, -80.0, 200.0, -200.0, 3e4, -3e4], device="cuda")
    x = torch.zeros(len(g), 8, device="cuda", dtype=BF)
    x[:, 0], x[:, 1] = g, 1.0
    wg, wu = torch.zeros(8, 8, device="cuda", dtype=BF), torch.zeros(8, 8, device="cuda", dtype=BF)
    wg[:, 0], wu[:, 1] = 1.0, 1.0
    x.requires_grad_()
    a = swiglu(x, wg, wu)
    want, _ = block.swiglu(x.detach(), wg, wu)
    # sig = 1 / (1 + 2^(-g log2 e)): the exponent's rounding is 2^-23 |g|
    _within("a", a.detach(), want, want.abs() * (2.0**-20 + 2.0**-22 * g.abs().double().clamp(max=130))[:, None] + 1e-36)
    assert torch.isfinite(torch.autograd.grad(a, x, torch.ones_like(a))[0]).all()


# -------------------------------------------------------------------------- quantised weights

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(8, 32), (3, 5, 96), (40, 4096), (0, 64)])
def test_mx_quantize(shape, dtype, bits):
    announce(f"mx_quantize {shape} {dtype} {bits}")
    x = _rand(*shape, seed=1, dtype=dtype) * torch.exp2(torch.arange(shape[-1], device="cuda") % 40 - 20).to(dtype)
    codes, scales = mx_quantize(x, bits)
    c, s = mx_cache.quantise(x.cpu(), bits) if x.numel() else (codes.cpu(), scales.cpu())
    assert torch.equal(codes.cpu(), c) and torch.equal(scales.cpu(), s)


LINEAR_SHAPES = [(1, 32, 8), (1, 4096, 520), (2, 96, 40), (7, 736, 104), (16, 128, 64), (17, 1024, 72), (32, 160, 136),
                 (33, 512, 264), (64, 2048, 48), (65, 288, 128), (150, 640, 328), (520, 256, 392), (1027, 96, 136),
                 (66, 1152, 72), (300, 128, 1032), (900, 384, 264),
                 (3, 128, 4104), (30, 288, 4360), (48, 96, 8192), (64, 1152, 8192), (1, 256, 8200), (32, 128, 8200),
                 (33, 128, 8200), (15, 2080, 12296), (18, 288, 12296), (16, 160, 16392), (17, 256, 16392),
                 (300, 416, 264), (700, 32, 520), (129, 4128, 136), (1100, 1056, 776), (513, 2080, 264)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("M, K, N", LINEAR_SHAPES)
def test_linear_mx(M, K, N, x8, bits):
    announce(f"linear_mx M={M} K={K} N={N} bits={bits} x8={x8}")
    x = _rand(M, K, seed=1, dtype=BF)
    codes, scales = mx_quantize(_rand(N, K, seed=2, scale=1 / math.sqrt(K)), bits)
    xs = None
    if x8:
        x, xs = mx_quantize(x, 8)
    y = linear_mx(x, codes, scales, xs)
    want, size, top = block.linear_mx(x, xs, codes, scales)
    _within("y", y.cpu(), want, 2 * K * U * size + (2.0**-10 * top if x8 else 0))
    assert torch.equal(y, linear_mx(x, codes, scales, xs))


@pytest.mark.parametrize("M", [2, 300])
def test_linear_mx_keeps_nan_in_place_and_takes_odd_scales(M):
    """A group of NaN in x reaches its row, one in W its column; groups of very different powers of two."""
    K, N = 192, 72
    x = _rand(M, K, seed=1, dtype=BF)
    x[:, 32:64] *= 2.0**40
    w = _rand(N, K, seed=2)
    w[:, 32:64] *= 2.0**-40
    w[5, 64:96] *= 2.0**60
    for bits in (4, 8):
        codes, scales = mx_quantize(w, bits)
        for xs in (None, True):
            xx, xx_s = (x, None) if xs is None else mx_quantize(x, 8)
            want, size, top = block.linear_mx(xx, xx_s, codes, scales)
            y = linear_mx(xx, codes, scales, xx_s)
            _within("y", y.cpu(), want, 2 * K * U * size + (0 if xs is None else 2.0**-10 * top))
            bad = scales.clone()
            bad[3, 5] = 255
            got = linear_mx(xx, codes, bad, xx_s)
            keep = [n for n in range(N) if n != 3]
            assert torch.isnan(got[:, 3]).all() and torch.equal(got[:, keep], y[:, keep])
            rows = [m for m in range(M) if m != 1]
            if xs is None:
                xb = xx.clone()
                xb[1, K - 1] = math.nan
                got = linear_mx(xb, codes, scales)
            else:
                sb = xx_s.clone()
                sb[1, 0] = 255
                got = linear_mx(xx, codes, scales, sb)
            assert torch.isnan(got[1]).all() and torch.equal(got[rows], y[rows])


# --------------------------------------------------------------------------- large calls

def test_calls_past_2_31_elements():
    """The last rows of tensors of more than 2^31 elements, against calls on those rows alone."""
    M, C = 2**31 // 4096 + 200, 4096
    announce(f"add_rms_norm {M} x {C}")
    x = torch.zeros(M, C, device="cuda", dtype=BF)
    r = torch.zeros(M, C, device="cuda", dtype=BF)
    x[-200:], r[-200:] = _rand(200, C, seed=1, dtype=BF), _rand(200, C, seed=2, dtype=BF)
    w = _rand(C, seed=3)
    y, h = add_rms_norm(x, r, w)
    want = add_rms_norm(x[-200:].clone(), r[-200:].clone(), w)
    assert torch.equal(y[-200:], want[0]) and torch.equal(h[-200:], want[1]) and not y[:-200].any()
    dr, _, _ = rms_norm_bwd(y, h, h, w, 1e-6, BF)
    assert torch.equal(dr[-200:], rms_norm_bwd(want[0], want[1], want[1], w, 1e-6, BF)[0])
    del y, dr, r
    codes, scales, _ = add_rms_norm_mx(h, None, w)
    wc, ws, _ = add_rms_norm_mx(h[-200:].clone(), None, w)
    assert torch.equal(codes[-200:], wc) and torch.equal(scales[-200:], ws)
    weight = mx_quantize(_rand(72, C, seed=4), 4)
    got = linear_mx(codes, *weight, scales)
    want, size, top = block.linear_mx(wc, ws, *weight)
    _within("y", got[-200:].cpu(), want, 2.0**-10 * top + 2 * C * U * size)
    del x, h, codes, scales, got
    M, K, N = 2**31 // 8192 + 300, 64, 8192
    announce(f"swiglu {M} x {K} x {N}")
    x = torch.zeros(M, K, device="cuda", dtype=BF)
    x[-300:] = _rand(300, K, seed=5, dtype=BF)
    wg, wu = _rand(N, K, seed=6, dtype=BF, scale=1 / 8), _rand(N, K, seed=7, dtype=BF, scale=1 / 8)
    t = [v.requires_grad_() for v in (x, wg, wu)]
    a = swiglu(*t)
    da = torch.zeros(M, N, device="cuda", dtype=BF)
    da[-300:] = _rand(300, N, seed=8, dtype=BF)
    dx, dwg, dwu = torch.autograd.grad(a, t, da)
    tail = x[-300:].detach()
    want, unit = block.swiglu(tail, wg.detach(), wu.detach())
    _within("a", a.detach()[-300:], want, 2 * K * U * unit + 2.0**-20 * want.abs())
    for g, (name, (want, size, unit)) in zip((dx[-300:], dwg, dwu), block.swiglu_grads(da[-300:], tail, wg.detach(), wu.detach()).items()):
        # the rows of zeros add nothing to a sum
        _within(name, g, want, (2.0**-8 + 2.0**-20 + 4 * N * U) * size + (2 * K * U * 1.01 + 2.0**-13) * unit)
    assert not a.detach()[:-300].any() and not dx[:-300].any()


# ------------------------------------------------------------------- paths, streams, graphs

def test_rows_behind_the_last_are_left():
    """Outputs are written up to their last row and no further (C ABI, buffers with rows to spare)."""
    lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
    for M in (1, 5, 37, 130, 513):
        K, N = 96, 136
        x, r = _rand(M, K, seed=1, dtype=BF), _rand(M, K, seed=2, dtype=BF)
        w, wg, wu = _rand(K, seed=3), _rand(N, K, seed=4, dtype=BF), _rand(N, K, seed=5, dtype=BF)
        codes, scales = mx_quantize(wg, 4)
        out = {n: torch.full((M + 2, c), 7.0, device="cuda", dtype=BF)
               for n, c in (("y", K), ("h", K), ("a", N), ("lin", N), ("dx", K), ("dr", K))}
        dw = torch.full((K + 8,), 7.0, device="cuda")
        dwg, dwu = (torch.full((N + 2, K), 7.0, device="cuda", dtype=BF) for _ in range(2))
        p = {n: t.data_ptr() for n, t in out.items()}
        kept = torch.full((5 * M * N + 16,), 7, device="cuda", dtype=torch.uint8)
        ws = torch.empty(max(lib.ttfa_swiglu_workspace_bytes(M, K, N), lib.ttfa_rms_norm_workspace_bytes(M, K),
                             lib.ttfa_linear_mx_workspace_bytes(M, K, N, 4, 0), 16), device="cuda", dtype=torch.uint8)
        da = _rand(M, N, seed=6, dtype=BF)
        assert lib.ttfa_rms_norm_fwd(x.data_ptr(), r.data_ptr(), w.data_ptr(), p["y"], p["h"], M, K, 0, 0, 0, 1e-6, s) == 0
        assert lib.ttfa_rms_norm_bwd(x.data_ptr(), None, r.data_ptr(), w.data_ptr(), None, p["dr"], dw.data_ptr(),
                                     ws.data_ptr(), M, K, 0, 0, 1e-6, s) == 0
        assert lib.ttfa_swiglu_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), p["a"], kept.data_ptr(), M, K, N,
                                   s) == 0
        assert lib.ttfa_swiglu_bwd(da.data_ptr(), kept.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), p["dx"], dwg.data_ptr(),
                                   dwu.data_ptr(), ws.data_ptr(), M, K, N, s) == 0
        assert lib.ttfa_linear_mx(x.data_ptr(), None, codes.data_ptr(), scales.data_ptr(), p["lin"], ws.data_ptr(), M, K,
                                  N, 4, s) == 0
        torch.cuda.synchronize()
        for n, t in out.items():
            assert (t[M:] == 7).all() and not (t[:M] == 7).all(), n
        assert (kept[5 * M * N:] == 7).all()
        assert (dw[K:] == 7).all() and (dwg[N:] == 7).all() and (dwu[N:] == 7).all()


def test_native_path_equals_the_ops():
    """The extension's calls and the custom ops: equal bits, forward and backward."""
    x, r, w = _rand(37, 96, seed=1, dtype=BF), _rand(37, 96, seed=2), _rand(96, seed=3)
    wg, wu = _rand(72, 96, seed=4, dtype=BF), _rand(72, 96, seed=5, dtype=BF)
    def grads(y, ts):
        return torch.autograd.grad(y, ts, [torch.ones_like(v) for v in y])
    t = [v.requires_grad_() for v in (x, r, w)]
    a, b = add_rms_norm(*t, 1e-6, BF), rms_norm_fwd(*t, 1e-6, BF)
    assert type(a[0].grad_fn).__name__ != type(b[0].grad_fn).__name__  # two paths
    for p, q in zip((*a, *grads(a, t)), (*b, *grads(b, t))):
        assert torch.equal(p, q)
    t = [v.requires_grad_() for v in (x.detach(), wg, wu)]
    a, b = swiglu(*t), swiglu_fwd(*t, True)[0]
    def grads(y, ts):
        return torch.autograd.grad(y, ts, [torch.ones_like(v) for v in y], retain_graph=True)
    for p, q in zip((a, *grads([a], t)), (b, *grads([b], t))):
        assert torch.equal(p, q)
    torch.library.opcheck(rms_norm_fwd, (x.detach(), r.detach(), w.detach(), 1e-6, BF))
    assert torch.equal(swiglu_fwd(*t, False)[0], a)
    for p, q in zip(grads([a], t), grads([swiglu_fwd(*t, False)[0]], t)):  # nothing kept: formed again
        assert torch.equal(p, q)
    torch.library.opcheck(swiglu_fwd, (x.detach(), wg.detach(), wu.detach(), True))


def test_saved_tensor_hooks():
    """A backward whose saved tensors come back elsewhere or in another layout."""
    x, r, w = (_rand(37, 96, seed=1, dtype=BF).requires_grad_(), _rand(37, 96, seed=2).requires_grad_(),
               _rand(96, seed=3).requires_grad_())
    wg, wu = _rand(72, 96, seed=4, dtype=BF).requires_grad_(), _rand(72, 96, seed=5, dtype=BF).requires_grad_()

    def run():
        y, h = add_rms_norm(x, r, w)
        return torch.autograd.grad(swiglu(y, wg, wu).float().sum() + h.sum(), (x, r, w, wg, wu))
    plain = run()
    with torch.autograd.graph.save_on_cpu():
        for p, q in zip(plain, run()):
            assert torch.equal(p, q)


def test_other_stream():
    s = torch.cuda.Stream()
    x, r, w = _rand(500, 768, seed=1, dtype=BF), _rand(500, 768, seed=2, dtype=BF), _rand(768, seed=3)
    wg, wu = _rand(520, 768, seed=4, dtype=BF), _rand(520, 768, seed=5, dtype=BF)
    codes, scales = mx_quantize(wg, 4)
    want = (*add_rms_norm(x, r, w), swiglu(x, wg, wu), linear_mx(x, codes, scales), *add_rms_norm_mx(x, r, w))
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = (*add_rms_norm(x, r, w), swiglu(x, wg, wu), linear_mx(x, codes, scales), *add_rms_norm_mx(x, r, w))
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_captured_step_replays():
    """A training step of norm and feed-forward and a serving step over quantised rows in one graph, replayed with
    new inputs and eager work between, bitwise the eager results."""
    M, C, N = 130, 96, 136
    x, r, w = _rand(M, C, seed=1, dtype=BF), _rand(M, C, seed=2), _rand(C, seed=3)
    wg, wu = _rand(N, C, seed=4, dtype=BF), _rand(N, C, seed=5, dtype=BF)
    da, weight = _rand(M, N, seed=6, dtype=BF), mx_quantize(wg, 4)
    t = [v.requires_grad_() for v in (x, r, w, wg, wu)]

    def step():
        y, h = add_rms_norm(x, r, w)
        a = swiglu(y, wg, wu)
        out = [a.detach(), h.detach(), *torch.autograd.grad((a, h), t, (da, torch.ones_like(h)))]
        codes, scales, h2 = add_rms_norm_mx(x.detach(), r.detach(), w.detach())
        return out + [codes, scales, h2, linear_mx(codes, *weight, scales), linear_mx(a.detach()[:, :C].contiguous(), *weight)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(_rand(M, C, seed=20 + i, dtype=BF))
            da.copy_(_rand(M, N, seed=30 + i, dtype=BF))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_serving_step_as_used():
    """Norm to 8 bits, gate and up projections in 4 bits, activation, norm again: the run against one in 64 bits
    over the values that the bytes stand for."""
    M, C, N = 5, 256, 512
    x, h0, w = _rand(M, C, seed=1, dtype=BF), _rand(M, C, seed=2, dtype=BF), 1 + 0.2 * _rand(C, seed=3)
    wg, wu, wd = (mx_quantize(_rand(*s, seed=i, scale=1 / 16), 4) for i, s in ((4, (N, C)), (5, (N, C)), (6, (C, N))))
    codes, scales, h = add_rms_norm_mx(x, h0, w)
    g, u = linear_mx(codes, *wg, scales), linear_mx(codes, *wu, scales)
    y = linear_mx((torch.nn.functional.silu(g) * u), *wd)
    out, _ = add_rms_norm(y, h, w)
    v = mx_cache.values(codes.cpu(), scales.cpu(), 8)
    W = [mx_cache.values(c.cpu(), s.cpu(), 4) for c, s in (wg, wu, wd)]
    a = torch.nn.functional.silu(v @ W[0].t()) * (v @ W[1].t())
    want, _ = block.add_rms_norm((a @ W[2].t()).float(), h.cpu().float(), w.cpu(), 1e-6)
    # four roundings to bf16 on the branch and two on the way out, each 2^-8 at most
    assert (out.cpu().double() - want).norm() <= 6 * 2.0**-8 * want.norm()


def test_one_tensor_twice():
    """The same tensor as input and residual, and as both weights: gradients are the sums of both uses'."""
    x, w, wg = (v.requires_grad_() for v in (_rand(37, 96, seed=1, dtype=BF), _rand(96, seed=3),
                                             _rand(72, 96, seed=4, dtype=BF)))
    r, wu = x.detach().clone().requires_grad_(), wg.detach().clone().requires_grad_()
    dy, dh, da = _rand(37, 96, seed=5, dtype=BF), _rand(37, 96, seed=6, dtype=BF), _rand(37, 72, seed=7, dtype=BF)
    one = torch.autograd.grad(add_rms_norm(x, x, w), (x, w), (dy, dh))
    two = torch.autograd.grad(add_rms_norm(x, r, w), (x, r, w), (dy, dh))
    assert torch.equal(one[0], two[0] + two[1]) and torch.equal(one[1], two[2])
    one = torch.autograd.grad(swiglu(x, wg, wg), (x, wg), da)
    two = torch.autograd.grad(swiglu(x, wg, wu), (x, wg, wu), da)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1] + two[2])


@pytest.mark.parametrize("leaf", range(3))
def test_norm_with_one_leaf(leaf):
    """Only one of x, residual and weight takes part in autograd: its gradient is the same."""
    ts = [_rand(37, 96, seed=1, dtype=BF), _rand(37, 96, seed=2), _rand(96, seed=3)]
    grads = (_rand(37, 96, seed=4, dtype=BF), _rand(37, 96, seed=5))
    every = [t.clone().requires_grad_() for t in ts]
    want = torch.autograd.grad(add_rms_norm(*every), every, grads)[leaf]
    ts[leaf].requires_grad_()
    y, h = add_rms_norm(*ts)
    assert torch.equal(torch.autograd.grad((y, h), ts[leaf], grads)[0], want)


def test_two_streams_at_once():
    """Training steps on two streams at the same time, with the same weights and rows of other numbers: bitwise
    what each gives alone.  2600 rows split the contraction of both backward products."""
    w, wg, wu = (_rand(768, seed=3).requires_grad_(), _rand(1040, 768, seed=4, dtype=BF).requires_grad_(),
                 _rand(1040, 768, seed=5, dtype=BF).requires_grad_())
    q = mx_quantize(wg.detach(), 4)

    def step(M):
        x, r = _rand(M, 768, seed=1, dtype=BF).requires_grad_(), _rand(M, 768, seed=2).requires_grad_()
        torch.cuda.current_stream().synchronize()
        for _ in range(5):
            y, h = add_rms_norm(x, r, w)
            a = swiglu(y, wg, wu)
            out = (a.detach(), h.detach(), *torch.autograd.grad((a, h), (x, r, w, wg, wu),
                                                                (torch.ones_like(a), torch.ones_like(h))),
                   linear_mx(y.detach(), *q))
        return out
    want = [step(M) for M in (2600, 300)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s, M in zip(streams, (2600, 300)):
        with torch.cuda.stream(s):
            got.append(step(M))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_two_graphs_in_turn():
    """Two graphs whose calls need workspaces, captured one after the other and replayed in turn."""
    wg, wu = _rand(1040, 768, seed=4, dtype=BF), _rand(1040, 768, seed=5, dtype=BF)
    weight = mx_quantize(wg, 8)
    xs = [_rand(M, 768, seed=M, dtype=BF) for M in (200, 520)]

    def step(x):
        a, saved = swiglu_fwd(x, wg, wu, True)
        return (a, *swiglu_bwd(torch.ones_like(a), saved, x, wg, wu, True, True), linear_mx(x, *weight))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x in xs:
            step(x)
    torch.cuda.current_stream().wait_stream(s)
    graphs, held = [torch.cuda.CUDAGraph() for _ in xs], []
    for g, x in zip(graphs, xs):
        with torch.cuda.graph(g):
            held.append(step(x))
    for i in range(3):
        for k, x in enumerate(xs):
            x.copy_(_rand(*x.shape, seed=100 * i + k, dtype=BF))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for k, x in enumerate(xs):
            assert all(torch.equal(a, b) for a, b in zip(held[k], step(x)))


def test_ops_hold_to_their_schemas():
    x, r, w = _rand(37, 96, seed=1, dtype=BF), _rand(37, 96, seed=2), _rand(96, seed=3)
    wg, wu, da = _rand(72, 96, seed=4, dtype=BF), _rand(72, 96, seed=5, dtype=BF), _rand(37, 72, seed=6, dtype=BF)
    saved, (codes, scales) = swiglu_fwd(x, wg, wu, True)[1], mx_quantize(wg, 4)
    ops = torch.ops.tinytrain
    for op, args in ((ops.rms_norm_bwd, (x, r, r, w, 1e-6, BF)), (ops.rms_norm_bwd, (x, None, x, w, 1e-6, BF)),
                     (ops.swiglu_bwd, (da, saved, x, wg, wu, True, False)), (ops.rms_norm_mx, (x, r, w, 1e-6)),
                     (ops.rms_norm_mx, (x, None, w, 1e-6)), (ops.mx_quantize, (r, 4)),
                     (ops.linear_mx, (x, codes, scales, None))):
        torch.library.opcheck(op, args)


def test_function_transforms():
    """Under vmap the operators are loops of their calls; tangents of recorded inputs and second derivatives,
    which have no formula, raise."""
    import torch.autograd.forward_ad as fw

    xs, r, w = _rand(3, 9, 96, seed=1, dtype=BF), _rand(9, 96, seed=2), _rand(96, seed=3)
    wg, wu = _rand(72, 96, seed=4, dtype=BF), _rand(72, 96, seed=5, dtype=BF)
    q = mx_quantize(wg, 4)
    for f in (lambda x: add_rms_norm(x, r, w), lambda x: (swiglu(x, wg, wu),), lambda x: add_rms_norm_mx(x, r, w),
              lambda x: (linear_mx(x, *q),), lambda x: mx_quantize(x, 8)):
        got = torch.vmap(f)(xs)
        for i, x in enumerate(xs):
            assert all(torch.equal(a[i], b) for a, b in zip(got, f(x)))
    for f in (lambda x: add_rms_norm(x, r, w)[0], lambda x: swiglu(x, wg, wu)):
        with fw.dual_level(), pytest.raises(NotImplementedError, match="forward mode AD"):
            f(fw.make_dual(xs[0].clone().requires_grad_(), torch.ones_like(xs[0])))
        x = xs[0].clone().requires_grad_()
        y = f(x)
        with pytest.raises(RuntimeError):
            g, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
            torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M, K, N", [(70, 160, 264), (300, 1152, 520), (129, 4128, 136), (65, 2080, 776)])
def test_linear_mx_workspace_ends_where_it_says(M, K, N, bits, x8):
    """Through the C ABI with exactly the workspace that is asked for: nothing behind it, nor behind y, is written."""
    lib = _lib.load()
    x, xs = _rand(M, K, seed=1, dtype=BF), None
    codes, scales = mx_quantize(_rand(N, K, seed=2, scale=1 / math.sqrt(K)), bits)
    if x8:
        x, xs = mx_quantize(x, 8)
    n = lib.ttfa_linear_mx_workspace_bytes(M, K, N, bits, int(x8))
    ws = torch.full((n + 4096,), 7, dtype=torch.uint8, device="cuda")
    y = torch.full((M + 3, N), 7.0, dtype=BF, device="cuda")
    _lib.check(lib.ttfa_linear_mx(x.data_ptr(), None if xs is None else xs.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                                  y.data_ptr(), ws.data_ptr(), M, K, N, bits, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (ws[n:] == 7).all() and (y[M:] == 7).all()
    assert torch.equal(y[:M], linear_mx(x, codes, scales, xs))


@pytest.mark.parametrize("M, K, N", [(70, 160, 264), (2600, 768, 1040), (999, 1000, 2600), (100, 2056, 72)])
def test_swiglu_workspace_ends_where_it_says(M, K, N):
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    x, wg, wu = _rand(M, K, seed=1, dtype=BF), _rand(N, K, seed=2, dtype=BF), _rand(N, K, seed=3, dtype=BF)
    da = _rand(M, N, seed=4, dtype=BF)
    a, saved = swiglu_fwd(x, wg, wu, True)
    n = lib.ttfa_swiglu_workspace_bytes(M, K, N)
    ws = torch.full((n + 4096,), 7, dtype=torch.uint8, device="cuda")
    dx, dg, du = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
    _lib.check(lib.ttfa_swiglu_bwd(da.data_ptr(), saved.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), dx.data_ptr(),
                                   dg.data_ptr(), du.data_ptr(), ws.data_ptr(), M, K, N, stream))
    torch.cuda.synchronize()
    assert (ws[n:] == 7).all()
    for p, q in zip((dx, dg, du), swiglu_bwd(da, saved, x, wg, wu, True, True)):
        assert torch.equal(p, q)
