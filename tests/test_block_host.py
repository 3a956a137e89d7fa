"""CPU tests of the block's operators (RMSNorm with the residual, gated feed-forward, products with quantised
weights): their oracle against autograd and differences, the C ABI's argument checks (they return before any
HIP call), the refusals of the Python operators, and tracing."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import block
from tinytrain_amd import _lib
from tinytrain_amd.kernels.linear_mx import linear_mx, mx_quantize
from tinytrain_amd.kernels.rms_norm import BlockInputError, add_rms_norm, add_rms_norm_mx, rms_norm, rms_norm_bwd
from tinytrain_amd.kernels.swiglu import swiglu, swiglu_bwd, swiglu_fwd

BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(),
                               reason="libttfa.so not built (python -m tinytrain_amd.build)")


# ---------------------------------------------------------------------------- the oracle

def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def _central(f, x, dout, at, step=1e-6):
    """d <f(x), dout> / dx[at] by central differences."""
    e = torch.zeros_like(x)
    e.view(-1)[at] = step
    return (((f(x + e) - f(x - e)) * dout).sum() / (2 * step)).item()


def test_norm_oracle_gradients():
    x, r, w = _rand(5, 24), _rand(5, 24, seed=1), 1 + 0.2 * _rand(24, seed=2)
    dy, dh, eps = _rand(5, 24, seed=3), _rand(5, 24, seed=4), 1e-3
    h = (x + r).requires_grad_()
    wg = w.clone().requires_grad_()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * wg
    want = torch.autograd.grad((y * dy).sum() + (h * dh).sum(), (h, wg))
    d, size, dw, dw_size = block.add_rms_norm_grads(dy, dh, h.detach(), w, eps)
    assert torch.allclose(d, want[0], rtol=1e-12) and torch.allclose(dw, want[1], rtol=1e-12)
    assert (size >= d.abs()).all() and (dw_size >= dw.abs()).all()
    f = lambda z: z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * w  # noqa: E731
    for at in (0, 50, 119):
        assert _central(f, h.detach(), dy, at) + dh.view(-1)[at].item() == pytest.approx(d.view(-1)[at].item(), rel=1e-6)


def test_swiglu_oracle_gradients():
    x, wg, wu, da = _rand(6, 16), _rand(24, 16, seed=1), _rand(24, 16, seed=2), _rand(6, 24, seed=3)
    t = [v.clone().requires_grad_() for v in (x, wg, wu)]
    a = torch.nn.functional.silu(t[0] @ t[1].t()) * (t[0] @ t[2].t())
    assert torch.allclose(block.swiglu(x, wg, wu)[0], a.detach(), rtol=1e-12)
    got = block.swiglu_grads(da, x, wg, wu)
    for (g, size, _), want in zip(got.values(), torch.autograd.grad(a, t, da)):
        assert torch.allclose(g, want, rtol=1e-10) and (size >= g.abs() * (1 - 1e-12)).all()
    for at in (0, 40, 95):
        assert _central(lambda v: block.swiglu(v, wg, wu)[0], x, da, at) == pytest.approx(
            got["dx"][0].view(-1)[at].item(), rel=1e-5, abs=1e-6)


# ----------------------------------------------------------------------------- the C ABI

P = [0x100000 + 0x1000 * i for i in range(9)]  # aligned stand-ins: validation returns before use
BIG = 1 << 30


def _norm(p=P, M=4, C=64, xt=0, rt=0, yt=0, eps=1e-6):
    return _lib.load().ttfa_rms_norm_fwd(*p[:5], M, C, xt, rt, yt, eps, None)


def _norm_mx(p=P, M=4, C=64, xt=0, rt=0, eps=1e-6):
    return _lib.load().ttfa_rms_norm_mx(*p[:6], M, C, xt, rt, eps, None)


def _norm_bwd(p=P, M=4000, C=64, rt=0, yt=0, eps=1e-6):
    return _lib.load().ttfa_rms_norm_bwd(*p[:8], M, C, rt, yt, eps, None)


def _swiglu_fwd(p=P, M=64, K=64, N=64):
    return _lib.load().ttfa_swiglu_fwd(*p[:5], M, K, N, None)


def _swiglu_bwd(p=P, M=64, K=64, N=64):
    return _lib.load().ttfa_swiglu_bwd(*p[:9], M, K, N, None)


def _quantize(p=P, M=4, K=64, bits=4, dt=0):
    return _lib.load().ttfa_mx_quantize(*p[:3], M, K, bits, dt, None)


def _linear(p=P, M=4, K=64, N=64, bits=4):
    return _lib.load().ttfa_linear_mx(*p[:6], M, K, N, bits, None)


@needs_lib
@pytest.mark.parametrize("entry, kw, code", [
    (_norm, dict(C=60), _lib.E_COLS), (_norm, dict(C=0), _lib.E_COLS), (_norm, dict(C=16392), _lib.E_COLS),
    (_norm, dict(M=0), _lib.E_SEQ), (_norm, dict(M=1 << 40), _lib.E_SEQ), (_norm, dict(xt=2), _lib.E_DTYPE),
    (_norm, dict(rt=-1), _lib.E_DTYPE), (_norm, dict(yt=7), _lib.E_DTYPE), (_norm, dict(eps=1.0), _lib.E_EPS),
    (_norm, dict(eps=-1e-9), _lib.E_EPS), (_norm, dict(eps=math.nan), _lib.E_EPS),
    (_norm_mx, dict(C=40), _lib.E_COLS), (_norm_mx, dict(M=-1), _lib.E_SEQ), (_norm_mx, dict(xt=2), _lib.E_DTYPE),
    (_norm_bwd, dict(C=4), _lib.E_COLS), (_norm_bwd, dict(M=0), _lib.E_SEQ), (_norm_bwd, dict(yt=2), _lib.E_DTYPE),
    (_swiglu_fwd, dict(M=0), _lib.E_SEQ), (_swiglu_fwd, dict(K=4), _lib.E_COLS), (_swiglu_fwd, dict(N=12), _lib.E_COLS),
    (_swiglu_fwd, dict(K=(1 << 20) + 8), _lib.E_COLS), (_swiglu_fwd, dict(M=BIG, N=1 << 20), _lib.E_SEQ),
    (_swiglu_bwd, dict(M=-3), _lib.E_SEQ), (_swiglu_bwd, dict(N=0), _lib.E_COLS),
    (_quantize, dict(bits=6), _lib.E_BITS), (_quantize, dict(K=48), _lib.E_COLS), (_quantize, dict(dt=3), _lib.E_DTYPE),
    (_quantize, dict(M=1 << 29), _lib.E_SEQ), (_linear, dict(bits=16), _lib.E_BITS), (_linear, dict(K=40), _lib.E_COLS),
    (_linear, dict(N=4), _lib.E_COLS), (_linear, dict(M=0), _lib.E_SEQ), (_linear, dict(M=BIG, N=1 << 20), _lib.E_SEQ)])
def test_argument_errors_return_codes(entry, kw, code):
    assert entry(**kw) == code
    assert _lib.strerror(code).startswith("ttfa:") and "unknown" not in _lib.strerror(code)


@needs_lib
@pytest.mark.parametrize("entry, required, n", [
    (_norm, (0, 2, 3), 5), (_norm_mx, (0, 2, 3, 4), 6), (_norm_bwd, (0, 2, 3, 5, 6, 7), 8),
    (_swiglu_fwd, (0, 1, 2, 3), 5), (_swiglu_bwd, (0, 1, 2, 3, 4, 8), 9), (_quantize, (0, 1, 2), 3),
    (_linear, (0, 2, 3, 4), 5)])
def test_null_and_misaligned_pointers(entry, required, n):
    for i in range(n):
        bad = list(P)
        bad[i] += 8
        assert entry(bad) == _lib.E_ALIGN, i
        bad[i] = None
        if i in required:
            assert entry(bad) == _lib.E_NULL, i


@needs_lib
def test_pointers_that_come_together():
    """A residual and its sum; the two weight gradients; at least one gradient."""
    for entry, pair in ((_norm, (1, 4)), (_norm_mx, (1, 5)), (_swiglu_bwd, (6, 7))):
        for i in pair:
            bad = list(P)
            bad[i] = None
            assert entry(bad) == _lib.E_NULL
    bad = list(P)
    bad[5] = bad[6] = bad[7] = None
    assert _swiglu_bwd(bad) == _lib.E_NULL


@needs_lib
def test_workspace_sizes():
    lib = _lib.load()
    assert lib.ttfa_rms_norm_workspace_bytes(0, 64) == lib.ttfa_rms_norm_workspace_bytes(4, 60) == -1
    assert lib.ttfa_rms_norm_workspace_bytes(1, 64) == 0
    assert lib.ttfa_rms_norm_workspace_bytes(1 << 20, 64) % (64 * 4) == 0
    assert lib.ttfa_swiglu_workspace_bytes(4, 64, 60) == lib.ttfa_swiglu_saved_bytes(4, 60) == -1
    assert lib.ttfa_swiglu_workspace_bytes(1 << 20, 64, 1 << 14) >= 4 << 34   # past 32 bits
    assert lib.ttfa_swiglu_saved_bytes(1 << 20, 1 << 14) == 5 << 34
    assert lib.ttfa_linear_mx_workspace_bytes(4, 64, 64, 5, 0) == -1
    assert lib.ttfa_linear_mx_workspace_bytes(1, 64, 64, 4, 0) >= 0


# ---------------------------------------------------------------------- Python refusals

def _e(*shape, dtype=BF, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


W = dict(dtype=F32)
REFUSED = [
    lambda: add_rms_norm(_e(4, 64, device="cpu"), _e(4, 64, device="cpu"), _e(64, device="cpu")),
    lambda: add_rms_norm(_e(4, 60), _e(4, 60), _e(60, **W)),
    lambda: add_rms_norm(_e(4, 64), _e(4, 56), _e(64, **W)),
    lambda: add_rms_norm(_e(4, 64), _e(4, 64, dtype=torch.float16), _e(64, **W)),
    lambda: add_rms_norm(_e(4, 64, dtype=torch.float16), _e(4, 64), _e(64, **W)),
    lambda: add_rms_norm(_e(4, 64), _e(4, 64), _e(32, **W)),
    lambda: add_rms_norm(_e(4, 64), _e(4, 64), _e(64, dtype=torch.int32)),
    lambda: add_rms_norm(_e(64, 64).t(), _e(64, 64), _e(64, **W)),
    lambda: add_rms_norm(_e(64, 64), _e(64, 64).t(), _e(64, **W)),
    lambda: add_rms_norm(_e(4, 64), _e(4, 64), _e(64, **W), dtype=torch.float16),
    lambda: add_rms_norm(_e(4, 64), None, _e(64, **W)),
    lambda: add_rms_norm(_e(4, 16392), _e(4, 16392), _e(16392, **W)),
    lambda: rms_norm(_e(()), _e(1, **W)),
    lambda: add_rms_norm_mx(_e(4, 40), _e(4, 40), _e(40, **W)),
    lambda: swiglu(_e(4, 64), _e(32, 64), _e(40, 64)),
    lambda: swiglu(_e(4, 64), _e(32, 56), _e(32, 56)),
    lambda: swiglu(_e(4, 64, dtype=F32), _e(32, 64, dtype=F32), _e(32, 64, dtype=F32)),
    lambda: swiglu(_e(4, 60), _e(32, 60), _e(32, 60)),
    lambda: swiglu(_e(4, 64), _e(33, 64), _e(33, 64)),
    lambda: swiglu(_e(4, 64), _e(64, 64).t(), _e(64, 64)),
    lambda: swiglu(_e(4, 64, device="cpu"), _e(32, 64, device="cpu"), _e(32, 64, device="cpu")),
    lambda: mx_quantize(_e(4, 48), 4),
    lambda: mx_quantize(_e(4, 64), 2),
    lambda: mx_quantize(_e(4, 64, dtype=torch.float16), 4),
    lambda: linear_mx(_e(4, 64), _e(32, 32, dtype=U8), _e(32, 3, dtype=U8)),
    lambda: linear_mx(_e(4, 64), _e(32, 40, dtype=U8), _e(32, 2, dtype=U8)),
    lambda: linear_mx(_e(4, 96), _e(32, 32, dtype=U8), _e(32, 2, dtype=U8)),
    lambda: linear_mx(_e(4, 64), _e(30, 32, dtype=U8), _e(30, 2, dtype=U8)),
    lambda: linear_mx(_e(4, 64, dtype=F32), _e(32, 32, dtype=U8), _e(32, 2, dtype=U8)),
    lambda: linear_mx(_e(4, 64, dtype=U8), _e(32, 32, dtype=U8), _e(32, 2, dtype=U8)),
    lambda: linear_mx(_e(4, 64), _e(32, 32, dtype=U8), _e(32, 2, dtype=U8), _e(4, 2, dtype=U8)),
    lambda: linear_mx(_e(4, 64, dtype=U8), _e(32, 32, dtype=U8), _e(32, 2, dtype=U8), _e(4, 1, dtype=U8)),
    lambda: linear_mx(_e(4, 64), _e(32, 32, dtype=U8, device="cpu"), _e(32, 2, dtype=U8)),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refusals(i, monkeypatch):
    """Outside the contract the ops raise; shapes and types are checked before the library is asked.  (Fake
    tensors run no op body, so the bodies are called on them directly.)"""
    from tinytrain_amd.kernels import linear_mx as lm, rms_norm as rn, swiglu as sw

    for mod, names in ((rn, ("rms_norm_fwd", "rms_norm_mx")), (sw, ("swiglu_fwd",)), (lm, ("_linear_mx", "mx_quantize"))):
        for name in names:
            monkeypatch.setattr(mod, name, getattr(mod, name)._init_fn)
    monkeypatch.setitem(globals(), "mx_quantize", lm.mx_quantize)
    with FakeTensorMode(), pytest.raises(BlockInputError):
        REFUSED[i]()


# -------------------------------------------------------------------------------- tracing

CALLS = {
    "rms_norm_fwd": (lambda x, r, w: add_rms_norm(x, r, w, 1e-6), lambda: [_e(3, 5, 64), _e(3, 5, 64, dtype=F32), _e(64, **W)]),
    "rms_norm_mx": (lambda x, r, w: add_rms_norm_mx(x, r, w), lambda: [_e(3, 5, 64), _e(3, 5, 64), _e(64, **W)]),
    "swiglu_fwd": (swiglu, lambda: [_e(3, 5, 64), _e(48, 64), _e(48, 64)]),
    "linear_mx": (linear_mx, lambda: [_e(3, 5, 64), _e(48, 32, dtype=U8), _e(48, 2, dtype=U8)]),
    "mx_quantize": (mx_quantize, lambda: [_e(48, 64)]),
}


@pytest.mark.parametrize("loaded", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_fullgraph_trace_is_one_op(name, loaded, monkeypatch):
    fn, args = CALLS[name]
    if loaded:
        if not (_lib.LIB_PATH.exists() and _lib.NATIVE_PATH.exists()):
            pytest.skip("the libraries are not built")
        _lib.native()
    else:
        monkeypatch.setattr(_lib, "_lib", None)
        monkeypatch.setattr(_lib, "_native", None)
    ops = []

    def backend(gm, _):
        ops.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function")
        return gm.forward

    torch._dynamo.reset()
    with FakeTensorMode():
        torch.compile(lambda *a: fn(*a), backend=backend, fullgraph=True)(*args())
    assert [o for o in ops if "tinytrain" in o] == [f"tinytrain.{name}.default"], ops


def test_fake_shapes():
    """Shapes and types of results and gradients without a GPU."""
    with FakeTensorMode():
        x, r, w = _e(3, 5, 64), _e(3, 5, 64, dtype=F32), _e(64, **W)
        y, h = add_rms_norm(x, r, w)
        assert (y.shape, y.dtype, h.dtype) == (x.shape, BF, F32)
        dr, dx, dw = rms_norm_bwd(y, h, h, w, 1e-6, BF)
        assert (dx.dtype, dr.dtype, dw.shape) == (BF, F32, w.shape) and dx.shape == dr.shape == x.shape
        assert rms_norm_bwd(y, None, x, w, 1e-6, BF)[1].numel() == 0
        assert rms_norm(r, w, dtype=BF).dtype == BF
        wg, wu = _e(48, 64), _e(48, 64)
        a = swiglu(x, wg, wu)
        assert a.shape == (3, 5, 48)
        kept = swiglu_fwd(x, wg, wu, True)[1]
        assert kept.shape == (5 * 15 * 48,) and swiglu_fwd(x, wg, wu, False)[1].numel() == 0
        dx, dg, du = swiglu_bwd(a, kept, x, wg, wu, True, False)
        assert dx.shape == x.shape and dg.numel() == du.numel() == 0
        assert swiglu_bwd(a, kept, x, wg, wu, False, True)[1].shape == wg.shape
        codes, scales, h = add_rms_norm_mx(x, None, w)
        assert codes.shape == (3, 5, 64) and scales.shape == (3, 5, 2) and h.shape == x.shape
        wc, ws = mx_quantize(_e(48, 64), 4)
        assert linear_mx(codes, wc, ws, scales).shape == (3, 5, 48)
