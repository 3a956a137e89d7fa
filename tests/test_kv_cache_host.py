"""CPU tests of the quantised KV cache: its oracle against the types' definitions, the C ABI's argument
checks (they return before any HIP call), the refusals of the Python operators, and tracing."""

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import mx_cache as mx
from tinytrain_amd import _lib
from tinytrain_amd.kernels import kv_cache as kv
from tinytrain_amd.kernels.flash_attn import FlashAttnInputError

needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(),
                               reason="libttfa.so not built (python -m tinytrain_amd.build)")


# ---------------------------------------------------------------------------- the oracle

def test_magnitudes_are_the_types():
    c = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(mx.magnitudes(8), c.view(torch.float8_e4m3fn).double())
    assert mx.magnitudes(4).tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantise_rounds_to_the_nearest_value(bits, dtype):
    """The error of an element is at most half the step above it, 2^e times half a step at the top;
    values that the format holds come back as they are."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(300, 64, generator=g) * torch.exp2(torch.randint(-100, 100, (300, 1), generator=g).float())
    x = x.to(dtype)
    c, s = mx.quantise(x, bits)
    y = mx.values(c, s, bits)
    e = torch.exp2(s.double() - 127).repeat_interleave(32, -1)
    half_top = {4: 1.0, 8: 16.0}[bits]
    assert ((y - x.double()).abs() <= half_top * e).all()
    if bits == 8:  # relative: 2^-4 of a normal element, 2^-10 units below
        assert ((y - x.double()).abs() <= torch.maximum(x.double().abs() / 16, e * 2.0**-10)).all()
    c2, s2 = mx.quantise(y.to(dtype), bits)
    assert torch.equal(mx.values(c2, s2, bits), y)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantise_borders(bits):
    """Ties go to the even code, the shared exponent changes right above `top`, clamps at the ends, and
    groups with NaN or infinity are NaN."""
    v = mx.magnitudes(bits)
    x = torch.zeros(len(v), 32, dtype=torch.float64)
    x[:, 0] = v[-1]                                          # fixes e = 0
    x[:-1, 1] = (v[1:] + v[:-1]) / 2
    c, s = mx.quantise(x, bits)
    assert (s == 127).all()
    y = mx.values(c, s, bits)[:-1, 1]
    even = torch.where(torch.arange(len(v) - 1) % 2 == 0, v[:-1], v[1:])
    assert torch.equal(y, even)
    top, lo, hi = mx.LIMITS[bits]
    for a, e in ((top, 0), (top * (1 + 2**-20), 1), (top / 2, -1), (0.0, lo), (2.0**-140, lo),
                 (3.0e38, min(hi, math.ceil(math.log2(3.0e38 / top))))):
        assert mx.quantise(torch.full((1, 32), a, dtype=torch.float64), bits)[1].item() == e + 127
    assert mx.values(*mx.quantise(torch.full((1, 32), 3.3e38), bits), bits).max() <= torch.finfo(torch.bfloat16).max
    for bad in (math.nan, math.inf, -math.inf):
        z = torch.ones(1, 64)
        z[0, 40] = bad
        c, s = mx.quantise(z, bits)
        y = mx.values(c, s, bits)
        assert torch.isnan(y[0, 32:]).all() and (y[0, :32] == 1).all() and not c[0, -32 * bits // 8:].any()


def test_oracle_window():
    """Row t sits at position len - T + t; what lies outside is neither written nor anything but zero."""
    cache = list(kv.mx_cache(4, 1, 6, 64, bits=8, device="cpu"))
    x = torch.arange(1, 4).view(1, 1, 3, 1).expand(4, 1, 3, 64).float()
    mx.append(cache, x, -x, [3, 1, 0, 8])
    k, v = mx.read(cache, [6] * 4, 6)
    assert k[..., 0].view(4, 6).tolist() == [[1, 2, 3, 0, 0, 0], [3, 0, 0, 0, 0, 0], [0] * 6, [0, 0, 0, 0, 0, 1]]
    assert torch.equal(v, -k)
    k, _ = mx.read(cache, [2, 0, -1, 7], 3)
    assert k[..., 0].view(4, 3).tolist() == [[0, 1, 2], [0, 0, 0], [0, 0, 0], [0, 1, 0]]


# ----------------------------------------------------------------------------- the C ABI

P = [0x100000 + 0x1000 * i for i in range(9)]  # aligned stand-ins: validation returns before use
OK = dict(B=1, Hq=4, Hkv=2, T=3, L=128, D=64, bits=4, dtype=_lib.TTFA_BF16, scale=0.125, strides=None)


def _append(ptrs=None, **kw):
    a = {**OK, **kw}
    s = (ctypes.c_longlong * 6)(*a["strides"]) if a["strides"] else None
    return _lib.load().ttfa_kv_append(*(ptrs or P[:7]), s, a["B"], a["Hkv"], a["T"], a["L"], a["D"],
                                      a["bits"], a["dtype"], None)


def _read(ptrs=None, **kw):
    a = {**OK, **kw}
    p = ptrs or P[:7]  # as _append's order: six aligned to 16, then the lengths
    return _lib.load().ttfa_kv_read(*p[2:6], p[6], p[0], p[1], a["B"], a["Hkv"], a["T"], a["L"], a["D"],
                                    a["bits"], a["dtype"], None)


def _decode(ptrs=None, **kw):
    a = {**OK, **kw}
    p = ptrs or P
    return _lib.load().ttfa_decode_mx_fwd(*p[:5], p[8], *p[5:8], a["B"], a["Hq"], a["Hkv"], a["T"], a["L"],
                                          a["D"], a["bits"], a["dtype"], a["scale"], None)


@needs_lib
@pytest.mark.parametrize("entry", [_append, _read, _decode])
@pytest.mark.parametrize("kw, code", [
    (dict(bits=2), _lib.E_BITS), (dict(bits=16), _lib.E_BITS), (dict(D=96), _lib.E_HEAD_DIM),
    (dict(Hkv=0), _lib.E_GROUP), (dict(B=0), _lib.E_SEQ), (dict(T=0), _lib.E_SEQ), (dict(L=0), _lib.E_SEQ),
    (dict(L=1 << 25), _lib.E_SEQ), (dict(B=1 << 20, Hkv=1 << 10, Hq=1 << 10), _lib.E_SEQ),
    (dict(dtype=2), _lib.E_DTYPE)])
def test_argument_errors_return_codes(entry, kw, code):
    assert entry(**kw) == code


@needs_lib
def test_argument_errors_of_one_entry():
    assert _decode(dtype=_lib.TTFA_F32) == _lib.E_DTYPE
    assert _decode(Hq=3) == _lib.E_GROUP
    assert _decode(T=17) == _lib.E_QROWS
    assert _decode(scale=math.nan) == _lib.E_SCALE
    for rows in (_append, _read):
        assert rows(B=1 << 10, Hkv=1 << 10, T=1 << 11) == _lib.E_SEQ  # 2^31 rows
    for bad in ([-8, 0, 0, 0, 0, 0], [0, 0, 0, 0, 12, 0], [0, 0, 0, 0, 0, 1 << 41]):
        assert _append(strides=bad) == _lib.E_STRIDE
    assert _append(strides=[0, 0, 0, 0, 0, 6], dtype=_lib.TTFA_F32) == _lib.E_STRIDE
    for code in (_lib.E_BITS, _lib.E_STRIDE):
        assert _lib.strerror(code).startswith("ttfa:") and "unknown" not in _lib.strerror(code)


@needs_lib
@pytest.mark.parametrize("entry, n", [(_append, 6), (_read, 6), (_decode, 8)])
def test_null_and_misaligned_pointers(entry, n):
    for i in range(n + 1):
        if entry is _decode and i == 7:
            continue   # the workspace: see test_workspace_bytes
        ptrs = list(P[:n + 1])
        ptrs[i] = None
        assert entry(ptrs=ptrs) == _lib.E_NULL
        ptrs[i] = P[i] + (2 if i == n else 8)   # the lengths, last, need 4 bytes
        assert entry(ptrs=ptrs) == _lib.E_ALIGN


@needs_lib
def test_workspace_bytes():
    w = lambda *a: _lib.load().ttfa_decode_mx_workspace_bytes(*a)  # noqa: E731
    assert w(1, 4, 2, 1, 128, 64, 3) == -1 and w(1, 4, 3, 1, 128, 64, 4) == -1
    assert w(1, 4, 2, 20, 128, 64, 4) == -1 and w(1, 4, 2, 1, 0, 64, 4) == -1
    for bits in (4, 8):
        assert w(3, 8, 2, 1, 512, 128, bits) == 0                   # one launch: not used
        n = w(2, 8, 2, 1, 50000, 128, bits)
        assert n % (2 * 8 * 130 * 4) == 0 and 1 < n // (2 * 8 * 130 * 4) <= 512
    for bad in (None, P[7] + 8):
        ptrs = [*P[:7], bad, P[8]]
        assert _decode(ptrs=ptrs, L=50000) == (_lib.E_NULL if bad is None else _lib.E_ALIGN)


# ------------------------------------------------------------------------ the Python operators

def _rows(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype)


def _cpu_cache(B=2, Hkv=2, L=10, D=64, bits=4):
    return kv.mx_cache(B, Hkv, L, D, bits, device="cpu")


def test_mx_cache_shapes():
    c = kv.mx_cache(2, 3, 7, 128, device="cpu")
    assert [tuple(t.shape) for t in c] == [(2, 3, 7, 64), (2, 3, 7, 4)] * 2
    assert all(t.dtype == torch.uint8 and not t.any() for t in c)
    assert kv.mx_cache(2, 3, 7, 64, 8, device="cpu").k_codes.shape[3] == 64
    for bad in (dict(bits=3), dict(bits=16), dict(D=96)):
        with pytest.raises(FlashAttnInputError):
            kv.mx_cache(**{**dict(B=1, Hkv=1, max_seqlen=4, D=64, device="cpu"), **bad})


LENS = torch.zeros(2, dtype=torch.int32)
BAD_CACHES = [
    (lambda c: (c[0][0], *c[1:]), LENS, "4-D uint8"),
    (lambda c: (c[0].to(torch.int8), *c[1:]), LENS, "uint8"),
    (lambda c: (c[0].transpose(1, 2), *c[1:]), LENS, "contiguous"),
    (lambda c: (*c[:2], c[2][:, :1].contiguous(), c[3]), LENS, "one cache"),
    (lambda c: (c[0][:, :, :5].contiguous(), c[1], c[2][:, :, :5].contiguous(), c[3]), LENS, "one cache"),
    (lambda c: (c[0], c[1][..., :1].contiguous(), c[2], c[3][..., :1].contiguous()), LENS, "head dim"),
    (lambda c: (c[0][..., :16].contiguous(), c[1], c[2][..., :16].contiguous(), c[3]), LENS, "bytes a row"),
    (lambda c: c, LENS.long(), "int32"),
    (lambda c: c, LENS[:1], "int32"),
    (lambda c: c, LENS, "ROCm GPU"),
]


@pytest.mark.parametrize("change, lens, match", BAD_CACHES)
def test_bad_caches_are_refused(change, lens, match):
    c = change(_cpu_cache())
    for call in (lambda: kv.kv_cache_append(_rows(2, 2, 3, 64), _rows(2, 2, 3, 64), *c, lens),
                 lambda: kv.kv_cache_read(*c, lens, 3),
                 lambda: kv.flash_attn_decode_mx(_rows(2, 4, 1, 64), *c, lens)):
        with pytest.raises(FlashAttnInputError, match=match):
            call()


@pytest.mark.parametrize("k, v, match", [
    (_rows(2, 2, 3, 64), _rows(2, 2, 2, 64), "must be"),
    (_rows(2, 4, 3, 64), _rows(2, 4, 3, 64), "must be"),
    (_rows(2, 2, 64), _rows(2, 2, 64), "must be"),
    (_rows(2, 2, 3, 128), _rows(2, 2, 3, 128), "must be"),
    (_rows(2, 2, 3, 64), _rows(2, 2, 3, 64, dtype=torch.float32), "bfloat16 or float32"),
    (_rows(2, 2, 3, 64, dtype=torch.float16), _rows(2, 2, 3, 64, dtype=torch.float16), "bfloat16 or float32"),
    (_rows(2, 2, 64, 3).transpose(2, 3), _rows(2, 2, 3, 64), "dense last"),
    (_rows(2, 2, 3, 68)[..., :64], _rows(2, 2, 3, 64), "16 bytes"),
])
def test_bad_rows_are_refused(k, v, match):
    with pytest.raises(FlashAttnInputError, match=match):
        kv.kv_cache_append(k, v, *_cpu_cache(), LENS)


@pytest.mark.parametrize("q, match", [
    (_rows(2, 4, 64), "must be"), (_rows(1, 4, 1, 64), "must be"), (_rows(2, 4, 1, 128), "must be"),
    (_rows(2, 3, 1, 64), "multiple"), (_rows(2, 4, 17, 64), "32 query rows"),
    (_rows(2, 4, 1, 64, dtype=torch.float32), "bfloat16"), (_rows(2, 2, 4, 64).transpose(1, 2), "contiguous"),
])
def test_bad_queries_are_refused(q, match):
    with pytest.raises(FlashAttnInputError, match=match):
        kv.flash_attn_decode_mx(q, *_cpu_cache(), LENS)


def test_bad_reads_are_refused():
    with pytest.raises(FlashAttnInputError, match="positive"):
        kv.kv_cache_read(*_cpu_cache(), LENS, 0)
    with pytest.raises(FlashAttnInputError, match="bfloat16 or float32"):
        kv.kv_cache_read(*_cpu_cache(), LENS, 3, torch.float16)


def test_fullgraph_trace_of_a_step_is_its_ops():
    """A whole step of generation under torch.compile: one node per operator, in order, with the
    cache's mutation known to the compiler (traced on fake tensors, without a GPU)."""
    ops = []

    def backend(gm, _):
        ops.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function")
        return gm.forward

    def step(q, k, v, cache, lens):
        kv.kv_cache_append(k, v, *cache, lens)
        o, lse = kv.flash_attn_decode_mx(q, *cache, lens)
        return o, lse, *kv.kv_cache_read(*cache, lens, 4)

    torch._dynamo.reset()
    with FakeTensorMode():
        cache = kv.mx_cache(2, 2, 90, 64, 8)
        t = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        lens = torch.empty(2, dtype=torch.int32, device="cuda")
        o, lse, k, v = torch.compile(step, backend=backend, fullgraph=True)(
            t(2, 4, 1, 64), t(2, 2, 1, 64), t(2, 2, 1, 64), cache, lens)
    assert [x for x in ops if "tinytrain" in x] == [
        f"tinytrain.{n}.default" for n in ("kv_cache_append", "flash_attn_decode_mx", "kv_cache_read")]
    assert o.shape == (2, 4, 1, 64) and lse.shape == (2, 4, 1) and k.shape == v.shape == (2, 2, 4, 64)
    schema = torch.ops.tinytrain.kv_cache_append.default._schema
    assert [a.name for a in schema.arguments if a.is_write] == ["k_codes", "k_scales", "v_codes", "v_scales"]


@needs_lib
def test_largest_calls():
    """Launches of 2^32 threads or more are refused; the calls below them get as far as the pointers."""
    null = [None] * 7
    for rows in (_append, _read):
        for dtype in (_lib.TTFA_BF16, _lib.TTFA_F32):
            most = ((1 << 34) - (1 << 13)) // (4 * 128)
            assert rows(ptrs=null, B=2, Hkv=2, T=most, D=128, dtype=dtype) == _lib.E_NULL
            assert rows(ptrs=null, B=2, Hkv=2, T=most + 1, D=128, dtype=dtype) == _lib.E_SEQ
    assert _decode(ptrs=[None] * 9, B=(1 << 22) - 1, Hq=4, Hkv=4, T=1) == _lib.E_NULL
    assert _decode(ptrs=[None] * 9, B=1 << 22, Hq=4, Hkv=4, T=1) == _lib.E_SEQ
    w = _lib.load().ttfa_decode_mx_workspace_bytes
    assert w(1 << 22, 4, 4, 1, 128, 64, 4) == -1 and w((1 << 22) - 1, 4, 4, 1, 128, 64, 4) == 0


def test_lengths_past_32_bits_are_refused():
    cache = [torch.empty(1, 1, 1 << 32, n, dtype=torch.uint8, device="meta") for n in (32, 2, 32, 2)]
    with pytest.raises(FlashAttnInputError, match="too large"):
        kv._check_cache(*cache, torch.zeros(1, dtype=torch.int32))


def test_oracle_positions_past_the_capacity():
    """Queries keep their positions where the newest rows no longer fit: row i of three sees
    len - 3 + i + 1 keys, or all that there are."""
    k = torch.zeros(5, 1, 6, 64, dtype=torch.float64)
    _, lse, _, _ = mx.decode(torch.zeros(5, 1, 3, 64), k, k, [6, 7, 8, 2**31 - 1, 1])
    assert lse.exp().round().view(5, 3).tolist() == [[4, 5, 6], [5, 6, 6], [6, 6, 6], [6, 6, 6], [0, 0, 1]]


@pytest.mark.parametrize("rows", [1 << 31, (1 << 32) + 1])
def test_row_counts_past_32_bits_are_refused(rows):
    """Expanded rows take no memory, so that such a call can be made: (1 << 32) + 1 rows are not one row."""
    k = _rows(1, 1, 1, 64).expand(1, 1, rows, 64)
    lens = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(FlashAttnInputError, match="too many"):
        kv.kv_cache_append(k, k, *_cpu_cache(1, 1), lens)
    with pytest.raises(FlashAttnInputError, match="too many"):
        kv.kv_cache_read(*_cpu_cache(1, 1), lens, rows)
