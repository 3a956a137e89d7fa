"""GPU tests of the quantised KV cache against its 64-bit oracle: what appends write and reads give, to the
bit; attention over the cache, within rounding; and the operators together, as a program uses them."""

import math

import pytest
import torch

from helpers import announce
from oracle import mx_cache as mx
from tinytrain_amd import _lib
from tinytrain_amd.kernels import kv_cache as kv
from tinytrain_amd.kernels.flash_attn import FlashAttnInputError, flash_attn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _lens(lens):
    return torch.tensor(lens, dtype=torch.int32, device=DEV)


def _noise_cache(B, Hkv, L, D, bits, seed=0):
    """A cache of random bytes (CPU), so that a stray write or a missed one shows."""
    g = torch.Generator().manual_seed(seed)
    n = (D * bits // 8, D // 32) * 2
    return [torch.randint(0, 255, (B, Hkv, L, m), dtype=torch.uint8, generator=g) for m in n]


def _gpu(cache):
    return [t.to(DEV) for t in cache]


def _cpu(ts):
    return [t.cpu() for t in ts]


def _wild(shape, seed, dtype):
    """Rows with zeros, tiny and huge groups, values on rounding borders, NaN and infinities."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).unflatten(-1, (-1, 32))
    kind = torch.randint(0, 12, x.shape[:-1], generator=g)[..., None]
    scale = torch.exp2(torch.randint(-30, 30, x.shape[:-1], generator=g).float())[..., None]
    border = torch.randint(-28, 29, x.shape, generator=g) / 4.0       # every e2m1 border, many e4m3 ones
    border[..., 0] = 7.0
    x = torch.where(kind < 3, border * scale, x * scale)
    x = torch.where(kind == 3, torch.zeros(()), x)
    x = torch.where(kind == 4, x * 1e-39, x)
    x = torch.where(kind == 5, torch.randn(x.shape, generator=g).clamp(-3, 3) * 1.1e38, x)
    x = torch.where(kind == 6, torch.where(torch.rand(x.shape, generator=g) < 0.6, torch.zeros(()), -x), x)
    spot = torch.randint(0, 32, x.shape[:-1], generator=g)[..., None] == torch.arange(32)
    x = torch.where((kind == 7) & spot, math.nan, x)
    x = torch.where((kind == 8) & spot, -math.inf, x)
    return x.flatten(-2).to(dtype)


# ------------------------------------------------------------------------- append and read

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B, Hkv, T, L, D, lens", [
    (1, 1, 1, 1, 64, [1]),
    (3, 2, 1, 40, 128, [40, 1, 17]),
    (4, 3, 37, 41, 64, [41, 37, 20, 0]),            # left padding, an empty sequence
    (5, 2, 9, 12, 128, [-3, 60, 14, 9, 12]),        # nothing, all past the end, some past the end
    (2, 1, 300, 257, 64, [257, 290]),               # more rows than the cache has
])
def test_append_writes_the_oracles_bytes(B, Hkv, T, L, D, lens, bits, dtype):
    announce(f"kv append B={B} Hkv={Hkv} T={T} L={L} D={D} bits={bits} {dtype} lens={lens}")
    k, v = _wild((B, Hkv, T, D), 1, dtype), _wild((B, Hkv, T, D), 2, dtype)
    want = _noise_cache(B, Hkv, L, D, bits)
    got = _gpu(want)
    kv.kv_cache_append(k.to(DEV), v.to(DEV), *got, _lens(lens))
    mx.append(want, k, v, lens)
    for name, a, b in zip(kv.MXCache._fields, _cpu(got), want):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("bits", [4, 8])
def test_append_of_every_bf16_value(bits):
    """Each finite bf16 value in a group of its own scale and in one of a larger scale."""
    announce(f"kv append all bf16 bits={bits}")
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    x = x[torch.isfinite(x)]
    k = torch.zeros(1, 1, len(x), 64, dtype=BF)
    k[0, 0, :, 5] = x
    k[0, 0, :, 32] = x
    k[0, 0, :, 40] = (x.float().abs().clamp(max=1e37) * 9.5).to(BF)
    got = _gpu(kv.mx_cache(1, 1, len(x), 64, bits, device="cpu"))
    kv.kv_cache_append(k.to(DEV), k.to(DEV), *got, _lens([len(x)]))
    c, s = mx.quantise(k, bits)
    for a, b in zip(_cpu(got), (c, s, c, s)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_of_strided_rows(dtype):
    """Rows as projections lay them out [B, T, H, D], slices of wider ones, an expanded batch, and K and
    V of different strides."""
    announce(f"kv append strides {dtype}")
    B, Hkv, T, L, D = 3, 2, 5, 9, 64
    lens = [9, 5, 3]
    dense = [_wild((B, Hkv, T, D), s, dtype) for s in (3, 4)]
    wide = torch.zeros(B, T, 2 * Hkv, D + 32, dtype=dtype, device=DEV)
    wide[:, :, ::2, 16:16 + D] = dense[0].transpose(1, 2).to(DEV)
    k = wide[:, :, ::2, 16:16 + D].transpose(1, 2)
    v = dense[1].transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    assert k.stride() != v.stride() and not k.is_contiguous()
    want = _noise_cache(B, Hkv, L, D, 4)
    got = _gpu(want)
    kv.kv_cache_append(k, v, *got, _lens(lens))
    mx.append(want, *dense, lens)
    assert all(torch.equal(a, b) for a, b in zip(_cpu(got), want))
    one = dense[0][:1].to(DEV)
    got, want = _gpu(want), want
    kv.kv_cache_append(one.expand(B, Hkv, T, D), one.expand(B, Hkv, T, D), *got, _lens(lens))
    mx.append(want, *(dense[0][:1].expand(B, Hkv, T, D),) * 2, lens)
    assert all(torch.equal(a, b) for a, b in zip(_cpu(got), want))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B, Hkv, rows, L, D, lens", [
    (1, 1, 1, 1, 64, [1]),
    (4, 3, 37, 41, 64, [41, 37, 20, 0]),
    (5, 2, 9, 12, 128, [-3, 60, 14, 9, 12]),
    (2, 1, 300, 257, 128, [257, 290]),
])
def test_read_gives_the_oracles_values(B, Hkv, rows, L, D, lens, bits, dtype):
    announce(f"kv read B={B} Hkv={Hkv} rows={rows} L={L} D={D} bits={bits} {dtype} lens={lens}")
    cache = list(kv.mx_cache(B, Hkv, L, D, bits, device="cpu"))
    mx.append(cache, _wild((B, Hkv, L, D), 5, BF), _wild((B, Hkv, L, D), 6, BF), [L] * B)
    got = kv.kv_cache_read(*_gpu(cache), _lens(lens), rows, dtype)
    for a, b in zip(got, mx.read(cache, lens, rows)):
        assert a.dtype == dtype and a.is_contiguous() and torch.equal(torch.isnan(a.cpu()), torch.isnan(b))
        assert torch.equal(a.cpu().double().nan_to_num(0.5), b.nan_to_num(0.5))


def test_every_code_reads_as_its_value():
    """All codes under all scales that an append can write, in both types."""
    announce("kv read all codes")
    for bits, lo, hi in ((4, 2, 252), (8, 10, 246)):
        n, D = hi - lo + 1, 64
        codes = torch.arange(256, dtype=torch.uint8)
        if bits == 8:
            codes[127] = codes[255] = 0
        codes = codes.view(1, -1, 1, D * bits // 8).expand(1, -1, n, -1).contiguous()
        scales = torch.arange(lo, hi + 1).to(torch.uint8).view(1, 1, n, 1).expand(1, codes.shape[1], n, 2).contiguous()
        cache = [codes, scales, codes.clone(), scales.clone()]
        for dtype in (BF, F32):
            k, v = kv.kv_cache_read(*_gpu(cache), _lens([n]), n, dtype)
            want = mx.values(codes, scales, bits)
            assert torch.equal(k.cpu().double(), want) and torch.equal(v, k)


# ------------------------------------------------------------------------------ attention

def _filled(B, Hkv, L, D, bits, seed=0, device="cpu"):
    """(cache, fp64 K, fp64 V): unit-RMS keys with uneven channels, normal values."""
    g = torch.Generator(device).manual_seed(seed)
    k = torch.randn(B, Hkv, L, D, generator=g, device=device)
    k = k * torch.rsqrt(k.pow(2).mean(-1, keepdim=True)) * (1 + 0.2 * torch.randn(D, generator=g, device=device))
    v = torch.randn(B, Hkv, L, D, generator=g, device=device)
    cache = []
    for x in (k, v):
        cache += mx.quantise(x.to(BF).cpu(), bits)
    return cache, mx.values(*cache[:2], bits), mx.values(*cache[2:], bits)


def _queries(B, Hq, Tq, D, seed=0):
    g = torch.Generator().manual_seed(seed + 1000)
    q = torch.randn(B, Hq, Tq, D, generator=g)
    return (q * torch.rsqrt(q.pow(2).mean(-1, keepdim=True))).to(BF)


def _cut(q, k):
    """The largest sum over eights of |q_d k_d|'s maximum, over a row's keys, / sqrt(D)."""
    G, D = q.shape[1] // k.shape[1], q.shape[3]
    q, k = q.double().abs().nan_to_num(0, 0, 0), k.abs().nan_to_num(0)
    rows = torch.zeros(*q.shape[:3], k.shape[2], dtype=torch.float64)
    for d in range(0, D, 8):
        top = 0.0
        for j in range(d, d + 8):
            x = q[..., j].unflatten(1, (-1, G))[..., None] * k[:, :, None, None, :, j]
            top = x if j == d else torch.maximum(top, x)
        rows += top.flatten(1, 2)
    return rows.amax(-1) / math.sqrt(D)


def _bounds(o, a, big, cut, L, D):
    """Element-wise bounds of O and LSE, from the roundings on the way.

    K, V and Q enter the products exactly, but for elements of Q below 2^-13 of the row's largest, which
    may lose 2^-21 of that.  Of eight consecutive products of a score the matrix unit cuts every bit
    below 2^-13 of the largest: less than 7 2^-13 of it for Q's first term, 2^-4 of that for its
    second.  7 (1 + 2^-4) < 7.5: the cuts, and what such small elements lose, stay within 2^-10 of `cut`, the
    sum of the eights' largest products.  The sums of the eights are fp32, of size S =
    `big` (|error| <= D 2^-24 S), scaled and shifted by the maximum in fp32 (two roundings of at most S
    each); exp2 and log2 are good to 2^-21; a sum of L terms in fp32 adds L 2^-24.  So a weight
    is off by d = 2^-10 cut + (D + 4) 2^-24 S + L 2^-24 + 2^-20, relatively, twice (weight and sum);
    rounding the weights to bf16 adds 2^-8 of A = sum p |v|, rounding O to bf16 2^-8 of itself."""
    d = 2.0**-10 * cut + (D + 4) * 2.0**-24 * big + L * 2.0**-24 + 2.0**-20
    return (2.0**-8 + 2 * d[..., None]) * a * (1 + 2.0**-8) + 2.0**-8 * o.abs(), 2 * d + 2.0**-20


def _check(q, cache, lens, k, v, got, L):
    o, lse, a, big = mx.decode(q, k, v, lens)
    tol_o, tol_lse = _bounds(o, a, big, _cut(q, k), L, q.shape[3])
    go, gl = (t.double().cpu() for t in got)
    assert got[0].dtype == BF and got[1].dtype == F32
    seen = torch.isfinite(lse)
    assert torch.equal(torch.isfinite(gl), seen) and (gl[~seen] == -math.inf).all()
    assert ((go - o).abs() <= tol_o).all(), ((go - o).abs() / tol_o.clamp(min=1e-30)).max()
    assert ((gl - lse)[seen].abs() <= tol_lse[seen]).all(), ((gl - lse)[seen].abs() / tol_lse[seen]).max()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B, Hq, Hkv, Tq, L, D, lens", [
    (1, 1, 1, 1, 1, 64, [1]),
    (2, 8, 2, 1, 512, 128, [512, 33]),               # one launch
    (4, 4, 4, 1, 31, 64, [31, 1, 0, -2]),            # inside one block, empty caches
    (3, 4, 2, 3, 97, 128, [2, 97, 64]),              # rows without keys
    (1, 16, 1, 1, 700, 128, [700]),                  # 16 columns, one tile
    (2, 17, 1, 1, 333, 64, [333, 32]),               # 17: two tiles
    (2, 32, 4, 4, 1500, 128, [1500, 777]),           # 32
    (2, 6, 2, 5, 600, 64, [600, 4]),                 # 15 columns, an odd number of rows
    (1, 12, 4, 1, 5000, 64, [4999]),                 # many chunks
    (1, 16, 8, 1, 5001, 128, [5001]),
    (9, 12, 12, 1, 1301, 64, [1301 - 160 * i for i in range(9)]),
    (20, 8, 8, 2, 900, 128, [max(900 - 47 * i, 0) for i in range(20)]),
    (3, 8, 2, 1, 600, 128, [700, 601, 600]),         # longer than the cache: clamped
])
def test_decode_matches_oracle(B, Hq, Hkv, Tq, L, D, lens, bits):
    announce(f"decode_mx B={B} Hq={Hq} Hkv={Hkv} Tq={Tq} L={L} D={D} bits={bits} lens={lens[:4]}")
    cache, k, v = _filled(B, Hkv, L, D, bits)
    q = _queries(B, Hq, Tq, D)
    got = kv.flash_attn_decode_mx(q.to(DEV), *_gpu(cache), _lens(lens))
    _check(q, cache, lens, k, v, got, L)


@pytest.mark.parametrize("bits, D", [(4, 128), (8, 64)])
def test_decode_of_sharp_and_flat_scores(bits, D):
    """Scores far apart (one key takes all, the maximum grows from block to block) and all equal."""
    announce(f"decode_mx sharp bits={bits}")
    B, Hkv, L = 2, 2, 3000
    cache, k, v = _filled(B, Hkv, L, D, bits, seed=3)
    q = _queries(B, 4, 1, D)
    ramp = torch.linspace(0.1, 30, L)[:, None] * q[:, ::2, 0, None].float().sign()
    c, s = mx.quantise(ramp.to(BF), bits)
    for codes, scales in ((c, s), mx.quantise(torch.zeros(B, Hkv, L, D), bits)):
        now = [codes, scales, *cache[2:]]
        got = kv.flash_attn_decode_mx(q.to(DEV), *_gpu(now), _lens([L, 1999]))
        _check(q, now, [L, 1999], mx.values(codes, scales, bits), v, got, L)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B, Hkv, L, D", [(1, 2, 500, 128), (3, 2, 4000, 64), (40, 4, 1000, 128)])
def test_decode_rows_do_not_depend_on_the_other_caches(B, Hkv, L, D, bits):
    """A sequence's bits go by the call's shape and its own cache: whatever lies behind its last row, and
    whatever the others hold (NaN everywhere, nothing)."""
    announce(f"decode_mx neighbours B={B} L={L} D={D} bits={bits}")
    cache, _, _ = _filled(B, Hkv, L, D, bits)
    q, n = _queries(B, 2 * Hkv, 1, D).to(DEV), L - 45
    lens = torch.full((B,), L, dtype=torch.int32)
    lens[0] = n
    want = kv.flash_attn_decode_mx(q, *_gpu(cache), lens.to(DEV))
    other = _gpu(cache)
    for t in other:
        t[0, :, n:] = 255
        t[1:] = 255
    for rest in (L, 40, 0):
        lens[1:] = rest
        got = kv.flash_attn_decode_mx(q, *other, lens.to(DEV))
        assert all(torch.equal(a[0], b[0]) for a, b in zip(got, want))


@pytest.mark.parametrize("L, D, lens, at", [
    (512, 128, [512, 20], [511, 19]), (512, 64, [500, 33], [499, 32]), (512, 64, [500, 33], [250, 0]),
    (3000, 128, [3000, 65], [2998, 64]), (3000, 64, [2999, 3], [2997, 0]), (3000, 128, [3000, 64], [2969, 62]),
])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_nan_groups_reach_the_rows_that_see_them(L, D, lens, at, which, bits):
    """A NaN group of K makes O and LSE of exactly the rows that see its key NaN; one of V makes the 32
    elements of O NaN that it adds to.  Every other value keeps its bits."""
    announce(f"decode_mx NaN L={L} D={D} lens={lens} at={at} {which} bits={bits}")
    Tq, Hkv, Hq = 3, 2, 4
    cache, _, _ = _filled(2, Hkv, L, D, bits, seed=5)
    q = _queries(2, Hq, Tq, D).to(DEV)
    clean = kv.flash_attn_decode_mx(q, *_gpu(cache), _lens(lens))
    codes, scales = (0, 1) if which == "k" else (2, 3)
    for b in range(2):
        cache[scales][b, 1, at[b], 1] = 255
        cache[codes][b, 1, at[b], 4 * bits:8 * bits] = 0
    o, lse = kv.flash_attn_decode_mx(q, *_gpu(cache), _lens(lens))
    pos = torch.tensor(lens)[:, None] + torch.arange(-Tq, 0)
    bad = torch.zeros(2, Hq, Tq, D, dtype=torch.bool)
    bad[:, 2:] = (torch.tensor(at)[:, None] <= pos)[:, None, :, None]
    rows = bad[..., 0].to(DEV) & (which == "k")
    if which == "v":
        bad[..., :32] = bad[..., 64:] = False
    bad = bad.to(DEV)
    assert torch.equal(torch.isnan(o), bad) and torch.equal(torch.isnan(lse), rows)
    assert torch.equal(o[~bad], clean[0][~bad]) and torch.equal(lse[~rows], clean[1][~rows])


def test_decode_agrees_with_attention_over_the_rows_read_back():
    """The last rows of the batched forward over kv_cache_read's K and V, within both paths' roundings."""
    announce("decode_mx vs forward over read rows")
    B, Hq, Hkv, T, D, Tq = 2, 8, 2, 700, 128, 2
    cache, k, v = _filled(B, Hkv, T, D, 4, seed=7)
    q = _queries(B, Hq, T, D).to(DEV)
    lens = _lens([T] * B)
    dense = kv.kv_cache_read(*_gpu(cache), lens, T)
    full = flash_attn(q, *dense)[:, :, T - Tq:]
    qt = q[:, :, T - Tq:].contiguous()
    o, _ = kv.flash_attn_decode_mx(qt, *_gpu(cache), lens)
    want, _, a, big = mx.decode(qt.cpu(), k, v, [T] * B)
    tol, _ = _bounds(want, a, big, _cut(qt.cpu(), k), T, D)
    assert ((o - full).double().abs().cpu() <= 2 * tol).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_beyond_32_bit_offsets(bits):
    """A cache whose codes pass 4 GiB: rows of its last head, and of the last positions of a long one."""
    announce(f"kv long cache bits={bits}")
    D, Hkv, B = 128, 2, 3
    L = 4_300_000_000 // (D * bits // 8 * B * Hkv) + 1
    cache = kv.mx_cache(B, Hkv, L, D, bits)
    assert cache.k_codes.numel() > 1 << 32
    k, v = (_wild((B, Hkv, 70, D), s, BF) for s in (8, 9))
    k, v = (torch.where(torch.isfinite(t.float()), t, 1.0).clamp(-4, 4) for t in (k, v))
    lens = [L, L - 31, L]
    kv.kv_cache_append(k.to(DEV), v.to(DEV), *cache, _lens(lens))
    got = kv.kv_cache_read(*cache, _lens(lens), 70)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x.cpu().double(), mx.values(*mx.quantise(y, bits), bits))
    # keys that are zeros everywhere else: their score is 0 and they add exp(0) each
    q = _queries(B, 4, 1, D)
    o, lse = kv.flash_attn_decode_mx(q.to(DEV), *cache, _lens(lens))
    kk, vv = (mx.values(*mx.quantise(y, bits), bits) for y in (k, v))
    for h in range(4):
        s = (kk[:, h // 2] @ q[:, h, 0].double()[..., None])[..., 0] / math.sqrt(D)
        w = torch.exp(s)
        total = w.sum(-1) + torch.tensor(lens) - 70
        want = (w[:, None] @ vv[:, h // 2])[:, 0] / total[:, None]
        size = (w[:, None] @ vv[:, h // 2].abs())[:, 0] / total[:, None]
        # sums of up to L terms in fp32, each lane's part of at most L / 64 of them
        tol = (2.0**-8 + L / 64 * 2.0**-24 + 2.0**-10) * size + 2.0**-8 * want.abs()
        assert ((o[:, h, 0].cpu().double() - want).abs() <= tol).all()
        assert ((lse[:, h, 0].cpu().double() - torch.log(total)).abs() <= L / 64 * 2.0**-24 + 2.0**-10).all()


# ------------------------------------------------------------------------------- together

@pytest.mark.parametrize("bits", [4, 8])
def test_generation_step_by_step(bits):
    """A left-padded batch of prompts, then tokens one at a time and two at once: after every step the
    cache is what the oracle holds and attention over it is right."""
    announce(f"kv generation bits={bits}")
    B, Hq, Hkv, D, T, L = 3, 4, 2, 64, 50, 64
    prompt = [50, 17, 1]
    want = list(kv.mx_cache(B, Hkv, L, D, bits, device="cpu"))
    cache = kv.mx_cache(B, Hkv, L, D, bits)
    lens = _lens(prompt)
    g = torch.Generator().manual_seed(4)
    for rows in (T, 1, 1, 2, 1, 4):
        if rows != T:
            lens += rows
        k, v = (torch.randn(B, Hkv, rows, D, generator=g).to(BF) for _ in range(2))
        q = _queries(B, Hq, min(rows, 8), D, seed=rows)
        kv.kv_cache_append(k.to(DEV), v.to(DEV), *cache, lens)
        got = kv.flash_attn_decode_mx(q.to(DEV), *cache, lens)
        now = lens.tolist()
        mx.append(want, k, v, now)
        assert all(torch.equal(a, b) for a, b in zip(_cpu(cache), want))
        _check(q, want, now, *mx.read(want, [L] * B, L), got, L)


def test_step_replays_in_a_graph():
    """A step of generation captured in a HIP graph and replayed, the lengths advanced in the graph, with
    eager work and synchronisations in between: every replay equals eager calls, bitwise."""
    announce("kv graph replays")
    B, Hq, Hkv, D, L = 2, 16, 8, 128, 6000
    filled, _, _ = _filled(B, Hkv, L, D, 4, seed=11)
    cache, eager = _gpu(filled), _gpu(filled)
    lens = _lens([5900, 100])
    q, k, v = (torch.empty(B, h, 1, D, dtype=BF, device=DEV) for h in (Hq, Hkv, Hkv))

    def step(c, n):
        n += 1
        kv.kv_cache_append(k, v, *c, n)
        return (*kv.flash_attn_decode_mx(q, *c, n), *kv.kv_cache_read(*c, n, 5))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in cache], lens.clone())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache, lens)
    mine = lens.clone()
    for r in range(4):
        for t, seed in ((q, 0), (k, 1), (v, 2)):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * r + seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager, mine)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r
        assert all(torch.equal(a, b) for a, b in zip(cache, eager)) and torch.equal(lens, mine), r


def test_native_path_and_ops_give_the_same_bits():
    announce("kv native path")
    ops = torch.ops.tinytrain
    filled, _, _ = _filled(2, 2, 300, 64, 8, seed=12)
    a, b = _gpu(filled), _gpu(filled)
    q, k = _queries(2, 4, 2, 64).to(DEV), _queries(2, 2, 7, 64, seed=1).to(DEV)
    lens = torch.stack([_lens([300, 150])] * 2, 1)[:, 0]         # strided lengths
    assert not lens.is_contiguous()
    version = a[0]._version
    assert kv.kv_cache_append(k, k, *a, lens) is None and a[0]._version > version
    ops.kv_cache_append(k, k, *b, lens)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and not torch.equal(a[0].cpu(), filled[0])
    for x, y in zip(kv.flash_attn_decode_mx(q, *a, lens), ops.flash_attn_decode_mx(q, *b, lens)):
        assert torch.equal(x, y)
    for dtype in (BF, F32):
        for x, y in zip(kv.kv_cache_read(*a, lens, 9, dtype), ops.kv_cache_read(*b, lens, 9, dtype)):
            assert torch.equal(x, y) and x.dtype == dtype
    with torch.inference_mode():
        c = kv.mx_cache(2, 2, 300, 64, 8)
        kv.kv_cache_append(k, k, *c, lens)
        assert torch.equal(kv.kv_cache_read(*c, lens, 7)[0], kv.kv_cache_read(*a, lens, 7)[0])
    torch.library.opcheck(kv.flash_attn_decode_mx, (q, *a, lens), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(kv.kv_cache_read, (*a, lens, 5), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(kv.kv_cache_append, (k, k, *a, lens), test_utils=("test_schema", "test_faketensor"))


def test_compiled_step_mutates_the_cache():
    announce("kv torch.compile")
    filled, _, _ = _filled(2, 2, 100, 64, 4, seed=13)
    a, b = _gpu(filled), _gpu(filled)
    q, k = _queries(2, 4, 1, 64).to(DEV), _queries(2, 2, 1, 64, seed=1).to(DEV)

    def step(q, k, v, c, lens):
        kv.kv_cache_append(k * 2, v, *c, lens)
        return kv.flash_attn_decode_mx(q, *c, lens)

    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    for n in (60, 61):
        want, got = step(q, k, k, a, _lens([n, 5])), compiled(q, k, k, b, _lens([n, 5]))
        assert all(torch.equal(x, y) for x, y in zip(want, got))
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_calls_on_side_streams_and_determinism():
    from concurrent.futures import ThreadPoolExecutor

    announce("kv streams")
    filled, _, _ = _filled(3, 4, 5000, 128, 4, seed=14)
    cache = _gpu(filled)
    q, lens = _queries(3, 8, 1, 128).to(DEV), _lens([5000, 4000, 7])
    k = _queries(3, 4, 4, 128, seed=2).to(DEV)
    kv.kv_cache_append(k, k, *cache, lens)
    want = (*kv.flash_attn_decode_mx(q, *cache, lens), *kv.kv_cache_read(*cache, lens, 50))
    torch.cuda.synchronize()

    def work(_):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            mine = [t.to(DEV) for t in filled]
            kv.kv_cache_append(k, k, *mine, lens)
            got = (*kv.flash_attn_decode_mx(q, *mine, lens), *kv.kv_cache_read(*mine, lens, 50))
        s.synchronize()
        return all(torch.equal(a, b) for a, b in zip(got, want))

    with ThreadPoolExecutor(4) as ex:
        assert all(ex.map(work, range(8)))


def test_refusals_on_the_gpu():
    announce("kv refusals")
    cache = kv.mx_cache(2, 2, 10, 64)
    lens, k = _lens([3, 3]), torch.zeros(2, 2, 3, 64, dtype=BF, device=DEV)
    with pytest.raises(FlashAttnInputError, match="four tensors"):
        kv.kv_cache_append(k, k, cache.k_codes, cache.k_scales, cache.k_codes, cache.v_scales, lens)
    with pytest.raises(FlashAttnInputError, match="ROCm GPU"):
        kv.kv_cache_append(k.cpu(), k, *cache, lens)
    with pytest.raises(FlashAttnInputError, match="ROCm GPU"):
        kv.kv_cache_read(*cache, lens.cpu(), 3)
    with pytest.raises(FlashAttnInputError, match="16 bytes"):
        kv.kv_cache_append(torch.zeros(2, 2, 3, 68, dtype=BF, device=DEV)[..., :64], k, *cache, lens)
    with pytest.raises(FlashAttnInputError, match="bfloat16"):
        kv.flash_attn_decode_mx(k.float(), *cache, lens)
    with pytest.raises(FlashAttnInputError, match="positive"):
        kv.kv_cache_read(*cache, lens, 0)
    with pytest.raises(_lib.TTFAError, match="aligned"):
        kv.kv_cache_append(torch.zeros(2 * 2 * 3 * 64 + 1, dtype=BF, device=DEV)[1:].view(2, 2, 3, 64), k, *cache, lens)
    with pytest.raises(_lib.TTFAError):
        kv.kv_cache_append(k[:, :, :0], k[:, :, :0], *cache, lens)
    assert not any(t.any() for t in cache)


# ------------------------------------------------------- both sides of the rules on sizes

def _decode_tiled(B, Hq, Hkv, Tq, L, D, bits, lens):
    """Attention of a batch that repeats three sequences (caches, queries, lengths) B times in turn: the first
    three against the oracle, every repeat bit by bit against its first."""
    cache, k, v = _filled(3, Hkv, L, D, bits, seed=L + B)
    q = _queries(3, Hq, Tq, D)
    turn = torch.arange(B, device=DEV) % 3
    got = kv.flash_attn_decode_mx(q.to(DEV)[turn], *(t[turn] for t in _gpu(cache)), _lens(lens)[turn])
    n = min(B, 3)
    _check(q[:n], cache, lens[:n], k[:n], v[:n], [t[:n] for t in got], L)
    assert all(torch.equal(t, t[:3][turn]) for t in got)


def _chunks(B, Hq, Hkv, Tq, L, D, bits):
    n = _lib.load().ttfa_decode_mx_workspace_bytes(B, Hq, Hkv, Tq, L, D, bits)
    return n // (B * Hq * Tq * (D + 2) * 4) or 1


@pytest.mark.parametrize("B, Hq, Hkv, Tq, L, D, bits, chunks", [
    (3, 4, 2, 1, 768, 64, 4, 1), (3, 4, 2, 1, 769, 64, 4, 4),               # one launch, or two
    (32, 8, 4, 1, 1024, 128, 8, 1), (32, 8, 4, 1, 1025, 128, 8, 2),
    (9, 8, 8, 1, 1024, 64, 8, 3), (33, 8, 4, 2, 1025, 128, 8, 1),           # 72 and 132 units
    (33, 8, 4, 2, 1472, 128, 4, 1), (33, 8, 4, 2, 1473, 128, 4, 1),         # four waves, eight
    (33, 16, 4, 8, 512, 128, 4, 1), (33, 20, 4, 5, 513, 64, 4, 1),          # two tiles: four, eight
    (33, 4, 4, 3, 1473, 64, 8, 1), (33, 20, 4, 4, 1500, 128, 8, 1),         # rows of 64 and 128 bytes
    (65, 8, 4, 1, 1984, 64, 8, 1), (65, 8, 4, 2, 1985, 128, 8, 1),          # 260 units: four, eight
    (65, 20, 4, 4, 1985, 128, 8, 1), (65, 16, 4, 8, 1985, 64, 4, 1),
    (149, 6, 3, 1, 2000, 64, 8, 1), (112, 4, 4, 6, 2000, 64, 4, 1),         # 447 and 448
    (1, 8, 8, 1, 8191, 128, 4, 16), (1, 8, 8, 1, 8192, 128, 4, 32),         # the two merges
    (1, 8, 8, 3, 16383, 64, 8, 16), (1, 8, 8, 3, 16384, 64, 8, 32),
    (66, 4, 4, 1, 4096, 64, 4, 1), (66, 4, 4, 1, 4097, 64, 4, 2),           # chunks for long among short
    (2, 17, 1, 1, 1333, 64, 8, 6), (2, 6, 2, 5, 1600, 64, 4, 7), (3, 11, 1, 2, 1100, 128, 4, 5),
    (2, 32, 1, 1, 32768, 128, 8, 128), (2, 1, 1, 32, 32767, 64, 4, 16),
])
def test_decode_on_both_sides_of_every_bound(B, Hq, Hkv, Tq, L, D, bits, chunks):
    announce(f"decode_mx bounds B={B} Hq={Hq} Hkv={Hkv} Tq={Tq} L={L} D={D} bits={bits}")
    assert _chunks(B, Hq, Hkv, Tq, L, D, bits) == chunks
    _decode_tiled(B, Hq, Hkv, Tq, L, D, bits, [L, 70, Tq - 1] if L % 2 else [L - 1, 300, 1])


@pytest.mark.parametrize("D, B, Hkv, T", [(128, 3, 5, 8738), (128, 3, 5, 8739), (64, 2, 7, 18725)])
@pytest.mark.parametrize("bits", [4, 8])
def test_moves_of_many_rows(D, B, Hkv, T, bits):
    """One and two rows at a time (2^21 lanes on), with a last workgroup that is part empty, rows before the
    cache's first and past its last."""
    announce(f"kv large moves D={D} B={B} Hkv={Hkv} T={T} bits={bits}")
    L, lens = T - 100, ([T - 100, T // 3, T - 90][:B])
    g = torch.Generator().manual_seed(T)
    k = torch.randn(B, Hkv, T, D, generator=g).to(BF)
    codes, scales = mx.quantise(k, bits)
    want = _noise_cache(B, Hkv, L, D, bits)
    got = _gpu(want)
    kv.kv_cache_append(k.to(DEV), -k.to(DEV), *got, _lens(lens))
    sign = 0x88 if bits == 4 else 0x80
    for b, n in enumerate(lens):
        lo, hi = max(n - T, 0), min(n, L)
        rows = slice(lo - n + T, hi - n + T)
        for c, m in ((0, 0), (2, sign)):
            want[c][b, :, lo:hi], want[c + 1][b, :, lo:hi] = codes[b, :, rows] ^ m, scales[b, :, rows]
    assert all(torch.equal(a, b) for a, b in zip(_cpu(got), want))
    plain = mx.values(codes, scales, bits).float()
    for dtype in (BF, F32):
        rk, rv = kv.kv_cache_read(*got, _lens(lens), T, dtype)
        assert torch.equal(rv, -rk)
        for b, n in enumerate(lens):
            lo, hi = max(T - n, 0), min(L - n + T, T)
            assert torch.equal(rk[b, :, lo:hi].cpu().float(), plain[b, :, lo:hi])
            assert not rk[b, :, :lo].any() and not rk[b, :, hi:].any()


# ------------------------------------------------------------------------- unusual queries

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B, Hkv, L, D", [(1, 1, 200, 64), (2, 1, 3000, 128), (33, 4, 600, 128)])
def test_unusual_queries(B, Hkv, L, D, bits):
    """Rows of zeros, tiny and huge rows, elements far below the row's largest, subnormal rows, and rows
    with a NaN or an infinity, which alone come out NaN."""
    announce(f"decode_mx queries B={B} Hkv={Hkv} L={L} D={D} bits={bits}")
    G = 12
    cache, k, v = _filled(B, Hkv, L, D, bits, seed=21)
    q = _queries(B, G * Hkv, 1, D).unflatten(1, (Hkv, G))
    q[:, :, 1] = 0
    q[:, :, 2] *= 2.0**-100
    q[:, :, 3] = (q[:, :, 3].float() * 2.0**-131).to(BF)
    q[:, :, 4] *= 2.0**100
    q[:, :, 5] = q[:, :, 5] * torch.exp2(-torch.arange(D) % 23.0).to(BF)
    q[:, :, 6, 0, D // 2:] *= 2.0**-18
    q[:, :, 7] *= 100
    q[:, :, 8, 0, 5] = math.nan
    q[:, :, 9, 0, D - 1] = math.inf
    q[:, :, 10, 0, 0] = -math.inf
    q = q.flatten(1, 2)
    lens = [L - i for i in range(B)]
    o, lse = kv.flash_attn_decode_mx(q.to(DEV), *_gpu(cache), _lens(lens))
    bad = torch.zeros(B, Hkv, G, 1, dtype=torch.bool)
    bad[:, :, 8:11] = True
    bad = bad.flatten(1, 2)
    assert torch.equal(torch.isnan(lse).cpu(), bad)
    assert torch.equal(torch.isnan(o).cpu(), bad[..., None].expand_as(o))
    clean = torch.where(bad[..., None], 0.0, q.float()).to(BF)
    wo, wl, a, big = mx.decode(clean, k, v, lens)
    # elements of q far below the row's largest may each lose 2^-21 of that
    kk = k.abs().sum(-1).amax(-1).repeat_interleave(G, 1)[..., None]
    lost = 2.0**-21 * clean.double().abs().amax(-1) * kk / math.sqrt(D)
    tol, tol_lse = _bounds(wo, a, big, _cut(clean, k) + 2.0**10 * lost, L, D)
    # weights below 2^-126 of the largest are 0 in fp32: each of L keys may miss that much of its value
    most = v.abs().amax((2, 3)).repeat_interleave(G, 1)[..., None, None]
    tol = tol + 2.0**-126 * L * most
    err = (o.cpu().double() - wo).abs()
    assert (err <= tol)[~bad].all(), (err / tol)[~bad].max()
    # a huge row keeps to the largest score, relatively
    assert ((lse.cpu().double() - wl).abs() <= tol_lse)[~bad].all()
    # its O stays a mixture of the values (weights and O rounded to bf16)
    assert (o.cpu().double().abs() <= most * (1 + 2.0**-6))[~bad].all()


def test_inputs_that_require_grad_are_read_alike():
    """The operators have no backward; under autograd they give what they give without."""
    announce("kv requires_grad")
    filled, _, _ = _filled(2, 2, 90, 64, 4, seed=31)
    a, b = _gpu(filled), _gpu(filled)
    q, k = _queries(2, 4, 1, 64).to(DEV), _queries(2, 2, 3, 64, seed=1).to(DEV)
    lens = _lens([90, 40])
    kv.kv_cache_append(k, k, *a, lens)
    want = kv.flash_attn_decode_mx(q, *a, lens)
    leaf = k.clone().requires_grad_()
    kv.kv_cache_append(leaf, leaf * 1, *b, lens)
    got = kv.flash_attn_decode_mx(q.clone().requires_grad_(), *b, lens)
    assert all(torch.equal(x, y) for x, y in zip((*a, *want), (*b, *got)))
    assert not any(t.requires_grad for t in b) and leaf.grad is None


def test_two_graphs_of_one_cache_keep_apart():
    """Two captured calls over one cache, replayed at once on two streams with new queries each time."""
    announce("kv two graphs")
    filled, _, _ = _filled(2, 4, 9000, 128, 4, seed=32)
    cache, lens = _gpu(filled), _lens([9000, 4500])
    qs = [_queries(2, 8, 1, 128, seed=s).to(DEV) for s in (0, 1)]
    kv.flash_attn_decode_mx(qs[0], *cache, lens)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in qs]
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(kv.flash_attn_decode_mx(q, *cache, lens))
    for r in range(4):
        for q, s in zip(qs, (2 * r, 2 * r + 1)):
            q.copy_(_queries(2, 8, 1, 128, seed=50 + s))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for q, out in zip(qs, outs):
            assert all(torch.equal(x, y) for x, y in zip(out, kv.flash_attn_decode_mx(q, *cache, lens))), r


@pytest.mark.parametrize("bits", [4, 8])
def test_moves_of_more_than_31_bits_of_elements(bits):
    """One call that writes, and one that reads, over 2^31 elements of K and of V: every 2^20th row and the last
    ones differ from the rest, in a batch of two."""
    announce(f"kv large calls bits={bits}")
    B, Hkv, D, T = 2, 1, 128, (1 << 23) + 77
    rows = torch.randn(2, D, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    k = rows[0].expand(B, Hkv, T, D)                      # strides 0: one row stands for all
    cache = kv.mx_cache(B, Hkv, T, D, bits)
    lens = _lens([T, T])
    kv.kv_cache_append(k, k, *cache, lens)
    odd = torch.arange(1 << 20, T, 1 << 20)
    for n in (*odd.tolist(), T):
        kv.kv_cache_append(rows[1].expand(B, Hkv, 1, D), rows[1].expand(B, Hkv, 1, D), *cache, _lens([n, n]))
    want = mx.values(*mx.quantise(rows.cpu(), bits), bits).to(BF).to(DEV)
    for x in kv.kv_cache_read(*cache, lens, T):
        assert x.numel() > 1 << 31
        one = torch.zeros(T, dtype=torch.bool, device=DEV)
        one[odd.to(DEV) - 1] = one[T - 1] = True
        for b in range(B):
            assert torch.equal((x[b, 0] == want[0]).all(-1), ~one) and torch.equal((x[b, 0] == want[1]).all(-1), one)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("ek, ev", [(110, 100), (-105, -100)])
def test_decode_of_scales_far_from_one(bits, ek, ev):
    """Keys scaled up or down by powers of two that the queries take back, values of 2^100 and 2^-100: the
    bits of the unscaled call, LSE and all, since only exponents differ."""
    announce(f"decode_mx exponents ek={ek} ev={ev} bits={bits}")
    B, Hq, Hkv, Tq, L, D = 2, 6, 2, 2, 1500, 128
    cache, k, v = _filled(B, Hkv, L, D, bits, seed=41)
    q = _queries(B, Hq, Tq, D)
    want = kv.flash_attn_decode_mx(q.to(DEV), *_gpu(cache), _lens([L, 70]))
    far = [t.clone() for t in cache]
    far[1] = (far[1].int() + ek).to(torch.uint8)
    far[3] = (far[3].int() + ev).to(torch.uint8)
    o, lse = kv.flash_attn_decode_mx((q.float() * 2.0**-ek).to(BF).to(DEV), *_gpu(far), _lens([L, 70]))
    assert torch.equal(lse, want[1]) and torch.equal(o.float(), want[0].float() * 2.0**ev)
    _check(q, cache, [L, 70], k, v, want, L)


# ------------------------------------------------------------------ lengths past the capacity

def _check_sharp(q, cache, lens, k, v, got, L):
    """_check where scores lie so far apart that weights underflow: a weight below 2^-126 of the row's largest
    is 0 or a subnormal of few bits in fp32, off by 2^-126 at most, so O misses up to 2^-126 |v| for each of L
    keys (which covers half a step, 2^-134, of O's own subnormals)."""
    o, lse, a, big = mx.decode(q, k, v, lens)
    tol_o, tol_lse = _bounds(o, a, big, _cut(q, k), L, q.shape[3])
    tol_o = tol_o + 2.0**-126 * L * v.abs().amax((2, 3)).repeat_interleave(q.shape[1] // k.shape[1], 1)[..., None, None]
    go, gl = (t.double().cpu() for t in got)
    assert torch.isfinite(lse).all() and ((gl - lse).abs() <= tol_lse).all(), ((gl - lse).abs() / tol_lse).max()
    assert ((go - o).abs() <= tol_o).all(), ((go - o).abs() / tol_o).max()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B, Hq, Hkv, Tq, L, D, over", [
    (4, 8, 2, 4, 64, 64, [1, 3, 4, 70]),                 # one launch, a whole number of blocks
    (3, 4, 2, 3, 97, 128, [1, 2, 2**31 - 1 - 97]),
    (2, 32, 4, 4, 333, 128, [2, 0]),                     # two tiles
    (3, 4, 4, 5, 5000, 128, [1, 4, 200]),                # several chunks
    (2, 3, 3, 6, 4992, 64, [5, 6]),
])
def test_queries_past_the_capacity_keep_their_positions(B, Hq, Hkv, Tq, L, D, over, bits):
    """Rows that no longer fit are not written, and every query still sees the keys up to its own position
    that the cache holds, its own among them."""
    announce(f"decode_mx past the capacity B={B} Tq={Tq} L={L} D={D} bits={bits} over={over}")
    want, _, _ = _filled(B, Hkv, L, D, bits, seed=51)
    cache, lens = _gpu(want), [L + n for n in over]
    g = torch.Generator().manual_seed(52)
    # keys far above the others, along the queries: a row that misses one is off by its whole weight
    q = _queries(B, Hq, Tq, D)
    k = (8 * q[:, ::Hq // Hkv].float()).to(BF)
    v = torch.randn(B, Hkv, Tq, D, generator=g).to(BF)
    kv.kv_cache_append(k.to(DEV), v.to(DEV), *cache, _lens(lens))
    mx.append(want, k, v, lens)
    assert all(torch.equal(a, b) for a, b in zip(_cpu(cache), want))
    got = kv.flash_attn_decode_mx(q.to(DEV), *cache, _lens(lens))
    _check_sharp(q, want, lens, *mx.read(want, [L] * B, L), got, L)


@pytest.mark.parametrize("L", [64, 333, 5000])
def test_nan_groups_past_the_capacity_reach_the_rows_that_see_them(L):
    """A NaN group of the cache's last V row, lengths one and two past the capacity: rows before it stay clean."""
    announce(f"decode_mx NaN past the capacity L={L}")
    B, Hq, Hkv, Tq, D = 2, 4, 2, 4, 64
    cache, _, _ = _filled(B, Hkv, L, D, 4, seed=53)
    q, lens = _queries(B, Hq, Tq, D).to(DEV), _lens([L + 1, L + 2])
    clean = kv.flash_attn_decode_mx(q, *_gpu(cache), lens)
    cache[3][:, :, L - 1, 1] = 255
    cache[2][:, :, L - 1, 16:] = 0
    o, lse = kv.flash_attn_decode_mx(q, *_gpu(cache), lens)
    bad = torch.zeros(B, Hq, Tq, D, dtype=torch.bool, device=DEV)
    bad[0, :, 2:, 32:] = bad[1, :, 1:, 32:] = True
    assert torch.equal(torch.isnan(o), bad) and torch.equal(lse, clean[1])
    assert torch.equal(o[~bad], clean[0][~bad])


# --------------------------------------------------------------------- queries next to zero

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [64, 128])
def test_queries_next_to_the_smallest_normal(D, bits):
    """Queries of 2^-124 against keys scaled up by as much: the bits of the same mantissas at size one."""
    announce(f"decode_mx queries of 2^-124 D={D} bits={bits}")
    B, Hq, Hkv, Tq, L, ek = 2, 6, 2, 2, 1500, 124
    cache, k, v = _filled(B, Hkv, L, D, bits, seed=54)
    tiny = (_queries(B, Hq, Tq, D).float() * 2.0**-ek).to(BF)
    q = (tiny.float() * 2.0**ek).to(BF)                  # exact: the subnormal ones have fewer bits
    far = [t.clone() for t in cache]
    far[1] = (far[1].int() + ek).to(torch.uint8)
    assert cache[1].int().max() + ek <= mx.LIMITS[bits][2] + 127 and (tiny.float().abs().amax(-1) >= 2.0**-126).all()
    want = kv.flash_attn_decode_mx(q.to(DEV), *_gpu(cache), _lens([L, 70]))
    got = kv.flash_attn_decode_mx(tiny.to(DEV), *_gpu(far), _lens([L, 70]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _check(q, cache, [L, 70], k, v, want, L)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq, Hkv, L, D", [(6, 1, 700, 64), (6, 1, 700, 128), (24, 1, 2000, 128)])
def test_queries_of_few_bits_left(Hq, Hkv, L, D, bits):
    """Rows whose elements all have one magnitude, from 2^-108 down to subnormals, over keys of up to 2^126
    along their signs: an error of the query's terms adds up over the row."""
    announce(f"decode_mx tiny queries Hq={Hq} L={L} D={D} bits={bits}")
    g = torch.Generator().manual_seed(55)
    sign = torch.randint(0, 2, (D,), generator=g) * 2 - 1
    size = torch.tensor([1.2109375 * 2.0**-124, 113 * 2.0**-133, 1.9921875 * 2.0**-117, 1.1484375 * 2.0**-120,
                         1.6796875 * 2.0**-126, 1.2109375 * 2.0**-109], dtype=torch.float64).repeat(Hq // 6)
    q = (size[:, None] * sign).view(1, Hq, 1, D).to(BF)
    assert torch.equal(q.double(), (size[:, None] * sign).view(1, Hq, 1, D))
    ramp = torch.linspace(0.1, 1, L).double()[:, None] * 2.0**126 * sign * (1 + 0.1 * torch.rand(D, generator=g))
    v = torch.randn(1, Hkv, L, D, generator=g).to(BF)
    cache = [*mx.quantise(ramp.view(1, 1, L, D).to(BF), bits), *mx.quantise(v, bits)]
    got = kv.flash_attn_decode_mx(q.to(DEV), *_gpu(cache), _lens([L]))
    _check_sharp(q, cache, [L], mx.values(*cache[:2], bits), mx.values(*cache[2:], bits), got, L)


# ---------------------------------------------------------------------------- large reads

@pytest.mark.parametrize("D, B, Hkv, T", [(128, 3, 5, 4369), (128, 3, 5, 4370), (64, 2, 7, 9362), (64, 2, 7, 9363),
                                          (128, 3, 5, 8738), (128, 3, 5, 8739)])
def test_large_reads_of_8_bits_in_fp32(D, B, Hkv, T):
    """Sizes around 2^21 lanes of four elements and around 2^24 elements, with a last workgroup that is part
    empty."""
    announce(f"kv large fp32 reads D={D} B={B} Hkv={Hkv} T={T}")
    codes = torch.randint(0, 256, (B, Hkv, T, D), dtype=torch.uint8, generator=torch.Generator().manual_seed(T))
    codes[(codes & 127) == 127] = 0
    scales = (120 + codes[..., ::32] % 15).to(torch.uint8)
    k, v = kv.kv_cache_read(*_gpu([codes, scales, codes ^ 0x80, scales]), _lens([T] * B), T, F32)
    assert torch.equal(k.cpu(), mx.values(codes, scales, 8).float()) and torch.equal(v, -k)


# ------------------------------------------------------------------------- fp32 roundings

@pytest.mark.parametrize("bits", [4, 8])
def test_append_of_fp32_values_next_to_every_border(bits):
    """The borders between neighbouring values of the type, under every power of two that a group may
    have, with the fp32 values just below and above them; and groups whose largest magnitude lies just below,
    at and above the border between two powers."""
    announce(f"kv append fp32 borders bits={bits}")
    top, lo, hi = mx.LIMITS[bits]
    v, inf = mx.magnitudes(bits), torch.tensor(math.inf)
    unit = torch.exp2(torch.arange(lo, hi + 1).double())[:, None]

    def near(x):
        x32 = x.float()
        assert torch.equal(x32.double(), x)
        return torch.stack([torch.nextafter(x32, -inf), x32, torch.nextafter(x32, inf)], -1)

    mids = near((v[1:] + v[:-1]) / 2 * unit).flatten(1)                                  # [powers, 3 borders]
    mids = torch.nn.functional.pad(mids, (0, -mids.shape[1] % 31)).unflatten(1, (-1, 31))
    largest = (v[-1] * unit).float()[:, None].expand(-1, mids.shape[1], 1)               # fixes the power
    groups = torch.cat([largest, mids], -1).flatten(0, 1)
    assert mx.quantise(groups, bits)[1].view(-1, mids.shape[1])[:, 0].tolist() == list(range(lo + 127, hi + 128))
    g = torch.Generator().manual_seed(56)
    tops = near(top * unit).flatten()[:, None]
    groups = torch.cat([groups, torch.cat([tops, tops * torch.rand(len(tops), 31, generator=g)], -1)])
    groups = groups * (torch.randint(0, 2, groups.shape, generator=g) * 2 - 1)
    groups = torch.nn.functional.pad(groups, (0, 0, 0, len(groups) % 2))
    k = groups.view(1, 1, -1, 64)
    T = k.shape[2]
    got = _gpu(kv.mx_cache(1, 1, T, 64, bits, device="cpu"))
    kv.kv_cache_append(k.to(DEV), -k.to(DEV), *got, _lens([T]))
    for a, b in zip(_cpu(got), (*mx.quantise(k, bits), *mx.quantise(-k, bits))):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------ transforms

def test_function_transforms():
    """Under vmap attention and reads are loops of their calls; what has no rule (writing a cache under vmap,
    tangents of recorded inputs) raises."""
    import torch.autograd.forward_ad as fw

    announce("kv transforms")
    filled, _, _ = _filled(2, 2, 90, 64, 8, seed=57)
    cache, lens = _gpu(filled), _lens([90, 40])
    qs = torch.stack([_queries(2, 4, 1, 64, seed=s) for s in (0, 1, 2)]).to(DEV)
    ks = torch.stack([_queries(2, 2, 1, 64, seed=s) for s in (3, 4)]).to(DEV)
    got = torch.vmap(lambda q: kv.flash_attn_decode_mx(q, *cache, lens))(qs)
    for i, q in enumerate(qs):
        assert all(torch.equal(x[i], y) for x, y in zip(got, kv.flash_attn_decode_mx(q, *cache, lens)))
    many = torch.stack([lens, lens - 30])
    got = torch.vmap(lambda n: kv.kv_cache_read(*cache, n, 9, F32))(many)
    for i, n in enumerate(many):
        assert all(torch.equal(x[i], y) for x, y in zip(got, kv.kv_cache_read(*cache, n, 9, F32)))
    with pytest.raises(RuntimeError, match="[Bb]atching rule"):
        torch.vmap(lambda k: kv.kv_cache_append(k, k, *cache, lens))(ks)
    assert all(torch.equal(a, b) for a, b in zip(_cpu(cache), filled))
    want = kv.flash_attn_decode_mx(qs[0], *cache, lens)
    with fw.dual_level():
        got = kv.flash_attn_decode_mx(fw.make_dual(qs[0], torch.ones_like(qs[0])), *cache, lens)
        assert all(torch.equal(fw.unpack_dual(x).primal, y) for x, y in zip(got, want))
        with pytest.raises(NotImplementedError, match="forward mode AD"):
            kv.flash_attn_decode_mx(fw.make_dual(qs[0].clone().requires_grad_(), torch.ones_like(qs[0])), *cache, lens)
