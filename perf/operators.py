"""Performance cases of the quantised KV cache: writing rows, reading them back, attending over it.

Every case is a dict of plain values; ``kind`` names what a pass does:

* ``append`` -- ``kv_cache_append`` of new K/V rows, then ``kv_cache_read`` of the same rows: what a
  program does whose prompt attention runs over the values that later steps will see
* ``read``   -- ``kv_cache_read`` of a part or the whole of a cache
* ``decode`` -- ``flash_attn_decode_mx``: new query rows against the cache

A cache row holds ``D`` elements in groups of 32 that share a power of two: e2m1 elements (``bits``
4, two to a byte, the lower dimension in the low nibble) or e4m3 elements (``bits`` 8), and one byte
``e + 127`` per group.  With ``own`` false a pass computes this in plain tensor operations.

K is unit-RMS per head with uneven channels (what a k norm with its weight produces), V ~ N(0, 1).
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6
_GROUP = 32
#: bits -> (largest magnitude, as a fraction of a power of two 2^x, that 2^(x - shift) may scale; shift; bounds of e)
_RULES = {4: (0.875, 3, -125, 125), 8: (0.90625, 9, -117, 119)}


# ------------------------------------------------------------------------------- cases

def _rows(name, kind, B, Hkv, T, L, D, bits, dtype="bf16", least=1.0, mix=0):
    return {"name": name, "kind": kind, "B": B, "Hkv": Hkv, "T": T, "L": L, "D": D, "bits": bits,
            "dtype": dtype, "least": least, "mix": mix}


def _decode(name, B, Hq, Hkv, Tq, L, D, bits, least, mix):
    return {"name": name, "kind": "decode", "B": B, "Hq": Hq, "Hkv": Hkv, "Tq": Tq, "L": L, "D": D,
            "bits": bits, "least": least, "mix": mix}


def listed():
    return [
        # The write of every generated token of a serving batch, each at its own position.
        _rows("append_token", "append", 32, 8, 1, 4096, 128, 4, least=0.1, mix=1),
        # One prompt of an fp32 debugging run, 112M model heads, ragged length, 8 bits.
        _rows("append_prompt_fp32", "append", 1, 2, 777, 1024, 128, 8, "fp32"),
        # A batch of left-padded prompts of uneven lengths.
        _rows("append_prompts", "append", 16, 8, 4000, 4096, 128, 4, least=0.3, mix=2),
        # A cached prefix handed to a long continuation.
        _rows("read_prefix", "read", 1, 8, 16384, 16384, 128, 4),
        # The recent rows of every sequence of a batch of the multi-head 112M shape.
        _rows("read_recent", "read", 32, 12, 1000, 2048, 64, 8, least=0.5, mix=3),
        # Interactive generation with the 112M model: one short cache.
        _decode("decode_single", 1, 8, 2, 1, 512, 128, 4, 0.5, 4),
        # One user's very long context.
        _decode("decode_long", 1, 16, 8, 1, 131072, 128, 4, 1.0, 5),
        # A serving batch, every request at its own position.
        _decode("decode_batch", 32, 16, 8, 1, 4096, 128, 4, 0.1, 6),
        # The same held in 8 bits.
        _decode("decode_batch_8bit", 32, 16, 8, 1, 4096, 128, 8, 0.1, 6),
        # The multi-head 112M shape, odd capacity.
        _decode("decode_mha", 64, 12, 12, 1, 2001, 64, 4, 0.1, 7),
        # Several new rows per sequence (drafted tokens checked at once), wide groups.
        _decode("decode_rows", 16, 32, 4, 4, 5000, 128, 4, 0.2, 8),
        # Large-batch serving of long contexts: the largest case.
        _decode("decode_large", 64, 16, 8, 1, 16384, 128, 4, 0.3, 9),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = {64: [(12, 12), (12, 4), (4, 4), (8, 2)], 128: [(16, 8), (8, 2), (8, 8), (32, 4), (6, 2)]}


def draw(rng: random.Random):
    kind = rng.choice(["append", "append", "read", "decode", "decode", "decode"])
    D, bits = rng.choice([64, 128]), rng.choice([4, 4, 8])
    Hq, Hkv = rng.choice(_HEADS[D])
    least, mix = rng.choice([0.1, 0.5, 1.0]), rng.randrange(1 << 20)
    B = _log(rng, 1, 64)
    if kind == "decode":
        L = min(_log(rng, 100, 131072), 262144 // B)  # the caches of a batch share the memory
        Tq = rng.choice([1, 1, 1, 2, 3, 4])
        return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "Tq": Tq, "L": L, "D": D, "bits": bits,
                "least": least, "mix": mix}
    T = min(_log(rng, 1, 16384), 32768 // B)
    return {"kind": kind, "B": B, "Hkv": Hkv, "T": T, "L": T + _log(rng, 1, 2048), "D": D,
            "bits": bits, "dtype": rng.choice(["bf16", "bf16", "fp32"]), "least": least, "mix": mix}


# ------------------------------------------------------------------------------ inputs

def _lengths(case):
    """Keys of every sequence, the new rows among them, from the case alone."""
    r = random.Random(case["mix"])
    if case["kind"] == "decode":
        lo = max(case["Tq"], int(case["least"] * case["L"]))
        return [r.randint(lo, case["L"]) for _ in range(case["B"])]
    if case["kind"] == "append" and case["T"] > 1:  # prompts: padded on the left to T rows
        return [r.randint(max(1, int(case["least"] * case["T"])), case["T"]) for _ in range(case["B"])]
    return [r.randint(max(1, int(case["least"] * case["L"])), case["L"]) for _ in range(case["B"])]


def _unit_rms(x):
    return x * torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + _EPS)


def _draws(seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device="cuda")


def _cache(rand, case, channels):
    """(k_codes, k_scales, v_codes, v_scales) of a cache filled to its capacity."""
    B, Hkv, L, D, bits = (case[n] for n in ("B", "Hkv", "L", "D", "bits"))
    out = [torch.empty(B, Hkv, L, n, dtype=torch.uint8, device="cuda")
           for n in (D * bits // 8, D // _GROUP) * 2]
    for b in range(B):
        for i, x in enumerate((_unit_rms(rand(Hkv, L, D)) * channels, rand(Hkv, L, D))):
            out[2 * i][b], out[2 * i + 1][b] = _quantise(x.to(torch.bfloat16), bits)
    return out


def prepare(case, seed):
    rand, B, Hkv, D = _draws(seed), case["B"], case["Hkv"], case["D"]
    s = {"kind": case["kind"], "bits": case["bits"],
         "lens": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")}
    channels = 1.0 + 0.2 * rand(D)
    if case["kind"] == "decode":
        s["cache"] = _cache(rand, case, channels)
        s["q"] = _unit_rms(rand(B, case["Hq"], case["Tq"], D)).to(torch.bfloat16)
        return s
    s["dtype"], s["rows"] = _DTYPES[case["dtype"]], case["T"]
    if case["kind"] == "read":
        s["cache"] = _cache(rand, case, channels)
        return s
    L, n = case["L"], D * case["bits"] // 8
    s["cache"] = [torch.zeros(B, Hkv, L, m, dtype=torch.uint8, device="cuda")
                  for m in (n, D // _GROUP, n, D // _GROUP)]
    s["k"] = (_unit_rms(rand(B, Hkv, case["T"], D)) * channels).to(s["dtype"])
    s["v"] = rand(B, Hkv, case["T"], D).to(s["dtype"])
    return s


# --------------------------------------------------------------------------- plain form

def _quantise(x, bits):
    """x [..., D] -> (codes uint8 [..., D * bits / 8], scales uint8 [..., D / 32])."""
    g = x.float().unflatten(-1, (-1, _GROUP))
    frac, shift, lo, hi = _RULES[bits]
    f, p = torch.frexp(g.abs().amax(dim=-1, keepdim=True))
    e = torch.where(f > frac, p - shift + 1, p - shift)
    e = torch.where(f == 0, torch.full_like(e, lo), e).clamp(lo, hi)
    y = g * torch.exp2(-e.float())
    a = y.abs()
    if bits == 4:
        c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
             + (a >= 3.5) + (a > 5))
    else:
        p = torch.frexp(a.clamp(min=2.0**-7))[1] - 1            # a is in 2^p .. 2^(p + 1),
        p = p.clamp(-6, 8)                                      # or below 2^-6
        c = ((p + 6) * 8 + torch.round(a * torch.exp2(3.0 - p.float())).int()).clamp(max=126)
        c = c.to(torch.uint8)
    c = torch.where(torch.signbit(y), c + (1 << (bits - 1)), c).flatten(-2)
    if bits == 4:
        c = c[..., 0::2] + c[..., 1::2] * 16
    return c, (e + 127).squeeze(-1).to(torch.uint8)


def _values(bits, device):
    """The value of every code."""
    c = torch.arange(1 << bits, device=device)
    m = 1 if bits == 4 else 3                                   # mantissa bits
    a, sign = c & ((1 << (bits - 1)) - 1), c >> (bits - 1)
    p, frac = a >> m, a & ((1 << m) - 1)
    bias = 1 if bits == 4 else 7
    v = (frac + torch.where(p > 0, 1 << m, 0)) * torch.exp2((p.clamp(min=1) - bias - m).float())
    return torch.where(sign > 0, -v, v)


def _dequantise(codes, scales, bits):
    """fp32 values [..., D] of codes [..., D * bits / 8] and scales [..., D / 32]."""
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    v = _values(bits, codes.device).index_select(0, codes.reshape(-1).int()).view(codes.shape)
    v = v.unflatten(-1, (-1, _GROUP)) * torch.exp2(scales.float() - 127.0).unsqueeze(-1)
    return v.flatten(-2)


def _window(s):
    """(batch index [B, 1], position [B, rows] of every row, whether it is in the cache)."""
    B, L = s["cache"][0].shape[0], s["cache"][0].shape[2]
    lens = s["lens"].long()[:, None]
    pos = lens - s["rows"] + torch.arange(s["rows"], device=lens.device)
    return torch.arange(B, device=lens.device)[:, None], pos, (pos >= 0) & (pos < L)


def _append_plain(s):
    batch, pos, _ = _window(s)
    at = pos.clamp(min=0)                   # a padding row is written as the first real one is
    i = at - pos[:, :1]
    for x, codes, scales in ((s["k"], *s["cache"][:2]), (s["v"], *s["cache"][2:])):
        new = _quantise(x.transpose(1, 2)[batch, i], s["bits"])  # [B, rows, Hkv, ...]
        codes.transpose(1, 2)[batch, at], scales.transpose(1, 2)[batch, at] = new


def _read_plain(s):
    batch, pos, inside = _window(s)
    at, out = pos.clamp(0, s["cache"][0].shape[2] - 1), []
    for codes, scales in (s["cache"][:2], s["cache"][2:]):
        x = _dequantise(codes.transpose(1, 2)[batch, at], scales.transpose(1, 2)[batch, at], s["bits"])
        x = x.masked_fill(~inside[:, :, None, None], 0.0).transpose(1, 2)
        out.append(x.to(s["dtype"]).contiguous())
    return tuple(out)


def _decode_plain(s):
    q, lens = s["q"].float(), s["lens"].long()
    B, Hq, Tq, D = q.shape
    Hkv, L = s["cache"][0].shape[1:3]
    k, v = (_dequantise(c, e, s["bits"]) for c, e in (s["cache"][:2], s["cache"][2:]))
    x = torch.matmul(q.view(B, Hkv, -1, D), k.transpose(2, 3)).view(B, Hq, Tq, L) / math.sqrt(D)
    last = lens[:, None] - Tq + torch.arange(Tq, device=q.device)             # [B, Tq]
    seen = torch.arange(L, device=q.device) <= last[:, :, None]               # [B, Tq, L]
    x = x.masked_fill(~seen[:, None], -math.inf)
    m = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - m)
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul((p / total).view(B, Hkv, -1, L), v).view(B, Hq, Tq, D)
    return o.to(s["q"].dtype), (m + torch.log(total)).squeeze(-1)


# -------------------------------------------------------------------------------- pass

def run(state):
    s = state
    if own:
        from tinytrain_amd.kernels.kv_cache import flash_attn_decode_mx, kv_cache_append, kv_cache_read

        if s["kind"] == "decode":
            return flash_attn_decode_mx(s["q"], *s["cache"], s["lens"])
        if s["kind"] == "append":
            kv_cache_append(s["k"], s["v"], *s["cache"], s["lens"])
        return kv_cache_read(*s["cache"], s["lens"], s["rows"], s["dtype"])
    if s["kind"] == "decode":
        return _decode_plain(s)
    if s["kind"] == "append":
        _append_plain(s)
    return _read_plain(s)


# -------------------------------------------------------------------------------- work

def work(case):
    Hkv, D = case["Hkv"], case["D"]
    row = D * case["bits"] // 8 + D // _GROUP                                  # a K or V row as held
    if case["kind"] == "decode":
        keys, rows = sum(_lengths(case)), case["B"] * case["Hq"] * case["Tq"]
        return {"bytes": 2 * keys * Hkv * row + rows * (4 * D + 4),
                "flops": 4 * D * case["Hq"] * case["Tq"] * keys}
    size = _DTYPES[case["dtype"]].itemsize
    held = sum(min(n, case["T"]) for n in _lengths(case)) * Hkv                 # rows inside the cache
    dense = case["B"] * case["T"] * Hkv * D * size
    if case["kind"] == "read":
        return {"bytes": 2 * (held * row + dense), "flops": 2 * 2 * held * D}
    return {"bytes": 2 * (held * D * size + held * row + dense), "flops": 2 * 6 * held * D}


# ------------------------------------------------------------------------ 64-bit results

def _rounded(x, bits):
    """What x [..., D] (fp64) reads back as: the definition, by logarithms and nearest values."""
    g = x.unflatten(-1, (-1, _GROUP))
    top, (_, _, lo, hi) = {4: 7.0, 8: 464.0}[bits], _RULES[bits]
    e = torch.ceil(torch.log2(g.abs().amax(-1, keepdim=True) / top)).clamp(lo, hi)
    y = g * torch.exp2(-e)
    if bits == 4:
        best, at = torch.full_like(y, math.inf), torch.zeros_like(y)
        for v in (0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):       # those of even codes win ties
            off = (y.abs() - v).abs()
            at = torch.where(off < best, v, at)
            best = torch.minimum(best, off)
    else:
        step = torch.exp2(torch.floor(torch.log2(y.abs())).clamp(min=-6) - 3)
        at = (torch.round(y.abs() / step) * step).clamp(max=448.0)
    return (torch.copysign(at, y) * torch.exp2(e)).flatten(-2)


def _held(codes, scales, bits):
    """fp64 values of cache rows, element by element from the bits."""
    if bits == 4:
        c = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.uint8, device=codes.device)
        c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
        mag = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=c.device)[(c % 8).long()]
        v = torch.where(c >= 8, -mag, mag)
    else:
        v = codes.view(torch.float8_e4m3fn).double()
    return v * torch.exp2(scales.double() - 127).repeat_interleave(_GROUP, dim=-1)


def exact(case, seed):
    s, lens = prepare(case, seed), _lengths(case)
    if case["kind"] == "decode":
        q = s["q"].double()
        B, Hq, Tq, D = q.shape
        Hkv = case["Hkv"]
        o, lse = torch.empty_like(q), torch.empty(B, Hq, Tq, dtype=torch.float64, device=q.device)
        for b, n in enumerate(lens):
            k, v = (_held(s["cache"][i][b, :, :n], s["cache"][i + 1][b, :, :n], case["bits"]) for i in (0, 2))
            late = torch.arange(n, device=q.device) > n - Tq + torch.arange(Tq, device=q.device)[:, None]
            for h in range(Hkv):
                rows = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                x = (q[b, rows].reshape(-1, D) @ k[h].t()).view(-1, Tq, n) / math.sqrt(D)
                x = x.masked_fill(late, -math.inf)
                lse[b, rows] = torch.logsumexp(x, -1)
                o[b, rows] = torch.softmax(x, -1) @ v[h]
        return o, lse
    out = []
    for i, name in ((0, "k"), (2, "v")):
        full = torch.zeros(case["B"], case["Hkv"], case["T"], case["D"], dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            m = min(n, case["T"])
            if case["kind"] == "append":
                full[b, :, -m:] = _rounded(s[name][b, :, -m:].double(), case["bits"])
            else:
                full[b, :, -m:] = _held(*(t[b, :, n - m:n] for t in s["cache"][i:i + 2]), case["bits"])
        out.append(full)
    return tuple(out)
