"""The quantised KV cache in 64 bits (test infrastructure only): its format, the rows that an append
writes and a read gives, and attention over the values that a cache stands for.

Written from the definition: the shared exponent e is the smallest integer with
max |x| <= top * 2^e, an element the nearest of the type's values, ties to the even code.
"""

from __future__ import annotations

import math

import torch

GROUP = 32
#: bits -> (largest value plus half of its last step, smallest and largest e)
LIMITS = {4: (7.0, -125, 125), 8: (464.0, -117, 119)}


def magnitudes(bits: int) -> torch.Tensor:
    """The type's magnitudes in the order of their codes: e2m1 (4 bits) or e4m3 (8)."""
    if bits == 4:
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    sub = [m * 2.0**-9 for m in range(8)]
    return torch.tensor(sub + [(8 + m) * 2.0**(e - 10) for e in range(1, 16) for m in range(8)][:-1],
                        dtype=torch.float64)


def quantise(x: torch.Tensor, bits: int):
    """(codes uint8 [..., D * bits / 8], scales uint8 [..., D / 32]) of x [..., D]."""
    top, lo, hi = LIMITS[bits]
    g = x.double().unflatten(-1, (-1, GROUP))
    a = g.abs().amax(-1)
    nan = ~torch.isfinite(g).all(-1)
    m, k = torch.frexp(torch.where(nan, 1.0, a) / top)
    e = torch.where(m == 0.5, k - 1, k)
    e = torch.where(a == 0, lo, e).clamp(lo, hi)
    y = torch.where(nan[..., None], 0.0, g) * torch.exp2(-e.double())[..., None]
    v = magnitudes(bits)
    mid = (v[1:] + v[:-1]) / 2
    c = torch.searchsorted(mid, y.abs())
    tie = (c < len(mid)) & (y.abs() == mid[c.clamp(max=len(mid) - 1)]) & (c % 2 == 1)
    c = (c + tie) | (torch.signbit(y).long() << (bits - 1))
    c = torch.where(nan[..., None], 0, c).flatten(-2)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    return c.to(torch.uint8), torch.where(nan, 255, e + 127).to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """fp64 values [..., D] of codes and scales; NaN for the scale 255."""
    c = codes.long()
    if bits == 4:
        c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    sign = 1 << (bits - 1)
    v = torch.cat([magnitudes(bits), torch.full((1,), math.nan, dtype=torch.float64)])[c & (sign - 1)]
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, math.nan, s).repeat_interleave(GROUP, -1)
    return torch.where(c >= sign, -v, v) * s


def append(cache, k, v, cache_seqlens) -> None:
    """The rows that ``kv_cache_append`` writes, in place (CPU tensors)."""
    T, L, bits = k.shape[2], cache[0].shape[2], 8 * cache[0].shape[3] // k.shape[3]
    for b, n in enumerate(cache_seqlens):
        for t in range(T):
            pos = n - T + t
            if 0 <= pos < L:
                cache[0][b, :, pos], cache[1][b, :, pos] = quantise(k[b, :, t], bits)
                cache[2][b, :, pos], cache[3][b, :, pos] = quantise(v[b, :, t], bits)


def read(cache, cache_seqlens, rows):
    """The fp64 rows that ``kv_cache_read`` gives."""
    D, L = GROUP * cache[1].shape[3], cache[0].shape[2]
    bits, out = 8 * cache[0].shape[3] // D, []
    for codes, scales in (cache[:2], cache[2:]):
        x = torch.zeros(*codes.shape[:2], rows, D, dtype=torch.float64)
        for b, n in enumerate(cache_seqlens):
            lo, hi = max(n - rows, 0), min(n, L)
            if lo < hi:
                x[b, :, lo - n + rows:hi - n + rows] = values(codes[b, :, lo:hi], scales[b, :, lo:hi], bits)
        out.append(x)
    return tuple(out)


def decode(q, k, v, cache_seqlens):
    """Attention of the newest rows q [B, Hq, Tq, D] over fp64 values k, v [B, Hkv, L, D], each row over the
    keys it sees and no others (a NaN elsewhere does not matter): row i sits at position
    cache_seqlens[b] - Tq + i and sees those up to it that the cache holds.

    Returns (O, LSE, A, S): A = sum p |v| and S = the row's largest sum |q_d k_d| / sqrt(D), the sizes
    that rounding errors of O and of the scores go by."""
    B, Hq, Tq, D = q.shape
    Hkv, Lmax = k.shape[1:3]
    G, dev = Hq // Hkv, q.device
    o, a = (torch.zeros(B, Hq, Tq, D, dtype=torch.float64, device=dev) for _ in range(2))
    lse = torch.full((B, Hq, Tq), -math.inf, dtype=torch.float64, device=dev)
    big = torch.zeros(B, Hq, Tq, dtype=torch.float64, device=dev)
    for b in range(B):
        for i in range(Tq):
            n = min(int(cache_seqlens[b]) - Tq + i + 1, Lmax)
            if n < 1:
                continue
            x = q[b, :, i].double().view(Hkv, G, D)
            kk, vv = k[b, :, :n].double(), v[b, :, :n].double()
            s = x @ kk.transpose(1, 2) / math.sqrt(D)
            lse[b, :, i] = torch.logsumexp(s, -1).flatten()
            p = torch.softmax(s, -1)
            o[b, :, i], a[b, :, i] = (p @ vv).view(Hq, D), (p @ vv.abs()).view(Hq, D)
            big[b, :, i] = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1).flatten() / math.sqrt(D)
    return o, lse, a, big
