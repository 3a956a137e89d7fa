"""64-bit restatements of the block's operators (RMSNorm with the residual, gated feed-forward, products with
quantised weights) with the sizes that rounding errors of their results go by."""

from __future__ import annotations

import torch

from . import mx_cache


def add_rms_norm(x, residual, weight, eps):
    """(y fp64, h): h in residual's type, as fp32 sums round to it; y from that h."""
    h = x if residual is None else (residual.float() + x.float()).to(residual.dtype)
    z = h.double()
    return z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * weight.double(), h


def add_rms_norm_grads(dy, dh, h, weight, eps):
    """(d, size of d's terms, dw, size of dw's terms), fp64."""
    z, g = h.double(), dy.double() * weight.double()
    s = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
    dh = torch.zeros_like(z) if dh is None else dh.double()
    d = dh + s * g - z * s**3 * (z * g).mean(-1, keepdim=True)
    size = dh.abs() + s * g.abs() + z.abs() * s**3 * (z * g).abs().mean(-1, keepdim=True)
    t = (dy.double() * z * s).reshape(-1, z.shape[-1])
    return d, size, t.sum(0), t.abs().sum(0)


def swiglu(x, wg, wu):
    """(a, bound of |da| per unit of relative error in the two products), fp64."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    gs, us = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()
    silu = g * torch.sigmoid(g)
    return silu * u, 1.1 * gs * u.abs() + silu.abs() * us  # |silu'| < 1.1


def swiglu_grads(da, x, wg, wu):
    """{name: (gradient, sum of its terms' magnitudes, sum of its terms' errors per unit of error in g and u)}."""
    x, wg, wu, da = x.double(), wg.double(), wu.double(), da.double()
    g, u = x @ wg.t(), x @ wu.t()
    gs, us = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()
    p = torch.sigmoid(g)
    slope = p * (1 + g * (1 - p))
    dg, du = da * u * slope, da * g * p
    # |silu''| <= 1/2; what an error in g, u (per unit of gs, us) does to dg and du
    eg = da.abs() * (us * slope.abs() + u.abs() * 0.5 * gs)
    eu = da.abs() * 1.1 * gs
    both = {"dx": (dg @ wg + du @ wu, dg.abs() @ wg.abs() + du.abs() @ wu.abs(), eg @ wg.abs() + eu @ wu.abs()),
            "dw_gate": (dg.t() @ x, dg.abs().t() @ x.abs(), eg.t() @ x.abs()),
            "dw_up": (du.t() @ x, du.abs().t() @ x.abs(), eu.t() @ x.abs())}
    return both


def linear_mx(x, x_scales, codes, scales):
    """(y, sum of the products' magnitudes, sum over every eight consecutive products of the largest one), fp64 on
    the CPU, from the values that the bytes stand for."""
    K = 32 * scales.shape[1]
    w = mx_cache.values(codes.cpu(), scales.cpu(), 8 * codes.shape[1] // K)
    x = x.cpu().double() if x_scales is None else mx_cache.values(x.cpu(), x_scales.cpu(), 8)
    top = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64)
    for k in range(0, K, 8):
        top += (x[:, None, k:k + 8] * w[None, :, k:k + 8]).abs().amax(-1)
    return x @ w.t(), x.abs() @ w.abs().t(), top
