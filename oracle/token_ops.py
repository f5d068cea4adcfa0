"""The token operators from their definitions, in 64 bits, with the error that a kernel of 32-bit
sums and one rounding per stored value may show.

Each function returns (value, bound) pairs: |kernel - value| <= bound elementwise.  The bounds count
roundings: a store rounds by at most half a step (eps / 2 relative, or half the smallest subnormal),
an fp32 operation by 2^-24, and the matrix cores' accumulation of 16-bit operands by at most 2^-23 a
term.  Their sums of 8-bit products, used for 16-bit outputs only, keep fewer bits: they are off by up
to 2^-12 of the sum of the magnitudes.
"""
from __future__ import annotations

import math

import torch

U = 2.0**-24


def half_step(value: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    f = torch.finfo(dtype)
    return torch.clamp(value.abs() * (f.eps / 2), min=f.smallest_normal * f.eps / 2)


def rms_norm(x, weight, residual, eps):
    """s, y and their bounds, both for a store in x's type and before it (fp32)."""
    s = x.double() + (residual.double() if residual is not None else 0)
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    # a row's sum of squares: a chain of at most 64 terms a lane, then a tree of 10 levels and 16
    # partial sums, each rounding by U, halved by the square root; six more operations form y
    rel = (90 / 2 + 8) * U
    return s, half_step(s, x.dtype) + s.abs() * 2 * U, y, y.abs() * rel


def e4m3_scale(y):
    """c = max |y| / 448 per row, 1 for rows of zeros."""
    c = y.abs().amax(-1) / 448
    return torch.where(c == 0, torch.ones_like(c), c)


def activation(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def linear(x, w, bias, act, residual, xs, ws, out_dtype):
    """(value, bound) of act(xs ws x w^T + bias) + residual."""
    K = x.shape[-1]
    codes = x.dtype == torch.float8_e4m3fn
    x, w = x.double(), w.double()
    if xs is not None:
        x = x * xs.double()[..., None]
    if ws is not None:
        w = w * ws.double()[:, None]
    z = x @ w.t()
    hw8 = 2.0**-12 if codes and out_dtype != torch.float32 else 0
    err = ((K * 2 + 4) * U + hw8) * (x.abs() @ w.t().abs())
    if bias is not None:
        z = z + bias.double()
    err = err + z.abs() * U
    y = activation(z, act)
    # no activation's slope passes 1.13; their exponential, erf and division are off by a few units
    # relative to |z| (each is |z| times a value in 0..1)
    err = 1.13 * err + z.abs() * 16 * U
    if residual is not None:
        y = y + residual.double()
    return y, err + y.abs() * U + half_step(y, out_dtype)


def cross_attention(q, k, v, scale=None, key_lengths=None, key_mask=None):
    """(value, bound): keys that do not count are taken out before anything is computed from them."""
    B, Lq, Hq, d = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    f = torch.finfo(q.dtype)
    for b in range(B):
        n = Lk if key_lengths is None else max(0, min(Lk, int(key_lengths[b])))
        at = torch.arange(n, device=q.device)
        if key_mask is not None:
            at = at[key_mask[b, :n]]
        if len(at) == 0:
            continue
        for h in range(Hq):
            g = h // (Hq // Hkv)
            kk, vv, qq = k[b, at, g].double(), v[b, at, g].double(), q[b, :, h].double()
            s = qq @ kk.t() * scale
            p = torch.softmax(s, -1)
            o = p @ vv
            # the scores' error (d terms, the product with the scale, the difference to the maximum),
            # which p takes on relatively; the rounding of p to the operands' type; the sums over the keys
            ds = ((2 * d + 8) * U * (qq.abs() @ kk.t().abs()) * abs(scale)).amax(-1, keepdim=True) + s.abs().amax(
                -1, keepdim=True) * 8 * U
            rel = f.eps / 2 + 4 * ds + (4 * len(at) + 64) * U
            tiny = f.smallest_normal * f.eps / 2 * len(at) * vv.abs().amax() if q.dtype == torch.float16 else 0
            out[b, :, h] = o
            bound[b, :, h] = rel * (p @ vv.abs()) + tiny
    return out, bound + half_step(out, q.dtype)
