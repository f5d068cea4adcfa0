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


def rotary(x, positions, frequencies, sections, interleaved):
    """(value, bound) of the first 2 P values of each head of x (B, L, heads, d) turned, the rest as it is."""
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    angle = positions.double()[..., axis] * frequencies.double()  # (B, L, P) or (L, P)
    cos, sin = torch.cos(angle)[..., None, :], torch.sin(angle)[..., None, :]
    n = len(axis)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y, err = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    x0, x1 = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    # the reduced angle is an fp32 number of half turns up to 1 (off by 2^-25, pi times that in radians), formed in 64
    # bits from a few roundings relative to the whole angle; sine and cosine are off by two units more, the products
    # and their sum round three times
    rel = math.pi * 2.0**-25 + 4 * U + angle.abs()[..., None, :] * 2.0**-50 + 3 * U
    err[..., a] = err[..., b] = (x0.abs() + x1.abs()) * rel
    # what is not turned is stored as it was
    bound = err + torch.where(err > 0, half_step(y, x.dtype), 0.0)
    return y, bound


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def e2m1_weight(weight, group_scale, K):
    """The (N, K) values, in 64 bits, of e2m1 codes two a byte and the e4m3 scales of their groups."""
    codes = torch.stack([weight & 15, weight >> 4], -1).flatten(1).long()
    group = next(g for g in (32, 64, 128) if -(-K // g) == group_scale.shape[1])
    values = torch.tensor(E2M1, dtype=torch.float64, device=weight.device)[codes]
    return values * torch.repeat_interleave(group_scale.double(), group, 1)[:, :K]


def linear_e2m1(x, weight, group_scale, row_scale, bias, act, residual, out_dtype):
    """(value, bound): the products of codes and scales are exact, so the linear operator's bound holds."""
    w = e2m1_weight(weight, group_scale, x.shape[-1])
    return linear(x, w, bias, act, residual, None, row_scale, out_dtype)


def decay_attention(q, k, v, decay, state=None, lengths=None, scale=None):
    """((value, bound) of the outputs, (value, bound) of the states), token after token."""
    B, L, H, dk = q.shape
    dv = v.shape[3]
    scale = 1 / math.sqrt(dk) if scale is None else scale
    S = torch.zeros((B, H, dk, dv), dtype=torch.float64, device=q.device) if state is None else state.double().clone()
    A, G, F = S.abs(), torch.zeros_like(S), torch.zeros_like(S[..., :1])  # sums of magnitudes, and what they are off by
    out = torch.zeros((B, L, H, dv), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    g = decay.double()[None, :, None, None]
    f = torch.finfo(q.dtype)
    # Relative to the sums of magnitudes.  A term of a state is a sum of 16-bit values, 24 bits of them, or with fp16 22;
    # it and its two or three parts round by up to 2 U each when they are added.  Fp16's second part is 2^11 times as large
    # as what it stands for and lies on steps of 2^-24 at the least, after the decay within its chunk: each token adds
    # up to |k| 2^-36, whatever its age (F; chunks' own decay is left out of it).  A term's decay after
    # m tokens is a product of powers, each off by its exponent's rounding (a logarithm off by a unit, a product: |ln g|
    # 2^-22 a token) and by a unit itself, one a chunk of 64 tokens and a few more.  Outputs take the weights Q K^T . D as
    # sums of two bf16 values on both types: the first is off by 2^-8 of the weight's power of two, so that the second lies
    # below that and is off by 2^-8 of it and half, 2^-17 together; they take the state whole in bf16, as a sum of two
    # values and off by 2^-22 in fp16.  They have sums of dk and 64 terms.
    each = torch.where(g > 0, -torch.log(g.clamp(min=1e-30)), 0.0) * 2.0**-22 + 2.0**-27 + 6 * U
    low = 2.0**-36 if q.dtype == torch.float16 else 0
    two = 2.0**-17 if q.dtype == torch.bfloat16 else 2.0**-17 + 2.0**-22
    n = torch.full((B,), L, device=q.device) if lengths is None else lengths.long().clamp(0, L)
    for t in range(int(n.max()) if B and L else 0):
        on = (t < n)[:, None, None, None]
        qt, kt, vt = (x[:, t].double() for x in (q, k, v))
        qt, kt, vt = (torch.where(on[..., 0], x, 0.0) for x in (qt, kt, vt))
        kv = kt[..., :, None] * vt[..., None, :]
        S = torch.where(on, g * S + kv, S)
        G, F = torch.where(on, g * (G + A * each), G), F + kt.abs()[..., None] * low
        A = torch.where(on, g * A + kv.abs(), A)
        o, a, e = ((x[..., None, :] @ m)[..., 0, :] * abs(scale) for x, m in ((qt, S), (qt.abs(), A), (qt.abs(), G + F)))
        out[:, t] = torch.where(on[..., 0], o * math.copysign(1, scale), 0.0)
        bound[:, t] = torch.where(on[..., 0], a * (two + (2 * dk + 160) * U) + e, 0.0)
    tiny = f.smallest_normal * f.eps if q.dtype == torch.float16 else 0
    return ((out, torch.where(out != 0, bound + half_step(out, q.dtype) + tiny, bound)),
            (S, A * (2.0**-21 if q.dtype == torch.float16 else 2.0**-22) + A * 140 * U + G + F))
