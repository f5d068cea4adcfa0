"""The operators of a reader of token streams, as cases that can be timed and compared.

Spikformer ends in a real-valued token stream.  A reader of it is a stack of pre-norm blocks whose
queries attend to those tokens; it is made of three operators, and a case's "op" names one:

  norm    s = x + residual, then s over its root mean square; in the input's type, or in 8 bits
          (e4m3) with one scale a row                                      (ops.rms_norm)
  linear  act(x w^T + bias) + residual on 16-bit operands, or on e4m3 operands with their scales
                                                                           (ops.linear)
  cross   attention of Lq queries to Lk encoder states, grouped heads, sequences of their own
          lengths, keys that a mask leaves out                             (ops.cross_attention)

With `own` false, `run` computes each from elementary torch operations in 32 bits.  `exact` has
the same from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
EPS = 1e-6
E4M3_MAX = 448.0

# what a drawn case may cost at most: values of a norm, products of a linear, scores (all heads) and
# key / value bytes of an attention: the largest listed ones of each
MOST_VALUES = 401_408 * 384
MOST_PRODUCTS = 8192 * 8192 * 8192
MOST_SCORES = 4 * 16 * 4096 * 4001
MOST_KV_BYTES = 8 * 16384 * 8 * 128 * 4


def listed():
    return [
        # the stream of a single image's one decoding token over four time steps
        dict(name="norm_token_f16", op="norm", rows=4, D=384, dtype="f16", out="same", residual=True),
        # the benchmark's whole token stream: 3136 tokens, batch 32, four time steps
        dict(name="norm_3136_f16_e4m3", op="norm", rows=4 * 32 * 3136, D=384, dtype="f16", out="e4m3", residual=True),
        # the first MLP product of one decoding token at four time steps
        dict(name="linear_token_f16", op="linear", M=4, N=1536, K=384, dtype="f16", out="f16", act="gelu", bias=True,
             residual=False),
        # a batch of decoding tokens through a wide projection back into the stream: the weights' bandwidth
        dict(name="linear_decode_bf16", op="linear", M=32, N=4096, K=8192, dtype="bf16", out="bf16", act="none",
             bias=True, residual=True),
        # class scores in 8 bits: no size a multiple of a tile's
        dict(name="linear_ragged_e4m3", op="linear", M=3001, N=1000, K=1552, dtype="e4m3", out="f32", act="none",
             bias=True, residual=False),
        # the token MLP of the benchmark's stream, a batch of 8
        dict(name="linear_mlp_f16", op="linear", M=4 * 8 * 3136, N=1536, K=384, dtype="f16", out="f16", act="gelu",
             bias=True, residual=False),
        # a long prompt's projection back into the stream
        dict(name="linear_8k_bf16", op="linear", M=8192, N=4096, K=8192, dtype="bf16", out="bf16", act="none",
             bias=True, residual=True),
        # the largest product, in 8 bits
        dict(name="linear_8k_e4m3", op="linear", M=8192, N=8192, K=8192, dtype="e4m3", out="bf16", act="silu",
             bias=True, residual=True),
        # one decoding token per sequence over 14x14 tokens, the encoder's own heads (8 of 48)
        dict(name="cross_token_196", op="cross", B=4, Lq=1, Lk=196, Hq=8, Hkv=8, d=48, dtype="f16", lengths="full",
             mask=False),
        # one decoding token per sequence over long encoder states of unequal lengths, grouped heads
        dict(name="cross_token_16k", op="cross", B=8, Lq=1, Lk=16384, Hq=32, Hkv=8, d=128, dtype="bf16",
             lengths="ragged", mask=False),
        # a readout of 64 learned tokens over the benchmark's stream, four time steps of a batch of 32
        dict(name="cross_readout_3136", op="cross", B=128, Lq=64, Lk=3136, Hq=8, Hkv=8, d=48, dtype="f16",
             lengths="full", mask=False),
        # a full prompt over a long encoder sequence with masked keys and an empty sequence
        dict(name="cross_4k", op="cross", B=4, Lq=4096, Lk=4001, Hq=16, Hkv=16, d=128, dtype="bf16",
             lengths="full", mask=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "cross"])
    if op == "norm":
        D = _log(rng, 8, 8192)
        if rng.random() < 0.6:
            D = max(8, D // 8 * 8)
        dtype = rng.choice(["f16", "bf16", "f32"])
        return dict(op=op, rows=min(_log(rng, 1, 400_000), MOST_VALUES // (2 * D)), D=D, dtype=dtype,
                    out=rng.choice(["same", "e4m3"]), residual=rng.random() < 0.7)
    if op == "linear":
        dtype = rng.choice(["f16", "bf16", "e4m3"])
        K = _log(rng, 32, 8192)
        if rng.random() < 0.85:  # rows of the operands begin at 16 bytes, as they do for almost every model
            K = max(32, K // 16 * 16)
        N = _log(rng, 16, 8192)
        M = min(_log(rng, 1, 100_000), MOST_PRODUCTS // (4 * N * K), (1 << 30) // (N + K))
        return dict(op=op, M=max(1, M), N=N, K=K, dtype=dtype,
                    out=rng.choice(["f16", "bf16", "f32"]) if dtype == "e4m3" else dtype,
                    act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.5)
    Hkv, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 4, 8])
    d = rng.choice([16, 32, 40, 48, 64, 80, 96, 128])
    B = _log(rng, 1, 64)
    Lk = max(1, min(_log(rng, 1, 16384), MOST_KV_BYTES // (2 * B * Hkv * d * 4)))
    Lq = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
    Lq = max(1, min(Lq, MOST_SCORES // (2 * B * Hkv * group * Lk)))
    return dict(op=op, B=B, Lq=Lq, Lk=Lk, Hq=Hkv * group, Hkv=Hkv, d=d, dtype=rng.choice(["f16", "bf16"]),
                lengths=rng.choice(["full", "ragged"]), mask=rng.random() < 0.3)


def _lengths(case):
    """The sequences' key counts: the same for every seed, so that the work of a case is one number."""
    B, Lk = case["B"], case["Lk"]
    if case["lengths"] == "full":
        return [Lk] * B
    r = random.Random(B * 100_003 + Lk)
    n = [r.randint(Lk // 4, Lk) for _ in range(B)]
    if B > 2:
        n[r.randrange(B)] = 0  # a slot of the batch that holds no sequence
    return n


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _to_e4m3(x):
    """(codes, scale per row) of a matrix whose rows are scaled to the type's range."""
    c = x.float().abs().amax(-1) / E4M3_MAX
    c = torch.where(c > 0, c, torch.ones_like(c))
    return (x.float() / c[:, None]).to(torch.float8_e4m3fn), c


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        shape = (case["rows"], case["D"])
        s["x"] = _randn(g, shape, dt, 0.7)
        # a token stream: its rows have grown by different amounts, some channels stand out
        s["residual"] = None
        if case["residual"]:
            grow = torch.exp(0.5 * torch.randn((case["rows"], 1), generator=g, device=DEV))
            s["residual"] = (torch.randn(shape, generator=g, device=DEV) * grow).to(dt)
        s["weight"] = (1 + 0.2 * torch.randn((case["D"],), generator=g, device=DEV)).to(dt)
        return s
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        odt = DTYPES[case["out"]]
        x = torch.randn((M, K), generator=g, device=DEV)
        w = torch.randn((N, K), generator=g, device=DEV) / math.sqrt(K)
        if case["dtype"] == "e4m3":
            s["x"], s["x_scale"] = _to_e4m3(x)
            s["weight"], s["weight_scale"] = _to_e4m3(w)
        else:
            s["x"], s["weight"], s["x_scale"], s["weight_scale"] = x.to(dt), w.to(dt), None, None
        s["bias"] = _randn(g, (N,), odt, 0.3) if case["bias"] else None
        s["residual"] = _randn(g, (M, N), odt) if case["residual"] else None
        return s
    B, Lq, Lk, Hq, Hkv, d = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hkv", "d"))
    s["q"] = _randn(g, (B, Lq, Hq, d), dt, 1.5)
    kv = _randn(g, (B, Lk, 2, Hkv, d), dt)  # one product makes both: they lie side by side
    s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
    s["key_lengths"] = None
    if case["lengths"] == "ragged":
        s["key_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    s["key_mask"] = None
    if case["mask"]:  # True: the key counts; one sequence has none
        s["key_mask"] = torch.rand((B, Lk), generator=g, device=DEV) > 0.2
        if B > 1:
            s["key_mask"][B // 2] = False
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "cross": _own_cross}[op](state)
    return {"norm": _plain_norm, "linear": _plain_linear, "cross": _plain_cross}[op](state)


def _own_norm(s):
    from sparsesnn_amd import ops
    if s["case"]["out"] == "e4m3":
        y, res, scale = ops.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS, out_dtype=torch.float8_e4m3fn)
        return {"y": y, "scale": scale, "stream": res}
    y, res = ops.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
    return {"y": y, "stream": res}


def _own_linear(s):
    from sparsesnn_amd import ops
    c = s["case"]
    return ops.linear(s["x"], s["weight"], s["bias"], activation=c["act"], residual=s["residual"],
                      x_scale=s["x_scale"], weight_scale=s["weight_scale"], out_dtype=DTYPES[c["out"]])


def _own_cross(s):
    from sparsesnn_amd import ops
    return ops.cross_attention(s["q"], s["k"], s["v"], key_lengths=s["key_lengths"], key_mask=s["key_mask"])


def _plain_norm(s):
    x = s["x"].float()
    stream = None
    if s["residual"] is not None:
        x = x + s["residual"].float()
        stream = x.to(s["x"].dtype)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if s["case"]["out"] == "same":
        return {"y": y.to(s["x"].dtype), "stream": stream}
    scale = y.abs().amax(-1) / E4M3_MAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return {"y": (y / scale[:, None]).to(torch.float8_e4m3fn), "scale": scale, "stream": stream}


def _activation(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_linear(s):
    z = s["x"].float() @ s["weight"].float().t()
    if s["x_scale"] is not None:
        z = z * s["x_scale"][:, None] * s["weight_scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    z = _activation(z, s["case"]["act"])
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(DTYPES[s["case"]["out"]])


def _plain_cross(s):
    c = s["case"]
    B, Lq, Lk, Hq, Hkv, d = (c[k] for k in ("B", "Lq", "Lk", "Hq", "Hkv", "d"))
    q = s["q"].float().view(B, Lq, Hkv, Hq // Hkv, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, d)
    k = s["k"].float().permute(0, 2, 3, 1)
    v = s["v"].float().permute(0, 2, 1, 3)
    scores = torch.matmul(q, k) * (1 / math.sqrt(d))  # (B, Hkv, group * Lq, Lk)
    counts = None
    if s["key_lengths"] is not None:
        counts = torch.arange(Lk, device=DEV) < s["key_lengths"][:, None]
    if s["key_mask"] is not None:
        counts = s["key_mask"] if counts is None else counts & s["key_mask"]
    if counts is not None:
        counts = counts[:, None, None, :]
        scores = scores.masked_fill(~counts, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if counts is not None:
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    if counts is not None:
        total = torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, v) / total
    return o.view(B, Hkv, Hq // Hkv, Lq, d).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, d).to(s["q"].dtype)


def work(case):
    b = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}
    if case["op"] == "norm":
        rows, D, e = case["rows"], case["D"], b[case["dtype"]]
        n = rows * D
        out = n * e if case["out"] == "same" else n + 4 * rows
        return {"bytes": n * e * (3 if case["residual"] else 1) + out + D * e, "flops": 6 * n}
    if case["op"] == "linear":
        M, N, K, e, o = case["M"], case["N"], case["K"], b[case["dtype"]], b[case["out"]]
        scales = 4 * (M + N) if case["dtype"] == "e4m3" else 0
        return {"bytes": (M + N) * K * e + M * N * o * (2 if case["residual"] else 1) + N * o * case["bias"] + scales,
                "flops": 2 * M * N * K}
    B, Lq, Hq, Hkv, d = (case[k] for k in ("B", "Lq", "Hq", "Hkv", "d"))
    keys = sum(_lengths(case))
    mask = B * case["Lk"] if case["mask"] else 0
    return {"bytes": 2 * (2 * B * Lq * Hq * d + 2 * keys * Hkv * d) + mask, "flops": 4 * keys * Lq * Hq * d}


# ------------------------------------------------------------------ the definitions in 64 bits

def _round_e4m3(v):
    """The nearest e4m3 value, ties to the even one: steps of 2^(e-3) at exponent e, 2^-9 below 2^-6."""
    v = v.clamp(-E4M3_MAX, E4M3_MAX)
    e = torch.frexp(v)[1] - 1
    step = torch.ldexp(torch.ones_like(v), e.clamp(min=-6) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    w = {k: (t.double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in s.items()}
    return {"norm": _exact_norm, "linear": _exact_linear, "cross": _exact_cross}[case["op"]](case, w)


def _exact_norm(case, w):
    total = w["x"] if w["residual"] is None else w["x"].add_(w["residual"])
    stream = None if w["residual"] is None else total
    rms = torch.linalg.vector_norm(total, dim=1).square_().div_(case["D"]).add_(EPS).sqrt_()
    y = total / rms[:, None]
    y *= w["weight"]
    if case["out"] == "same":
        return {"y": y, "stream": stream}
    largest = torch.maximum(y.max(1).values, -y.min(1).values)
    scale = torch.where(largest > 0, largest / E4M3_MAX, 1.0)
    return {"y": _round_e4m3(y / scale[:, None]), "scale": scale, "stream": stream}


def _exact_linear(case, w):
    x, weight = w["x"], w["weight"]
    if w["x_scale"] is not None:
        x, weight = x * w["x_scale"][:, None], weight * w["weight_scale"][:, None]
    z = torch.mm(x, weight.t().contiguous())
    if w["bias"] is not None:
        z += w["bias"]
    act = case["act"]
    if act == "relu":
        z = torch.where(z > 0, z, 0.0)
    elif act == "gelu":
        z = z * torch.special.ndtr(z)
    elif act == "gelu_tanh":
        z = z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    elif act == "silu":
        z = z / (1 + torch.exp(-z))
    if w["residual"] is not None:
        z += w["residual"]
    return z


def _exact_cross(case, w):
    q, k, v = w["q"], w["k"], w["v"]
    B, Lq, Hq, d = q.shape
    group = Hq // case["Hkv"]
    counts = torch.ones((B, case["Lk"]), dtype=torch.bool, device=q.device)
    if w["key_lengths"] is not None:
        for b, n in enumerate(w["key_lengths"].tolist()):
            counts[b, n:] = False
    if w["key_mask"] is not None:
        counts &= w["key_mask"]
    out = torch.zeros_like(q)
    for b in range(B):
        at = counts[b].nonzero()[:, 0]
        if len(at) == 0:
            continue
        for h in range(case["Hkv"]):  # the group's queries read the same keys
            kk, vv = k[b, at, h], v[b, at, h]
            qq = q[b, :, h * group:(h + 1) * group].reshape(-1, d)
            p = torch.softmax(qq @ kk.t().contiguous() / math.sqrt(d), -1)
            out[b, :, h * group:(h + 1) * group] = (p @ vv).view(Lq, group, d)
    return out
