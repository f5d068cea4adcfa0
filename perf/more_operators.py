"""The operators of a reader that decodes tokens over time, as cases that can be timed and compared.

A TokenReader's queries attend to an encoder's tokens.  Decoding a stream of them, one token or a whole clip at
a time, takes three more operators; a case's "op" names one:

  rotary   queries and keys turned by their tokens' positions on several axes (time, height, width)
                                                                           (ops.rotary)
  decay    causal linear attention whose state leaks by a factor a head and token, S = g S + k^T v, o = scale q S:
           a prompt, or a single token with its state                      (ops.decay_attention)
  linear4  act(x w^T + bias) + residual with w in 4 bits (e2m1, two codes a byte, the lower first), an 8-bit
           scale (e4m3) a group of a row's values and an fp32 scale a row  (ops.linear_e2m1)

With `own` false, `run` computes each from elementary torch operations in 32 bits.  `exact` has
the same from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]

# what a drawn case may cost at most: values of a rotary, of a decay's tokens and states and its tokens
# one after the other, products and weights of a linear: the largest listed ones of each, or a part of them
MOST_ROTARY = 8 * 12544 * 16 * 48
MOST_TOKENS = 65536
MOST_TOKEN_VALUES = 65536 * 16 * 128
MOST_STATE_VALUES = 128 * 32 * 128 * 128
MOST_PRODUCTS = 4096 * 4096 * 8192
MOST_WEIGHTS = 8192 * 8192


def listed():
    return [
        # one decoding token per sequence, the encoder's own heads (8 of 48), a third of the pairs an axis
        dict(name="rotary_token_f16", op="rotary", B=4, L=1, Hq=8, Hkv=8, d=48, sections="8,8,8", dtype="f16",
             interleaved=False, positions="grid"),
        # the benchmark's clip: four time steps of 56 x 56 tokens, a batch of 8
        dict(name="rotary_clip_f16", op="rotary", B=8, L=12544, Hq=8, Hkv=8, d=48, sections="8,8,8", dtype="f16",
             interleaved=False, positions="grid"),
        # a long video prompt, grouped heads, neighbouring pairs, positions far from zero
        dict(name="rotary_long_bf16", op="rotary", B=1, L=32768, Hq=32, Hkv=8, d=128, sections="16,24,24",
             dtype="bf16", interleaved=True, positions="far"),
        # one decoding token per sequence at four time steps
        dict(name="decay_token_f16", op="decay", B=4, L=1, H=8, dk=48, dv=48, dtype="f16", lengths="full", state=True),
        # one decoding token of a large batch with wide heads: the states' bandwidth
        dict(name="decay_token_bf16", op="decay", B=128, L=1, H=32, dk=128, dv=128, dtype="bf16", lengths="full",
             state=True),
        # prompts of unequal lengths, one empty: no size a multiple of a tile's, keys narrower than values
        dict(name="decay_ragged_bf16", op="decay", B=6, L=777, H=12, dk=64, dv=80, dtype="bf16", lengths="ragged",
             state=True),
        # the benchmark's clip, token after token
        dict(name="decay_clip_f16", op="decay", B=8, L=12544, H=8, dk=48, dv=48, dtype="f16", lengths="full",
             state=False),
        # a single long stream: few heads, many tokens
        dict(name="decay_long_bf16", op="decay", B=1, L=65536, H=16, dk=128, dv=128, dtype="bf16", lengths="full",
             state=True),
        # the first MLP product of one decoding token at four time steps
        dict(name="linear4_token_f16", op="linear4", M=4, N=1536, K=384, group=32, dtype="f16", act="gelu", bias=True,
             residual=False),
        # a few decoding tokens through a wide projection back into the stream: the weights' bandwidth
        dict(name="linear4_decode_bf16", op="linear4", M=8, N=8192, K=8192, group=32, dtype="bf16", act="none",
             bias=True, residual=True),
        # class scores of a batch of tokens: the last group is short, no size a multiple of a tile's
        dict(name="linear4_ragged_f16", op="linear4", M=29, N=1000, K=1554, group=64, dtype="f16", act="none",
             bias=True, residual=False),
        # a prompt through the same kind of projection
        dict(name="linear4_prompt_bf16", op="linear4", M=4096, N=4096, K=8192, group=128, dtype="bf16", act="silu",
             bias=True, residual=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "decay", "linear4"])
    if op == "rotary":
        d = rng.choice([16, 32, 40, 48, 64, 80, 96, 128])
        axes = rng.choice([1, 2, 3])
        pairs = rng.choice([d // 2, d // 2, d // 4])  # all of a head, or its first half
        cut = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0] + cut, cut + [pairs])]
        Hkv, group, B = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 4]), _log(rng, 1, 64)
        L = max(1, min(_log(rng, 1, 65536), MOST_ROTARY // (B * Hkv * (group + 1) * d)))
        return dict(op=op, B=B, L=L, Hq=Hkv * group, Hkv=Hkv, d=d, sections=",".join(map(str, sections)),
                    dtype=rng.choice(["f16", "bf16", "f32"]), interleaved=rng.random() < 0.5,
                    positions=rng.choice(["grid", "far"]))
    if op == "decay":
        dk, dv = rng.choice([16, 32, 40, 48, 64, 80, 96, 128]), rng.choice([16, 32, 48, 64, 80, 96, 128, 256])
        H, B = rng.choice([1, 2, 4, 8, 12, 16, 32]), _log(rng, 1, 128)
        B = max(1, min(B, MOST_STATE_VALUES // (H * dk * dv)))
        L = 1 if rng.random() < 0.35 else _log(rng, 2, MOST_TOKENS)
        L = max(1, min(L, MOST_TOKEN_VALUES // (B * H * max(dk, dv))))
        return dict(op=op, B=B, L=L, H=H, dk=dk, dv=dv, dtype=rng.choice(["f16", "bf16"]),
                    lengths=rng.choice(["full", "full", "ragged"]), state=L == 1 or rng.random() < 0.5)
    group = rng.choice([32, 64, 128])
    K = _log(rng, 32, 8192)
    K = max(32, K // 32 * 32) if rng.random() < 0.85 else K // 2 * 2
    N = min(_log(rng, 16, 8192), MOST_WEIGHTS // K)
    M = _log(rng, 1, 64) if rng.random() < 0.7 else _log(rng, 65, 20000)
    M = max(1, min(M, MOST_PRODUCTS // (2 * N * K), (1 << 28) // (N + K)))
    return dict(op=op, M=M, N=N, K=K, group=group, dtype=rng.choice(["f16", "bf16"]),
                act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7,
                residual=rng.random() < 0.5)


def _lengths(case):
    """The sequences' token counts: the same for every seed, so that the work of a case is one number."""
    B, L = case["B"], case["L"]
    if case["lengths"] == "full":
        return [L] * B
    r = random.Random(B * 100_003 + L)
    n = [r.randint(L // 4, L) for _ in range(B)]
    if B > 2:
        n[r.randrange(B)] = 0  # a slot of the batch that holds no sequence
    return n


def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _grid(case, g):
    """(B, L, axes) positions of tokens in scan order on a grid of as many axes, from a place of the clip on."""
    B, L, axes = case["B"], case["L"], len(_sections(case))
    side = max(2, int(round(L ** (1 / max(2, axes)))))
    far = 1_000_000 if case["positions"] == "far" else 64
    first = torch.randint(0, far, (B, 1), generator=g, device=DEV)
    at = torch.arange(L, device=DEV)[None, :] + first * (side ** (axes - 1) if axes > 1 else 1)
    cols = [at // side ** (axes - 1 - a) % (side if a else 1 << 60) for a in range(axes)]
    return torch.stack(cols, -1).to(torch.int32)


def _quantize(w, group):
    """(codes two a byte, group scales, row scales) of a weight: rows to the largest group scale, groups to the
    largest code."""
    N, K = w.shape
    groups = -(-K // group)
    row = w.abs().amax(-1) / (6 * 448)
    row = torch.where(row > 0, row, torch.ones_like(row))
    padded = torch.zeros((N, groups * group), device=w.device)
    padded[:, :K] = w / row[:, None]
    padded = padded.view(N, groups, group)
    scale = (padded.abs().amax(-1) / 6).to(torch.float8_e4m3fn)
    s = scale.float()[:, :, None]
    v = (padded / torch.where(s > 0, s, torch.ones_like(s))).view(N, -1)[:, :K]
    codes = torch.bucketize(v.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device))
    codes = (codes + 8 * (v < 0)).to(torch.uint8)
    return codes[:, ::2] | codes[:, 1::2] << 4, scale, row


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        B, L, Hq, Hkv, d = (case[k] for k in ("B", "L", "Hq", "Hkv", "d"))
        # one product makes queries, keys and values: they lie side by side
        qkv = _randn(g, (B, L, Hq + 2 * Hkv, d), dt)
        s["q"], s["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
        s["positions"] = _grid(case, g)
        # every axis has a spectrum of its own, from 1 to 1 / 10000 radians a step
        s["frequencies"] = torch.cat([10000.0 ** -(torch.arange(n, device=DEV) / n) for n in _sections(case)]).float()
        return s
    if case["op"] == "decay":
        B, L, H, dk, dv = (case[k] for k in ("B", "L", "H", "dk", "dv"))
        s["q"], s["k"] = _randn(g, (B, L, H, dk), dt), _randn(g, (B, L, H, dk), dt, dk**-0.5)
        s["v"] = _randn(g, (B, L, H, dv), dt)
        # heads that forget within a few tokens, and heads that keep a clip
        keep = torch.linspace(1, 11, H, device=DEV) + 0.5 * torch.rand(H, generator=g, device=DEV)
        s["decay"] = 1 - torch.exp2(-keep)
        s["state"] = _randn(g, (B, H, dk, dv), torch.float32) if case["state"] else None
        s["lengths"] = None
        if case["lengths"] == "ragged":
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
        return s
    M, N, K = case["M"], case["N"], case["K"]
    s["x"] = _randn(g, (M, K), dt)
    w = torch.randn((N, K), generator=g, device=DEV) / math.sqrt(K)
    s["weight"], s["group_scale"], s["row_scale"] = _quantize(w, case["group"])
    s["bias"] = _randn(g, (N,), dt, 0.3) if case["bias"] else None
    s["residual"] = _randn(g, (M, N), dt) if case["residual"] else None
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "decay": _own_decay, "linear4": _own_linear4}[op](state)
    return {"rotary": _plain_rotary, "decay": _plain_decay, "linear4": _plain_linear4}[op](state)


def _own_rotary(s):
    from sparsesnn_amd import ops
    return ops.rotary(s["q"], s["k"], s["positions"], s["frequencies"], _sections(s["case"]),
                      interleaved=s["case"]["interleaved"])


def _own_decay(s):
    from sparsesnn_amd import ops
    out, state = ops.decay_attention(s["q"], s["k"], s["v"], s["decay"], state=s["state"], lengths=s["lengths"])
    return {"out": out, "state": state}


def _own_linear4(s):
    from sparsesnn_amd import ops
    return ops.linear_e2m1(s["x"], s["weight"], s["group_scale"], s["row_scale"], s["bias"],
                           activation=s["case"]["act"], residual=s["residual"])


def _plain_rotary(s):
    sections = torch.tensor(_sections(s["case"]), device=DEV)
    axis = torch.repeat_interleave(torch.arange(len(sections), device=DEV), sections,
                                   output_size=s["frequencies"].numel())
    angle = s["positions"][:, :, axis].double() * s["frequencies"].double()  # (B, L, pairs): far positions
    angle = angle - 2 * math.pi * torch.round(angle / (2 * math.pi))
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    turn = _turn_neighbours if s["case"]["interleaved"] else _turn_halves
    return turn(s["q"], cos, sin), turn(s["k"], cos, sin)


def _turn_halves(x, cos, sin):
    n = cos.shape[-1]
    a, b = x[..., :n].float(), x[..., n:2 * n].float()
    return torch.cat([(a * cos - b * sin).to(x.dtype), (a * sin + b * cos).to(x.dtype), x[..., 2 * n:]], -1)


def _turn_neighbours(x, cos, sin):
    n = cos.shape[-1]
    a, b = x[..., 0:2 * n:2].float(), x[..., 1:2 * n:2].float()
    turned = torch.stack([(a * cos - b * sin).to(x.dtype), (a * sin + b * cos).to(x.dtype)], -1)
    return torch.cat([turned.flatten(-2), x[..., 2 * n:]], -1)


def _powers(decay, n):
    """decay ** n for every head (last axis), in 64 bits before it is rounded: far powers of values near one."""
    return torch.pow(decay.double(), n.double()).float()


def _plain_decay(s):
    c = s["case"]
    B, L, H, dk, dv = (c[k] for k in ("B", "L", "H", "dk", "dv"))
    decay, scale = s["decay"], 1 / math.sqrt(dk)
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    start = s["state"]
    n = torch.full((B,), L, device=DEV) if s["lengths"] is None else s["lengths"].long()
    at = torch.arange(L, device=DEV)
    if s["lengths"] is not None:
        there = (at < n[:, None])[:, :, None, None]
        k, v = k.masked_fill(~there, 0), v.masked_fill(~there, 0)
    # the state behind the last token: every token's product with what it has leaked by then
    left = (n[:, None] - 1 - at).clamp(min=0)[:, :, None]  # (B, L, 1)
    weighted = k * _powers(decay, left)[..., None]
    state = torch.matmul(weighted.permute(0, 2, 3, 1), v.transpose(1, 2))  # (B, H, dk, dv)
    if start is not None:
        state = state + _powers(decay, n[:, None])[..., None, None] * start
    # chunks of C tokens: products inside a chunk, and the state that the chunk begins with
    C = 256 if L > 4096 else 64 if L > 64 else L
    chunks = -(-L // C)
    pad = chunks * C - L
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pad)).view(B, chunks, C, H, -1).permute(0, 3, 1, 2, 4)
               for t in (q, k, v))  # (B, H, chunks, C, d)
    i = torch.arange(C, device=DEV)
    apart = i[:, None] - i
    inside = _powers(decay, apart.clamp(min=0)[..., None]).masked_fill((apart < 0)[..., None], 0).permute(2, 0, 1)
    scores = torch.matmul(q, k.transpose(-1, -2)) * inside[None, :, None]
    out = torch.matmul(scores, v)
    from_state = None
    if chunks > 1:
        kv = torch.matmul((k * _powers(decay, (C - 1 - i)[:, None]).t()[None, :, None, :, None]).transpose(-1, -2), v)
        j = torch.arange(chunks, device=DEV)
        behind = j[:, None] - 1 - j
        between = _powers(decay, (C * behind.clamp(min=0))[..., None]).masked_fill((behind < 0)[..., None], 0)
        from_state = torch.matmul(between.permute(2, 0, 1), kv.reshape(B, H, chunks, dk * dv)).view(B, H, chunks, dk, dv)
    if start is not None:
        passed = _powers(decay, (C * torch.arange(chunks, device=DEV))[:, None]).t()[None, :, :, None, None]
        begun = passed * start[:, :, None]
        from_state = begun if from_state is None else from_state + begun
    if from_state is not None:
        out = out + torch.matmul(q, from_state) * _powers(decay, (i + 1)[:, None]).t()[None, :, None, :, None]
    out = (out * scale).permute(0, 2, 3, 1, 4).reshape(B, chunks * C, H, dv)[:, :L]
    if s["lengths"] is not None:
        out = out.masked_fill(~there, 0)
    return {"out": out.to(s["q"].dtype), "state": state}


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


def _plain_linear4(s):
    c = s["case"]
    N, K = c["N"], c["K"]
    values = torch.tensor(E2M1, device=DEV)
    w = torch.stack([values[(s["weight"] & 15).int()], values[(s["weight"] >> 4).int()]], -1).view(N, K)
    w = w * torch.repeat_interleave(s["group_scale"].float(), c["group"], 1)[:, :K]
    z = s["x"].float() @ w.t() * s["row_scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    z = _activation(z, c["act"])
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(s["x"].dtype)


def work(case):
    e = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "rotary":
        values = case["B"] * case["L"] * (case["Hq"] + case["Hkv"]) * case["d"]
        axes = len(_sections(case))
        return {"bytes": 2 * values * e + case["B"] * case["L"] * axes * 4, "flops": 3 * values}
    if case["op"] == "decay":
        B, L, H, dk, dv = (case[k] for k in ("B", "L", "H", "dk", "dv"))
        tokens = sum(_lengths(case))
        states = B * H * dk * dv
        return {"bytes": tokens * H * (2 * dk + dv) * e + B * L * H * dv * e + 4 * states * (2 if case["state"] else 1),
                "flops": 4 * tokens * H * dk * dv}
    M, N, K = case["M"], case["N"], case["K"]
    groups = -(-K // case["group"])
    return {"bytes": N * K // 2 + N * groups + 4 * N + M * K * e + M * N * e * (2 if case["residual"] else 1)
            + N * e * case["bias"], "flops": 2 * M * N * K}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "decay": _exact_decay, "linear4": _exact_linear4}[case["op"]](case, s)


def _exact_rotary(case, s):
    """Each pair as a complex number, times exp(i angle)."""
    out = []
    pos, freq = s["positions"].double(), s["frequencies"].double()
    first, turns = 0, []
    for a, n in enumerate(_sections(case)):
        turns.append(torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                                 pos[:, :, a:a + 1] * freq[first:first + n]))
        first += n
    turn = torch.cat(turns, -1)[:, :, None]
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        r = y[..., :2 * first]
        z = torch.complex(r[..., 0::2], r[..., 1::2]) if case["interleaved"] else torch.complex(*r.chunk(2, -1))
        z = z * turn
        if case["interleaved"]:
            r[..., 0::2], r[..., 1::2] = z.real, z.imag
        else:
            r[..., :first], r[..., first:] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_decay(case, s):
    """Token after token."""
    B, L, H, dk, dv = (case[k] for k in ("B", "L", "H", "dk", "dv"))
    state = torch.zeros((B * H, dk, dv), dtype=torch.float64, device=DEV)
    if s["state"] is not None:
        state += s["state"].double().view(B * H, dk, dv)
    out = torch.zeros((B, L, H, dv), dtype=torch.float64, device=DEV)
    n = _lengths(case)
    live = torch.tensor(n, device=DEV).repeat_interleave(H)
    g = s["decay"].double().repeat(B)
    full = min(n) == L
    for t in range(max(n)):
        q, k, v = (s[x][:, t].double().reshape(B * H, -1) for x in ("q", "k", "v"))
        if full:
            state *= g[:, None, None]
            state.baddbmm_(k[:, :, None].contiguous(), v[:, None].contiguous())
            out[:, t] = torch.bmm(q[:, None], state).view(B, H, dv)
            continue
        on = (t < live)[:, None, None]
        state = torch.where(on, state * g[:, None, None] + k[:, :, None] * v[:, None], state)
        out[:, t] = torch.where(on, torch.bmm(q[:, None], state), 0.0).view(B, H, dv)
    return {"out": out / math.sqrt(dk), "state": state.view(B, H, dk, dv)}


def _exact_linear4(case, s):
    N, K, group = case["N"], case["K"], case["group"]
    w = torch.empty((N, K), dtype=torch.float64, device=DEV)
    for half in (0, 1):
        c = (s["weight"] >> (4 * half)).to(torch.int64) & 15
        e, m = c >> 1 & 3, (c & 1).double()
        size = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1))
        w[:, half::2] = torch.where(c >= 8, -size, size)
    for i in range(s["group_scale"].shape[1]):
        w[:, i * group:(i + 1) * group] *= s["group_scale"][:, i:i + 1].double()
    z = torch.mm(s["x"].double(), (w * s["row_scale"].double()[:, None]).t().contiguous())
    if s["bias"] is not None:
        z += s["bias"].double()
    act = case["act"]
    if act == "relu":
        z = torch.where(z > 0, z, 0.0)
    elif act == "gelu":
        z = z * torch.special.ndtr(z)
    elif act == "gelu_tanh":
        z = z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    elif act == "silu":
        z = z / (1 + torch.exp(-z))
    if s["residual"] is not None:
        z += s["residual"].double()
    return z
