"""A reader of token streams: queries that attend to an encoder's tokens, out of the token operators.

Spikformer's forward (models/spikformer.py:148-149, 277-288 in the reference) ends in a real-valued token
stream (T*B, N, C) of which its head keeps the mean.  A TokenReader keeps the tokens: a stack of pre-norm
blocks, each

    y      = norm(x)                      ops.rms_norm
    a      = cross(y Wq^T, K, V) Wo^T     ops.linear, ops.cross_attention, ops.linear
    x, y8  = x + a, norm(x + a) in e4m3   ops.rms_norm: the residual's addition, 8-bit codes and scales
    x      = x + gelu(y8 W1^T) W2^T       ops.linear on 8-bit operands, ops.linear with the residual

over x, the stream of its queries (learned ones, or tokens that are being decoded).  `encode` makes every
block's keys and values of the tokens once; `read` may then be called any number of times, for one query
row or many.  Nothing in `read` waits for the device, so it can be captured into a graph.

Tokens that are decoded one after the other see each other through a mixer, which a block has where its params
do, ahead of the attention:

    q, k, v = norm(x) Wqkv^T              ops.rms_norm, ops.linear
    q, k   = turned by (t, h, w)          ops.rotary
    x      = x + decay(q, k, v) Wo^T      ops.decay_attention on the block's state, ops.linear with the residual

Its state (`start`) leaks by a factor a head and token, as a neuron's membrane does, and is all that a token needs
of those before it: `read` takes a prompt, and then a token at a time, updating the state in place.  With
`four_bit` what `read` multiplies with is held in 4 bits (ops.linear_e2m1): few tokens take the time of reading the
weights.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import ops
from ._lib import SEngineError

E4M3_MAX = 448.0


def random_reader_params(seed: int = 0, embed: int = 384, depth: int = 2, mlp_ratio: int = 4,
                         num_classes: int = 1000, queries: int = 1, mixer_heads: int = 0) -> dict:
    """Random weights of the shapes a TokenReader takes; mixer_heads: the heads of every block's mixer, none for 0."""
    g = torch.Generator().manual_seed(seed)

    def w(n, k):
        return torch.randn((n, k), generator=g) / math.sqrt(k)

    p = {"queries": torch.randn((queries, embed), generator=g),
         "norm.weight": 1 + 0.1 * torch.randn(embed, generator=g), "head.weight": w(num_classes, embed),
         "head.bias": 0.1 * torch.randn(num_classes, generator=g)}
    for i in range(depth):
        pre = f"block.{i}."
        for n, (rows, cols) in {"q": (embed, embed), "kv": (2 * embed, embed), "out": (embed, embed),
                                "fc1": (embed * mlp_ratio, embed), "fc2": (embed, embed * mlp_ratio)}.items():
            p[pre + n + ".weight"] = w(rows, cols)
            p[pre + n + ".bias"] = 0.1 * torch.randn(rows, generator=g)
        for n in ("norm1", "norm2", "norm_kv"):
            p[pre + n + ".weight"] = 1 + 0.1 * torch.randn(embed, generator=g)
    for i in range(depth if mixer_heads else 0):
        pre = f"block.{i}."
        for n, rows in (("mix", 3 * embed), ("mix_out", embed)):
            p[pre + n + ".weight"] = w(rows, embed)
            p[pre + n + ".bias"] = 0.1 * torch.randn(rows, generator=g)
        p[pre + "norm_mix.weight"] = 1 + 0.1 * torch.randn(embed, generator=g)
        # from heads that keep a few tokens to heads that keep some hundred
        p[pre + "mix.decay"] = 1 - torch.exp2(-torch.linspace(1, 8, mixer_heads))
    return p


def e4m3_rows(w: torch.Tensor):
    """(codes, scales) of a weight whose rows are scaled to e4m3's range."""
    c = w.float().abs().amax(-1) / E4M3_MAX
    c = torch.where(c > 0, c, torch.ones_like(c))
    return (w.float() / c[:, None]).to(torch.float8_e4m3fn), c


E2M1_MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between neighbouring sizes of e2m1 codes
E2M1_MAX = 6.0


def e2m1_groups(w: torch.Tensor, group: int = 32):
    """(codes, group scales, row scales) of a weight (N, K) in 4 bits, as ops.linear_e2m1 takes them: a row scaled to
    the range of its groups' scales (e4m3), a group to that of its codes, which are the nearest ones."""
    if w.dim() != 2 or w.shape[1] % 2 or group not in (32, 64, 128):
        raise SEngineError(f"e2m1_groups: expected (N, K) with an even K and groups of 32, 64 or 128, got {tuple(w.shape)} "
                           f"in groups of {group}")
    N, K = w.shape
    groups = -(-K // group)
    w = w.detach().float()
    row = w.abs().amax(-1) / (E2M1_MAX * E4M3_MAX) if K else w.new_zeros(N)
    row = torch.where(row > 0, row, torch.ones_like(row))
    v = torch.nn.functional.pad(w / row[:, None], (0, groups * group - K)).view(N, groups, group)
    scale = (v.abs().amax(-1) / E2M1_MAX).clamp(max=E4M3_MAX).to(torch.float8_e4m3fn)
    s = scale.float()[:, :, None]
    v = (v / torch.where(s > 0, s, torch.ones_like(s))).view(N, groups * group)[:, :K]
    codes = torch.bucketize(v.abs(), w.new_tensor(E2M1_MIDDLES))
    codes = (codes + 8 * (v < 0)).to(torch.uint8)
    return codes[:, ::2] | codes[:, 1::2] << 4, scale, row


class TokenReader:
    """params as random_reader_params names them; dtype float16 or bfloat16; eight_bit: the first MLP
    product runs on e4m3 operands; four_bit: the products of `read` are with 4-bit weights instead.
    sections: pairs of a head's values that turn by a token's position on each axis (ops.rotary), an axis'
    frequencies from 1 down to 1 / base radians a step."""

    def __init__(self, params: dict, heads: int = 8, dtype: torch.dtype = torch.float16, eight_bit: bool = True,
                 eps: float = 1e-6, device="cuda", four_bit: bool = False, sections=None, base: float = 10000.0):
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.dtype, self.heads, self.eps, self.eight_bit = dtype, heads, eps, eight_bit and not four_bit
        self.p = {k: v.detach().to(dev, dtype).contiguous() for k, v in params.items() if not k.endswith(".decay")}
        self.embed = self.p["norm.weight"].numel()
        if self.embed % heads or self.embed // heads % 8:
            raise SEngineError(f"TokenReader: {self.embed} channels do not split into {heads} heads of a multiple of 8 "
                               "values")
        self.depth = 0
        while f"block.{self.depth}.q.weight" in params:
            self.depth += 1
        self.fc1 = None
        if self.eight_bit:
            self.fc1 = [e4m3_rows(params[f"block.{i}.fc1.weight"].detach().to(dev)) for i in range(self.depth)]
        self.decay = [None] * self.depth  # of the blocks that have a mixer
        for i in range(self.depth):
            decay = params.get(f"block.{i}.mix.decay")
            if decay is not None:
                if decay.numel() != heads:
                    raise SEngineError(f"TokenReader: block {i}'s mixer has {decay.numel()} decays for {heads} heads")
                self.decay[i] = decay.detach().to(dev, torch.float32).contiguous()
        self.four = {}
        if four_bit:
            read = ("q", "out", "fc1", "fc2", "mix", "mix_out")
            for k, v in params.items():
                if k.endswith(".weight") and (k == "head.weight" or k.split(".")[-2] in read):
                    self.four[k] = e2m1_groups(v.detach().to(dev))
                    del self.p[k]
        self.sections = self.frequencies = None
        if sections is not None:
            self.sections = tuple(sections)
            self.frequencies = torch.cat([base ** -(torch.arange(n, dtype=torch.float64) / max(n, 1))
                                          for n in self.sections]).to(dev, torch.float32)

    def _linear(self, y: torch.Tensor, name: str, activation: str = "none", **kw) -> torch.Tensor:
        """One of `read`'s products."""
        four = self.four.get(name + ".weight")
        if four is not None:
            return ops.linear_e2m1(y, *four, self.p[name + ".bias"], activation, **kw)
        return ops.linear(y, self.p[name + ".weight"], self.p[name + ".bias"], activation, **kw)

    def _turned(self, q, k, positions):
        if positions is None:
            return q, k
        if self.sections is None:
            raise SEngineError("TokenReader: positions need the sections of a head's pairs")
        return ops.rotary(q, k, positions, self.frequencies, self.sections)

    def start(self, B: int):
        """The mixers' states of B sequences without a token: a list for `read`, which updates them in place."""
        d = self.embed // self.heads
        dev = self.p["norm.weight"].device
        return [None if g is None else torch.zeros((B, self.heads, d, d), dtype=torch.float32, device=dev)
                for g in self.decay]

    def encode(self, tokens: torch.Tensor, positions: Optional[torch.Tensor] = None):
        """Every block's (keys, values) of the tokens (B, N, C): each (B, N, heads, C / heads).  positions, as
        ops.rotary takes them, turn the keys."""
        if tokens.dim() != 3 or tokens.shape[-1] != self.embed:
            raise SEngineError(f"encode: expected (B, N, {self.embed}), got {tuple(tokens.shape)}")
        B, N, C = tokens.shape
        d = C // self.heads
        memory = []
        for i in range(self.depth):
            pre = f"block.{i}."
            y, _ = ops.rms_norm(tokens, self.p[pre + "norm_kv.weight"], eps=self.eps)
            kv = ops.linear(y, self.p[pre + "kv.weight"], self.p[pre + "kv.bias"]).view(B, N, 2, self.heads, d)
            k = kv[:, :, 0]
            if positions is not None:
                k = self._turned(k, None, positions)[0]
            memory.append((k, kv[:, :, 1]))
        return memory

    def read(self, memory, x: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None,
             key_mask: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, state=None,
             lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Logits (B, Lq, classes) in fp32 of the query stream x (B, Lq, C), the learned queries by
        default; key_lengths and key_mask as ops.cross_attention takes them.  positions, as ops.rotary takes
        them, are those of x: they turn the queries, and the mixers' queries and keys.  state (of `start`) is what
        the mixers begin with and is updated in place, nothing where None; lengths as ops.decay_attention takes
        them: the tokens of x that are of each sequence."""
        B = memory[0][0].shape[0]
        if x is None:
            x = self.p["queries"].expand(B, -1, -1).contiguous()
        Lq, C = x.shape[1], self.embed
        d = C // self.heads
        for i, (k, v) in enumerate(memory):
            pre = f"block.{i}."
            if self.decay[i] is not None:
                y, _ = ops.rms_norm(x, self.p[pre + "norm_mix.weight"], eps=self.eps)
                qkv = self._linear(y, pre + "mix").view(B, Lq, 3, self.heads, d)
                mq, mk = self._turned(qkv[:, :, 0], qkv[:, :, 1], positions)
                held = None if state is None else state[i]
                o, _ = ops.decay_attention(mq, mk, qkv[:, :, 2], self.decay[i], state=held, lengths=lengths,
                                           state_out=held)
                x = self._linear(o.view(B, Lq, C), pre + "mix_out", residual=x)
            y, _ = ops.rms_norm(x, self.p[pre + "norm1.weight"], eps=self.eps)
            q = self._linear(y, pre + "q").view(B, Lq, self.heads, d)
            if positions is not None:
                q = self._turned(q, None, positions)[0]
            o = ops.cross_attention(q, k, v, key_lengths=key_lengths, key_mask=key_mask)
            a = self._linear(o.view(B, Lq, C), pre + "out")
            norm2 = self.p[pre + "norm2.weight"]
            if self.eight_bit:
                y, x, scale = ops.rms_norm(a, norm2, x, eps=self.eps, out_dtype=torch.float8_e4m3fn)
                codes, wscale = self.fc1[i]
                h = ops.linear(y, codes, self.p[pre + "fc1.bias"], "gelu", x_scale=scale, weight_scale=wscale,
                               out_dtype=self.dtype)
            else:
                y, x = ops.rms_norm(a, norm2, x, eps=self.eps)
                h = self._linear(y, pre + "fc1", "gelu")
            x = self._linear(h, pre + "fc2", residual=x, out=x)
        y, _ = ops.rms_norm(x, self.p["norm.weight"], eps=self.eps)
        return self._linear(y, "head", out_dtype=torch.float32)
