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
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import ops
from ._lib import SEngineError

E4M3_MAX = 448.0


def random_reader_params(seed: int = 0, embed: int = 384, depth: int = 2, mlp_ratio: int = 4,
                         num_classes: int = 1000, queries: int = 1) -> dict:
    """Random weights of the shapes a TokenReader takes."""
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
    return p


def e4m3_rows(w: torch.Tensor):
    """(codes, scales) of a weight whose rows are scaled to e4m3's range."""
    c = w.float().abs().amax(-1) / E4M3_MAX
    c = torch.where(c > 0, c, torch.ones_like(c))
    return (w.float() / c[:, None]).to(torch.float8_e4m3fn), c


class TokenReader:
    """params as random_reader_params names them; dtype float16 or bfloat16; eight_bit: the first MLP
    product runs on e4m3 operands."""

    def __init__(self, params: dict, heads: int = 8, dtype: torch.dtype = torch.float16, eight_bit: bool = True,
                 eps: float = 1e-6, device="cuda"):
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.dtype, self.heads, self.eps, self.eight_bit = dtype, heads, eps, eight_bit
        self.p = {k: v.detach().to(dev, dtype).contiguous() for k, v in params.items()}
        self.embed = self.p["norm.weight"].numel()
        if self.embed % heads or self.embed // heads % 8:
            raise SEngineError(f"TokenReader: {self.embed} channels do not split into {heads} heads of a multiple of 8 "
                               "values")
        self.depth = 0
        while f"block.{self.depth}.q.weight" in params:
            self.depth += 1
        self.fc1 = None
        if eight_bit:
            self.fc1 = [e4m3_rows(params[f"block.{i}.fc1.weight"].detach().to(dev)) for i in range(self.depth)]

    def encode(self, tokens: torch.Tensor):
        """Every block's (keys, values) of the tokens (B, N, C): each (B, N, heads, C / heads)."""
        if tokens.dim() != 3 or tokens.shape[-1] != self.embed:
            raise SEngineError(f"encode: expected (B, N, {self.embed}), got {tuple(tokens.shape)}")
        B, N, C = tokens.shape
        d = C // self.heads
        memory = []
        for i in range(self.depth):
            pre = f"block.{i}."
            y, _ = ops.rms_norm(tokens, self.p[pre + "norm_kv.weight"], eps=self.eps)
            kv = ops.linear(y, self.p[pre + "kv.weight"], self.p[pre + "kv.bias"]).view(B, N, 2, self.heads, d)
            memory.append((kv[:, :, 0], kv[:, :, 1]))
        return memory

    def read(self, memory, x: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None,
             key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Logits (B, Lq, classes) in fp32 of the query stream x (B, Lq, C), the learned queries by
        default; key_lengths and key_mask as ops.cross_attention takes them."""
        B = memory[0][0].shape[0]
        if x is None:
            x = self.p["queries"].expand(B, -1, -1).contiguous()
        Lq, C = x.shape[1], self.embed
        for i, (k, v) in enumerate(memory):
            pre = f"block.{i}."
            w = lambda name: (self.p[pre + name + ".weight"], self.p[pre + name + ".bias"])
            y, _ = ops.rms_norm(x, self.p[pre + "norm1.weight"], eps=self.eps)
            q = ops.linear(y, *w("q")).view(B, Lq, self.heads, C // self.heads)
            o = ops.cross_attention(q, k, v, key_lengths=key_lengths, key_mask=key_mask)
            a = ops.linear(o.view(B, Lq, C), *w("out"))
            norm2 = self.p[pre + "norm2.weight"]
            if self.eight_bit:
                y, x, scale = ops.rms_norm(a, norm2, x, eps=self.eps, out_dtype=torch.float8_e4m3fn)
                codes, wscale = self.fc1[i]
                h = ops.linear(y, codes, self.p[pre + "fc1.bias"], "gelu", x_scale=scale, weight_scale=wscale,
                               out_dtype=self.dtype)
            else:
                y, x = ops.rms_norm(a, norm2, x, eps=self.eps)
                h = ops.linear(y, *w("fc1"), "gelu")
            x = ops.linear(h, *w("fc2"), residual=x, out=x)
        y, _ = ops.rms_norm(x, self.p["norm.weight"], eps=self.eps)
        return ops.linear(y, self.p["head.weight"], self.p["head.bias"], out_dtype=torch.float32)
