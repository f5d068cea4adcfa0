"""TokenReader (norm, linear, cross attention together) against the same network in 64 bits, on random tokens
and on a Spikformer engine's stream, eager and captured."""
import math

import pytest
import torch

from sparsesnn_amd import token_reader as tr
from sparsesnn_amd.ops import SEngineError

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _norm(x, w, eps=1e-6):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


def plain(reader, tokens, x, key_mask=None):
    """The network in 64 bits on the reader's own (rounded) weights, without its 8-bit rounding."""
    p = {k: v.double() for k, v in reader.p.items()}
    B, N, C = tokens.shape
    H = reader.heads
    lin = lambda y, n: y @ p[n + ".weight"].t() + p[n + ".bias"]
    x, tokens = x.double(), tokens.double()
    for i in range(reader.depth):
        pre = f"block.{i}."
        kv = lin(_norm(tokens, p[pre + "norm_kv.weight"]), pre + "kv").view(B, N, 2, H, C // H)
        q = lin(_norm(x, p[pre + "norm1.weight"]), pre + "q").view(B, -1, H, C // H)
        o = torch.zeros_like(q)
        for b in range(B):
            for h in range(H):
                s = q[b, :, h] @ kv[b, :, 0, h].t() / math.sqrt(C // H)
                if key_mask is not None:
                    s[:, ~key_mask[b]] = -math.inf
                o[b, :, h] = torch.softmax(s, -1) @ kv[b, :, 1, h]
        x = x + lin(o.reshape(B, -1, C), pre + "out")
        h = lin(_norm(x, p[pre + "norm2.weight"]), pre + "fc1")
        x = x + lin(h * torch.special.ndtr(h), pre + "fc2")
    return lin(_norm(x, p["norm.weight"]), "head")


def _tolerance(reader):
    """Relative to the logits' norm: a block stores about eight tensors, each off by at most half a step, and their
    effects on the stream add up at worst; 8-bit operands of the first MLP product add half a step of e4m3 each."""
    blocks = reader.depth * 8 * torch.finfo(reader.dtype).eps / 2
    return blocks + (reader.depth * 2 * 2.0**-4 if reader.eight_bit else 0)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Lq,N", [(1, 196), (5, 50), (64, 300)])
def test_reader(dev, eight_bit, dtype, Lq, N):
    reader = tr.TokenReader(tr.random_reader_params(1, embed=96, depth=2, num_classes=70, queries=Lq), heads=2,
                            dtype=dtype, eight_bit=eight_bit, device=dev)
    g = torch.Generator(device=dev).manual_seed(Lq)
    tokens = torch.randint(0, 6, (3, N, 96), generator=g, device=dev).to(dtype)  # spike counts
    mask = torch.rand(3, N, generator=g, device=dev) > 0.2
    memory = reader.encode(tokens)
    for m in (None, mask):
        got = reader.read(memory, key_mask=m)
        want = plain(reader, tokens, reader.p["queries"].expand(3, -1, -1), m)
        assert got.shape == (3, Lq, 70) and got.dtype == torch.float32
        assert float((got.double() - want).norm() / want.norm()) <= _tolerance(reader)


def test_reader_of_a_spikformer_stream_captured(dev):
    """Tokens of a Spikformer engine; the reading captured and replayed with the engine's work in between."""
    from sparsesnn_amd.spikformer import SpikformerEngine, random_params

    eng = SpikformerEngine(random_params(0, embed=384, depth=1, num_classes=10), batch=2, T=4, embed=384, heads=8, depth=1,
                           in_hw=(32, 32))
    stream, planes = eng.block_input(len(eng.blocks))
    assert planes == 0
    reader = tr.TokenReader(tr.random_reader_params(2, embed=384, depth=2, num_classes=10), heads=8, device=dev)
    g = torch.Generator(device=dev).manual_seed(5)
    tokens = stream.clone()
    reader.read(reader.encode(tokens))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = reader.read(reader.encode(tokens)).view(4, 2, 1, 10).mean(0)
    for _ in range(3):
        eng.forward(torch.rand(2, 3, 32, 32, generator=g, device=dev))
        tokens.copy_(stream)
        want = reader.read(reader.encode(tokens)).view(4, 2, 1, 10).mean(0)
        logits.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want)


def test_reader_refuses(dev):
    p = tr.random_reader_params(0, embed=96, depth=1)
    with pytest.raises(SEngineError, match="heads"):
        tr.TokenReader(p, heads=5, device=dev)
    reader = tr.TokenReader(p, heads=4, device=dev)
    with pytest.raises(SEngineError, match="encode"):
        reader.encode(torch.zeros(2, 5, 64, dtype=F16, device=dev))
