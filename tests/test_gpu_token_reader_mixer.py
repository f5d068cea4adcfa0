"""TokenReader with mixers, positions and 4-bit weights: every operator's result on the way against its formula, a stream
read token by token against the whole, a captured step, and sequences of their own lengths."""
import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import token_reader as tr
from sparsesnn_amd.ops import SEngineError
from tests.test_gpu_token_ops import _check_norm, _within

pytestmark = pytest.mark.gpu
F16, BF16, I32 = torch.float16, torch.bfloat16, torch.int32
EMBED, HEADS, DEPTH, SECTIONS = 96, 2, 2, (8, 8, 6)


def _reader(dev, dtype, four_bit, seed=1, queries=1):
    params = tr.random_reader_params(seed, embed=EMBED, depth=DEPTH, num_classes=70, queries=queries, mixer_heads=HEADS)
    return params, tr.TokenReader(params, heads=HEADS, dtype=dtype, eight_bit=False, four_bit=four_bit, sections=SECTIONS,
                                  device=dev)


def _positions(n, side, dev):
    i = torch.arange(n, device=dev)
    return torch.stack([i // (side * side), i // side % side, i % side], -1).to(I32)


def test_params_without_a_mixer_are_as_they_were():
    a = tr.random_reader_params(3, embed=64, depth=2)
    b = tr.random_reader_params(3, embed=64, depth=2, mixer_heads=4)
    assert set(a) < set(b) and all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Lq,N", [(1, 196), (70, 300)])
def test_every_step(dev, monkeypatch, four_bit, dtype, Lq, N):
    given = []

    def recorded(name):
        f = getattr(tr.ops, name)

        def call(*args, **kw):
            out = f(*args, **kw)
            given.append((name, [None if t is None else t.clone() for t in (out if isinstance(out, tuple) else (out,))]))
            return out

        monkeypatch.setattr(tr.ops, name, call)

    params, reader = _reader(dev, dtype, four_bit, queries=Lq)
    p = {k: v.to(dev, dtype) for k, v in params.items()}
    g = torch.Generator(device=dev).manual_seed(Lq)
    B, d = 3, EMBED // HEADS
    tokens = torch.randint(0, 6, (B, N, EMBED), generator=g, device=dev).to(dtype)
    key_positions, positions = _positions(N, 14, dev), _positions(Lq, 14, dev) + 1000
    start = [torch.randn(B, HEADS, d, d, generator=g, device=dev) for _ in range(DEPTH)]
    state = [s.clone() for s in start]
    for name in ("rms_norm", "linear", "linear_e2m1", "rotary", "cross_attention", "decay_attention"):
        recorded(name)
    logits = reader.read(reader.encode(tokens, key_positions), positions=positions, state=state)
    steps = iter(given)

    def norm(x, weight, residual=None):
        name, got = next(steps)
        assert name == "rms_norm"
        _check_norm(x, p[weight + ".weight"], residual, 1e-6, None, got)
        return got

    def linear(x, layer, act="none", residual=None, out_dtype=dtype, four=four_bit):
        name, (got,) = next(steps)
        assert name == ("linear_e2m1" if four else "linear") and got.dtype == out_dtype
        if four:
            parts = tr.e2m1_groups(params[layer + ".weight"].to(dev))
            _within(got, *ref.linear_e2m1(x, *parts, p[layer + ".bias"], act, residual, out_dtype))
        else:
            _within(got, *ref.linear(x, p[layer + ".weight"], p[layer + ".bias"], act, residual, None, None, out_dtype))
        return got

    def turned(pos, *xs):
        name, got = next(steps)
        assert name == "rotary"
        for x, y in zip(xs, got):
            _within(y, *ref.rotary(x, pos, reader.frequencies, SECTIONS, False))
        return got

    kv = []
    for i in range(DEPTH):
        y = norm(tokens, f"block.{i}.norm_kv")[0]
        m = linear(y, f"block.{i}.kv", four=False).view(B, N, 2, HEADS, d)
        kv.append((turned(key_positions, m[:, :, 0])[0], m[:, :, 1]))
    x = p["queries"].expand(B, -1, -1)
    for i in range(DEPTH):
        pre = f"block.{i}."
        qkv = linear(norm(x, pre + "norm_mix")[0], pre + "mix").view(B, Lq, 3, HEADS, d)
        mq, mk = turned(positions, qkv[:, :, 0], qkv[:, :, 1])
        name, (o, s) = next(steps)
        assert name == "decay_attention"
        want = ref.decay_attention(mq, mk, qkv[:, :, 2], params[pre + "mix.decay"].to(dev), start[i])
        _within(o, *want[0])
        _within(s, *want[1])
        assert torch.equal(s, state[i])
        x = linear(o.view(B, Lq, EMBED), pre + "mix_out", residual=x)
        q = linear(norm(x, pre + "norm1")[0], pre + "q").view(B, Lq, HEADS, d)
        q = turned(positions, q)[0]
        name, (o,) = next(steps)
        assert name == "cross_attention"
        _within(o, *ref.cross_attention(q, *kv[i]))
        a = linear(o.view(B, Lq, EMBED), pre + "out")
        y, x = norm(a, pre + "norm2", x)
        h = linear(y, pre + "fc1", "gelu")
        x = linear(h, pre + "fc2", residual=x)
    want = linear(norm(x, "norm")[0], "head", out_dtype=torch.float32)
    assert next(steps, None) is None and torch.equal(logits, want)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_stream_token_by_token(dev, four_bit, dtype):
    """A prompt and then single tokens on the state give what the whole stream gives in one call."""
    _, reader = _reader(dev, dtype, four_bit)
    g = torch.Generator(device=dev).manual_seed(7)
    B, L, prompt = 3, 100, 90
    memory = reader.encode(torch.randint(0, 6, (B, 196, EMBED), generator=g, device=dev).to(dtype), _positions(196, 14, dev))
    x = torch.randn(B, L, EMBED, generator=g, device=dev).to(dtype)
    pos = _positions(L, 5, dev)
    before = x.clone()
    whole = reader.read(memory, x, positions=pos, state=reader.start(B))
    state = reader.start(B)
    parts = [reader.read(memory, x[:, :prompt].contiguous(), positions=pos[:prompt], state=state)]
    for t in range(prompt, L):
        parts.append(reader.read(memory, x[:, t:t + 1].contiguous(), positions=pos[t:t + 1], state=state))
    got = torch.cat(parts, 1)
    assert torch.equal(x, before)
    # Other kernels give the same sums in other orders: each of a block's twelve stored tensors may be rounded the other
    # way, by a step of its type, and their effects on the stream add up at worst
    assert float((got - whole).norm() / whole.norm()) <= DEPTH * 12 * torch.finfo(dtype).eps
    alone = reader.read(memory, x, positions=pos)  # no state: the mixers begin with nothing and keep nothing
    assert torch.equal(alone, whole)
    assert float((reader.read(memory, x[:, prompt:].contiguous(), positions=pos[prompt:]) - whole[:, prompt:]).norm()) > 1


def test_a_captured_step(dev):
    """One token's step, captured; replays advance the state as eager steps do."""
    _, reader = _reader(dev, F16, True)
    g = torch.Generator(device=dev).manual_seed(8)
    B = 4
    memory = reader.encode(torch.randint(0, 6, (B, 196, EMBED), generator=g, device=dev).to(F16))
    x, pos = torch.randn(B, 1, EMBED, generator=g, device=dev).to(F16), torch.zeros(1, 3, dtype=I32, device=dev)
    state, twin = reader.start(B), reader.start(B)
    reader.read(memory, x, positions=pos, state=state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = reader.read(memory, x, positions=pos, state=state)
    for s in state:
        s.zero_()
    for i in range(4):
        x.copy_(torch.randn(B, 1, EMBED, generator=g, device=dev))
        pos.fill_(i)
        want = reader.read(memory, x, positions=pos, state=twin)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want) and all(torch.equal(a, b) for a, b in zip(state, twin)), i


def test_lengths_and_refusals(dev):
    _, reader = _reader(dev, BF16, False)
    g = torch.Generator(device=dev).manual_seed(9)
    memory = reader.encode(torch.randint(0, 6, (3, 50, EMBED), generator=g, device=dev).to(BF16))
    x = torch.randn(3, 40, EMBED, generator=g, device=dev).to(BF16)
    n = torch.tensor([40, 17, 0], dtype=I32, device=dev)
    state = reader.start(3)
    padded = reader.read(memory, x, state=state, lengths=n)
    x[1, 17:], x[2] = 7.0, -7.0  # what lies behind the tokens
    again = reader.start(3)
    other = reader.read(memory, x, state=again, lengths=n)
    assert torch.equal(padded[0], other[0]) and torch.equal(padded[1, :17], other[1, :17])
    assert all(torch.equal(a, b) for a, b in zip(state, again)) and all((s[2] == 0).all() for s in state)
    with pytest.raises(SEngineError, match="sections"):
        tr.TokenReader(tr.random_reader_params(0, embed=96, depth=1), heads=2, device=dev).encode(
            torch.zeros(1, 4, 96, dtype=F16, device=dev), torch.zeros(4, 3, dtype=I32, device=dev))
    with pytest.raises(SEngineError, match="state"):
        reader.read(memory, x, state=reader.start(2))
    with pytest.raises(SEngineError, match="decays"):
        tr.TokenReader(tr.random_reader_params(0, embed=96, depth=1, mixer_heads=4), heads=2, device=dev)


@pytest.mark.parametrize("Lq", [0, 5])
def test_nothing_to_read(dev, Lq):
    _, reader = _reader(dev, F16, True)
    memory = reader.encode(torch.ones(2 if Lq == 0 else 0, 50, EMBED, dtype=F16, device=dev))
    B = memory[0][0].shape[0]
    x = torch.zeros(B, Lq, EMBED, dtype=F16, device=dev)
    assert reader.read(memory, x, positions=torch.zeros(Lq, 3, dtype=I32, device=dev), state=reader.start(B)).shape == (B, Lq, 70)
