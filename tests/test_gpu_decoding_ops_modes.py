"""Rotary positions, decaying linear attention and the linear operator with 4-bit weights: gradients, tangents and
recordings are refused, also where a call's checks are remembered; other streams, other current devices, graphs."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from sparsesnn_amd import ops
from sparsesnn_amd.token_reader import e2m1_groups
from tests.test_gpu_token_ops import _gen, _randn

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def _calls(dev, M=6, N=40):
    g = _gen(dev, 1)
    q, k, v = (_randn(g, 2, 20, 3, 32, dtype=F16) for _ in range(3))
    pos, freq = torch.arange(20, dtype=F32, device=dev)[:, None], 1 / (1 + torch.arange(16, dtype=F32, device=dev))
    decay, state = torch.full((3,), 0.9, device=dev), _randn(g, 2, 3, 32, 32)
    codes, scale, row = e2m1_groups(_randn(g, N, 64))
    x, bias, res = _randn(g, M, 64, dtype=F16), _randn(g, N, dtype=F16), _randn(g, M, N, dtype=F16)
    return [(lambda a, b, p, f: ops.rotary(a, b, p, f, (16,)), [q, k, pos, freq]),
            (lambda a, b, c, d, s: ops.decay_attention(a, b, c, d, state=s), [q, k, v, decay, state]),
            (lambda a, r, b, t: ops.linear_e2m1(a, codes, scale, r, b, residual=t), [x, row, bias, res])]


def _pair(t):
    return t if isinstance(t, tuple) else (t,)


def test_gradients_and_tangents_are_refused(dev):
    for f, args in _calls(dev):
        want = f(*args)
        for i in range(len(args)):
            asks = [*args]
            asks[i] = args[i].clone().requires_grad_()
            for _ in range(2):
                with pytest.raises(ops.SEngineError, match="gradient"):
                    f(*asks)
            with torch.no_grad():
                assert all(torch.equal(a, b) for a, b in zip(_pair(f(*asks)), _pair(want)))
            with fwd.dual_level():
                dual = [*args]
                dual[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(ops.SEngineError, match="tangent"):
                    f(*dual)
        assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(_pair(f(*args)), _pair(want)))


def test_recordings_are_refused(dev):
    for f, args in _calls(dev):
        f(*args)
        with pytest.raises(ops.SEngineError, match="record"):
            torch.jit.trace(f, tuple(args), check_trace=False)
        with pytest.raises(ops.SEngineError, match="record"):
            make_fx(f)(*args)


def test_remembered_calls_look_at_their_tensors(dev):
    g = _gen(dev, 2)
    q, v, decay = _randn(g, 1, 5, 2, 16, dtype=F16), _randn(g, 1, 5, 2, 24, dtype=F16), torch.full((2,), 0.5, device=dev)
    for _ in range(2):
        ops.decay_attention(q, q, v, decay)
    odd = torch.empty(q.numel() + 1, dtype=F16, device=dev)[1:].view(q.shape)
    with pytest.raises(ops.SEngineError, match="q: must begin"):
        ops.decay_attention(odd, q, v, decay)
    state = torch.zeros(2 * 16 * 24 + 1, device=dev)[1:].view(1, 2, 16, 24)
    with pytest.raises(ops.SEngineError, match="state: must begin"):
        ops.decay_attention(q, q, v, decay, state=state)
    with pytest.raises(ops.SEngineError, match="decay"):
        ops.decay_attention(q, q, v, decay.double())
    pos, freq = torch.zeros(5, 1, dtype=torch.int32, device=dev), torch.ones(8, device=dev)
    ops.rotary(q, None, pos, freq, (8,))
    with pytest.raises(ops.SEngineError, match="frequencies"):
        ops.rotary(q, None, pos, freq, (7,))
    with pytest.raises(ops.SEngineError, match="positions"):
        ops.rotary(q, None, pos.long(), freq, (8,))
    with pytest.raises(TypeError, match="q must be"):
        ops.rotary([1.0], None, pos, freq, (8,))
    with pytest.raises(TypeError):
        ops.decay_attention(q, q, v, decay, scale="1")


def test_another_current_device(dev, monkeypatch):
    """Where the tensors' device is not the current one it is made so for the launch."""
    calls = _calls(dev)
    want = [f(*args) for f, args in calls]
    entered = []

    @contextlib.contextmanager
    def device(d):
        entered.append(d)
        yield

    monkeypatch.setattr(ops, "_current_device", lambda: dev.index + 1)
    monkeypatch.setattr(torch.cuda, "device", device)
    for (f, args), w in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(_pair(f(*args)), _pair(w)))
    assert entered == [dev] * 3


def test_side_streams_and_graphs(dev):
    """Few and many rows (the widened weight in scratch memory), on a stream beside and captured; two graphs replayed in
    turn with eager work in between."""
    calls = _calls(dev) + _calls(dev, M=3000, N=400)[2:]
    want = [f(*args) for f, args in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [f(*args) for f, args in calls]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(_pair(a), _pair(b)))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = [f(*args) for f, args in calls]
        graphs.append((graph, held))
    for i in range(3):
        for _, args in calls:
            args[0].copy_(args[0].flip(0) * 0.5)
        want = [f(*args) for f, args in calls]
        for graph, held in graphs:
            for t in held:
                for x in _pair(t):
                    x.fill_(-7)
        for graph, held in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, held in graphs:
            for a, b in zip(held, want):
                assert all(torch.equal(x, y) for x, y in zip(_pair(a), _pair(b))), i
