"""Calls of the token operators whose checks are remembered: new values, other layouts and what must still
be refused."""
import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _linear_case, _qkv, _randn, _within

pytestmark = pytest.mark.gpu
F16 = torch.float16


def test_every_call_has_its_own_values_and_layout(dev):
    g = _gen(dev, 11)
    for i in range(3):
        for rows in (5, 40):
            x, w, _, _ = _linear_case(g, rows, 72, 64, F16)
            wide = torch.zeros(rows, 96, dtype=F16, device=dev)
            wide[:, :64] = x
            want = ref.linear(x, w, None, "silu", None, None, None, F16)
            _within(ops.linear(x, w, activation="silu"), *want)
            _within(ops.linear(wide[:, :64], w, activation="silu"), *want)
            s, s_bound, y, y_bound = ref.rms_norm(x, None, x, 1e-6)
            for t in (x, wide[:, :64]):
                got = ops.rms_norm(t, residual=t)
                _within(got[0], y, y_bound + ref.half_step(y, F16))
                _within(got[1], s, s_bound)
                assert got[0].is_contiguous() and got[1].is_contiguous()
        q, k, v = _qkv(g, 2, 3, 50 + i, 4, 2, 32, F16)
        n = torch.tensor([50, i], dtype=torch.int32, device=dev)
        _within(ops.cross_attention(q, k, v), *ref.cross_attention(q, k, v))
        _within(ops.cross_attention(q, k, v, key_lengths=n), *ref.cross_attention(q, k, v, None, n))


def test_remembered_calls_still_refuse(dev):
    g = _gen(dev, 12)
    x, w, _, _ = _linear_case(g, 4, 32, 64, F16)
    q, k, v = _qkv(g, 1, 2, 9, 2, 2, 32, F16)
    b = _randn(g, 32, dtype=F16)
    for _ in range(2):
        ops.linear(x, w, b)
        ops.rms_norm(x, x[0].contiguous(), x)
        ops.cross_attention(q, k, v)
    grad = lambda t: t.clone().requires_grad_()
    for call in (lambda: ops.linear(grad(x), w, b), lambda: ops.linear(x, grad(w), b), lambda: ops.linear(x, w, grad(b)),
                 lambda: ops.rms_norm(grad(x), x[0].contiguous(), x), lambda: ops.rms_norm(x, x[0].contiguous(), grad(x)),
                 lambda: ops.cross_attention(grad(q), k.contiguous(), v.contiguous()),
                 lambda: ops.cross_attention(q, k, grad(v))):
        with pytest.raises(ops.SEngineError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    odd = torch.empty(q.numel() + 1, dtype=F16, device=dev)[1:].view(q.shape)  # q's layout at an odd address
    with pytest.raises(ops.SEngineError, match="16 bytes"):
        ops.cross_attention(odd, k, v)
    with pytest.raises(ops.SEngineError, match="weight"):
        ops.linear(x, w.float(), b)
    with pytest.raises(ValueError, match="activation"):
        ops.linear(x, w, b, activation="tanh")
