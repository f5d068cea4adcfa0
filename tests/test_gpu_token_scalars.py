"""eps and scale given as something else than a Python float: the value at the call counts, and a gradient is refused."""
import numpy as np
import pytest
import torch

from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _qkv, _randn

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_a_tensor_changed_in_place(dev, where):
    g = _gen(dev, 1)
    x = _randn(g, 5, 64, dtype=F16)
    q, k, v = _qkv(g, 1, 3, 40, 2, 2, 32, F16)
    value = torch.tensor(0.25, device=where)
    first = ops.rms_norm(x, eps=value)[0], ops.cross_attention(q, k, v, scale=value)
    value.fill_(2.0)
    second = ops.rms_norm(x, eps=value)[0], ops.cross_attention(q, k, v, scale=value)
    for got, number in ((first, 0.25), (second, 2.0)):
        assert torch.equal(got[0], ops.rms_norm(x, eps=number)[0])
        assert torch.equal(got[1], ops.cross_attention(q, k, v, scale=number))
    assert not torch.equal(first[0], second[0]) and not torch.equal(first[1], second[1])


def test_other_numbers(dev):
    g = _gen(dev, 2)
    x = _randn(g, 5, 64, dtype=F16)
    q, k, v = _qkv(g, 1, 3, 40, 2, 2, 32, F16)
    for one in (1, True, np.float32(1), np.float64(1), np.array(1.0)):
        assert torch.equal(ops.rms_norm(x, eps=one)[0], ops.rms_norm(x, eps=1.0)[0])
        assert torch.equal(ops.cross_attention(q, k, v, scale=one), ops.cross_attention(q, k, v, scale=1.0))


def test_a_gradient_is_refused(dev):
    g = _gen(dev, 3)
    x = _randn(g, 5, 64, dtype=F16)
    q, k, v = _qkv(g, 1, 3, 40, 2, 2, 32, F16)
    value = torch.nn.Parameter(torch.tensor(0.5, device=dev))
    for call in (lambda: ops.rms_norm(x, eps=value), lambda: ops.cross_attention(q, k, v, scale=value)):
        for _ in range(2):
            with pytest.raises(ops.SEngineError, match="gradient"):
                call()
        with torch.no_grad():
            call()
