"""States at both ends of fp32's range, with a scale that brings the outputs back."""
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _randn, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-100, -60, 60, 120, 124])
@pytest.mark.parametrize("L", [5, 100, 700])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_far_states(dev, power, L, dtype):
    """A state of about 2^power, keys of zero and a scale of its inverse."""
    g = _gen(dev, L + power)
    H, dk, dv = 3, 32, 48
    q, v = _randn(g, 2, L, H, dk, dtype=dtype, scale=1 / math.sqrt(dk)), _randn(g, 2, L, H, dv, dtype=dtype)
    k = torch.zeros_like(q)
    decay = torch.tensor([1.0, 0.999, 0.99], device=dev)  # what is left stays a normal fp32 value
    state = _randn(g, 2, H, dk, dv).clamp(-4, 4) * 2.0**power
    got = ops.decay_attention(q, k, v, decay, state=state, scale=2.0**-power)
    want = ref.decay_attention(q, k, v, decay, state, None, 2.0**-power)
    _within(got[0], *want[0])
    _within(got[1], *want[1])
