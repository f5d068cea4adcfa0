"""fp16 attention over so many keys that those far below the largest weigh something together."""
import math

import pytest
import torch

from sparsesnn_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Lq", [1, 20, 130])
@pytest.mark.parametrize("Lk,below", [(1 << 20, 18.0), (1 << 20, 16.5), (300_001, 17.0)])
@pytest.mark.parametrize("B", [1, 300])  # in parts of the keys, and in one
@pytest.mark.parametrize("at", [0, -1])
def test_many_small_weights(dev, Lq, Lk, below, at, B):
    """One key scores `below` above all others, whose values are 1 against its 0: the result is the others' share.
    A weight is held to half a step of 2^-24 at 2^7 times its value where the largest one is the reference, so that the
    share is off by at most Lk 2^-32, beside the relative roundings (of the weights and of the result, 2^-11 each, and
    of the scores, whose error of 2^-20 the share takes on)."""
    d = 16
    q = torch.zeros(B, Lq, 1, d, dtype=torch.float16, device=dev)
    q[..., 0] = 1
    k = torch.zeros(1, Lk, 1, d, dtype=torch.float16, device=dev)
    v = torch.ones_like(k)
    k[:, at, :, 0], v[:, at] = below, 0
    share = (Lk - 1) / (Lk - 1 + math.exp(below))
    k, v = k.expand(B, Lk, 1, d), v.expand(B, Lk, 1, d)
    got = ops.cross_attention(q, k, v, scale=1.0).double()
    assert float((got - share).abs().max()) <= Lk * 2.0**-32 + share * (2 * 2.0**-11 + 2.0**-18)
