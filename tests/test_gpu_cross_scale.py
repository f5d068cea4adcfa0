"""Cross attention with a scale of zero: every key that counts weighs the same, whatever the last tile holds."""
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _qkv, _within

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("B,Lq,Hq,Hkv,d", [(2, 1, 2, 2, 64), (1, 9, 4, 2, 128), (2, 40, 2, 2, 48), (1, 200, 2, 1, 96),
                                           (130, 130, 2, 2, 24), (64, 257, 4, 4, 72)])
@pytest.mark.parametrize("Lk", [1, 63, 64, 65, 1400])
@pytest.mark.parametrize("dtype,zero", [(F16, 0.0), (BF16, -0.0)])
def test_scale_of_zero(dev, B, Lq, Hq, Hkv, d, Lk, dtype, zero):
    if B > 2 and Lk > 65:
        Lk = 130
    g = _gen(dev, B + Lq + Lk)
    q, k, v = _qkv(g, B, Lq, Lk, Hq, Hkv, d, dtype)
    n = torch.randint(0, Lk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    mask = torch.rand(B, Lk, generator=g, device=dev) > 0.3
    for lengths, m in ((None, None), (n, None), (None, mask), (n, mask)):
        rows = slice(0, 3)  # the oracle goes through the heads one by one
        got = ops.cross_attention(q, k, v, scale=zero, key_lengths=lengths, key_mask=m)
        assert got.isfinite().all()
        _within(got[rows], *ref.cross_attention(q[rows], k[rows], v[rows], 0.0, None if lengths is None else lengths[rows],
                                                None if m is None else m[rows]))


@pytest.mark.parametrize("Lq", [2, 64])
def test_scale_of_zero_with_merged_heads(dev, Lq):
    g = _gen(dev, Lq)
    Lk = (1 << 24) // (8 * 8 * 48) + 3
    q, k, v = _qkv(g, 8, Lq, Lk, 8, 8, 48, F16)
    _within(ops.cross_attention(q, k, v, scale=0.0), *ref.cross_attention(q, k, v, 0.0))


@pytest.mark.parametrize("Lq", [1, 40, 150])
def test_scale_of_zero_keeps_what_is_not_a_number(dev, Lq):
    """Zero times an infinite or undefined score is not a number, as the formula has it."""
    q, k, v = _qkv(_gen(dev, 3), 1, Lq, 70, 3, 3, 64, F16)
    k[0, 5, 1, 3], q[0, 0, 0, 7], q[0, 0, 2, 9] = math.inf, math.nan, math.inf
    got = ops.cross_attention(q, k, v, scale=0.0)
    bad = got.isnan().all(-1)
    assert bad[0, :, 1].all() and bad[0, 0].all()
    want = v[:, :, [0, 2]].double().mean(1, keepdim=True).expand(1, max(Lq - 1, 1), 2, 64)
    if Lq > 1:
        _within(got[:, 1:, [0, 2]], want, ref.half_step(want, F16) + 2.0**-20)
