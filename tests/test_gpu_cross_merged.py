"""Cross attention whose neighbouring key heads are copied as one row (large stretches of heads of up to 48
values): rows on one wave a head and on two, lengths, masks, parts, and heads that hold no numbers."""
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _qkv, _within

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,d", [(8, 2, 5501, 8, 8, 48), (9, 64, 5000, 8, 8, 48), (2, 20, 33000, 16, 8, 32),
                                              (3, 3, 90001, 12, 4, 16), (130, 33, 700, 4, 4, 48), (1, 1, 90000, 4, 4, 48)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_merged_heads(dev, B, Lq, Lk, Hq, Hkv, d, dtype):
    g = _gen(dev, B + Lq + Lk + d)
    q, k, v = _qkv(g, B, Lq, Lk, Hq, Hkv, d, dtype)
    lengths = torch.randint(0, Lk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    mask = torch.rand(B, Lk, generator=g, device=dev) > 0.3
    mask[B // 2, Lk // 3:] = False
    for n, m in ((None, None), (lengths, mask)):
        _within(ops.cross_attention(q, k, v, key_lengths=n, key_mask=m), *ref.cross_attention(q, k, v, None, n, m))


@pytest.mark.parametrize("Lq", [1, 30])
@pytest.mark.parametrize("d", [16, 32, 48])
def test_merged_heads_do_not_touch_each_other(dev, Lq, d):
    g = _gen(dev, Lq + d)
    Lk = (1 << 24) // (2 * 8 * d) + 5
    q, k, v = _qkv(g, 2, Lq, Lk, 8, 8, d, F16)
    want = ops.cross_attention(q, k, v)
    kv = torch.stack([k, v], 2)
    for bad in (math.nan, math.inf):
        for h in (0, 6):
            kv[:, :, 0, h], kv[:, :, 1, h] = bad, bad
        got = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1])
        keep = [h for h in range(8) if h not in (0, 6)]
        assert torch.equal(got[:, :, keep], want[:, :, keep])
        assert got[:, :, [0, 6]].isnan().all()
