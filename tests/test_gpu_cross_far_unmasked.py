"""Caches whose keys lie far apart, sequence first: without a mask a tile's 64 keys have to be near, not a stretch's."""
import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _randn, _within

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("stride", [1 << 18, (1 << 18) + 8, 1 << 21, (1 << 24) - 16, 1 << 24, (1 << 24) + 8])
@pytest.mark.parametrize("Lq", [1, 40, 130])
def test_keys_far_apart(dev, stride, Lq):
    """The values of a key's row are those of a dense cache, and with a mask too; up to strides of 2^24 elements the
    bits are the dense cache's as well."""
    Lk, H, d = 150, 2, 64
    g = _gen(dev, Lq)
    kv = _randn(g, 1, Lk, 2, H, d, dtype=BF16)
    wide = torch.empty(Lk * stride, dtype=BF16, device=dev).view(Lk, stride)
    wide[:, :2 * H * d] = kv.view(Lk, -1)
    k, v = (wide[:, i * H * d:(i + 1) * H * d].view(Lk, H, d)[None] for i in range(2))
    q = _randn(g, 1, Lq, H, d, dtype=BF16, scale=1.5)
    n = torch.tensor([147], dtype=torch.int32, device=dev)
    mask = torch.rand(1, Lk, generator=g, device=dev) > 0.3
    for lengths, m in ((None, None), (n, None), (n, mask)):
        got = ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=m)
        _within(got, *ref.cross_attention(q, kv[:, :, 0], kv[:, :, 1], None, lengths, m))
        if m is None and stride <= (1 << 24) - 16:
            assert torch.equal(got, ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], key_lengths=lengths))
