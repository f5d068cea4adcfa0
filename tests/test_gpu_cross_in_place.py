"""Cross attention whose output is its queries' own memory, on every form of the kernels."""
import pytest
import torch

from sparsesnn_amd import ops
from tests.test_gpu_cross_routes import _call
from tests.test_gpu_token_ops import _gen, _qkv

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,d", [
    (2, 1, 196, 8, 8, 48), (1, 1, 5000, 16, 4, 64), (2, 40, 300, 4, 2, 80), (1, 64, 3000, 2, 2, 128),
    (40, 300, 200, 4, 4, 64), (30, 300, 100, 8, 8, 128), (8, 2, 5501, 8, 8, 48), (9, 64, 5000, 8, 8, 48)])
def test_output_over_the_queries(dev, B, Lq, Lk, Hq, Hkv, d):
    g = _gen(dev, B + Lq)
    q, k, v = _qkv(g, B, Lq, Lk, Hq, Hkv, d, BF16)
    mask = torch.rand(B, Lk, generator=g, device=dev) > 0.3
    for m in (None, mask):
        want = ops.cross_attention(q, k, v, key_mask=m)
        over = q.clone()
        assert ops.cross_attention(over, k, v, key_mask=m, out=over) is over
        assert torch.equal(over, want)


def test_output_over_the_queries_of_any_alignment(dev):
    wide = torch.randn(2, 50, 3, 2, 53, generator=_gen(dev, 1), device=dev).to(F16)
    q, k, v = (wide[:, :, i, :, 3:51] for i in range(3))
    want = torch.zeros_like(q)
    _call(q, k, v, want)
    _call(q, k, v, q)
    assert torch.equal(q, want)
