"""Rows further apart than 32-bit offsets reach: token rows, outputs and a long cache's keys."""
import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _randn, _within

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _wide(rows, stride, device):
    return torch.empty(rows * stride, dtype=F16, device=device).view(rows, stride)


def test_norm_and_linear_over_four_gigabytes(dev):
    rows, stride = 40000, 65536  # 2.6e9 elements
    g = _gen(dev, 1)
    w, x = _randn(g, 24, 64, dtype=F16, scale=0.1), _randn(g, rows, 64, dtype=F16)
    wide = _wide(rows, stride, dev)
    wide[:, 8:72] = x
    out = wide[:, 128:152]
    ops.linear(wide[:, 8:72], w, activation="silu", out=out)
    _within(out, *ref.linear(x, w, None, "silu", None, None, None, F16))
    got = wide[:, 256:320]
    ops.rms_norm(wide[:, 8:72], residual=x, out=got)
    _, _, y, bound = ref.rms_norm(x, None, x, 1e-6)
    _within(got, y, bound + ref.half_step(y, F16))
    few = torch.cat([x[:1], x[-1:]])
    at = wide[::rows - 1, 8:72]  # two rows, 2.6e9 elements apart
    assert torch.equal(ops.linear(at, w), ops.linear(few, w))


@pytest.mark.parametrize("Lq", [1, 40, 150])
@pytest.mark.parametrize("masked", [False, True])
def test_a_cache_over_four_gigabytes(dev, Lq, masked):
    Lk, stride, H, d = 20000, 131072, 2, 64
    g = _gen(dev, Lq)
    kv = _randn(g, 1, Lk, 2, H, d, dtype=F16)
    wide = _wide(Lk, stride, dev)
    wide[:, :2 * H * d] = kv.view(Lk, -1)
    k, v = (wide[:, i * H * d:(i + 1) * H * d].view(Lk, H, d)[None] for i in range(2))
    q = _randn(g, 1, Lq, H, d, dtype=F16, scale=1.5)
    mask = torch.rand(1, Lk, generator=g, device=dev) > 0.5 if masked else None
    if masked:
        mask[0, :5000] = False
    _within(ops.cross_attention(q, k, v, key_mask=mask), *ref.cross_attention(q, kv[:, :, 0], kv[:, :, 1], None, None, mask))
