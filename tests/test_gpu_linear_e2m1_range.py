"""The linear operator with 4-bit weights at both ends of bf16's range: x times a code may pass it where x times code and scale
does not, on the route that reads the codes and on the one that widens them."""
import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _within

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _case(g, M, N, K, group, size, scales):
    x = (torch.rand(M, K, generator=g, device=g.device) + 1) * size
    x = torch.where(torch.rand(M, K, generator=g, device=g.device) < 0.5, -x, x).to(BF16)
    w = torch.randint(0, 256, (N, K // 2), generator=g, device=g.device, dtype=torch.uint8)
    s = torch.tensor(scales, device=g.device)[torch.randint(0, len(scales), (N, -(-K // group)), generator=g, device=g.device)]
    return x, w, s.to(E4M3)


@pytest.mark.parametrize("M,N,K,group", [(1, 40, 384, 32), (8, 8200, 128, 64), (20, 70, 130, 128), (50, 33, 256, 32),
                                         (300, 4200, 128, 128), (9000, 40, 96, 32)])
def test_products_of_codes_past_the_range(dev, M, N, K, group):
    """x up to 2^127, where six times it is past the range, with scales of 2^-9 to 0."""
    g = _gen(dev, M + K)
    x, w, s = _case(g, M, N, K, group, 2.0**126, [2.0**-9, -(2.0**-9), 0.0, 1.75 * 2.0**-8])
    row = torch.exp2(-120 - torch.rand(N, generator=g, device=dev))
    y = ops.linear_e2m1(x, w, s, row)
    _within(y, *ref.linear_e2m1(x, w, s, row, None, "none", None, BF16))
    assert y.isfinite().all()


@pytest.mark.parametrize("M,N,K,group", [(1, 40, 384, 32), (20, 70, 130, 128), (300, 4200, 128, 128)])
def test_tiny_values(dev, M, N, K, group):
    """x down to 2^-110: the products stay within the range, and the results are as exact as others."""
    g = _gen(dev, M + N)
    x, w, s = _case(g, M, N, K, group, 2.0**-110, [2.0**-9, 448.0, -0.0625, 13.0])
    row = torch.exp2(100 + torch.rand(N, generator=g, device=dev))
    _within(ops.linear_e2m1(x, w, s, row), *ref.linear_e2m1(x, w, s, row, None, "none", None, BF16))


def test_scales_that_are_not_numbers(dev):
    g = _gen(dev, 3)
    x, w, s = _case(g, 8, 20, 256, 32, 1.0, [0.5])
    s.view(torch.uint8)[4, 3], s.view(torch.uint8)[7, 0] = 0x7F, 0xFF
    y = ops.linear_e2m1(x, w, s)
    assert y[:, 4].isnan().all() and y[:, 7].isnan().all()
    assert y[:, [n for n in range(20) if n not in (4, 7)]].isfinite().all()
