"""The norm of more rows than one launch has threads for."""
import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen

pytestmark = pytest.mark.gpu
F16, E4M3 = torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("rows", [2**27, 2**27 + 1, 2**28 + 3])
@pytest.mark.parametrize("D", [1, 3])
def test_many_rows(dev, rows, D):
    g = _gen(dev, D)
    x = torch.randn(rows, D, generator=g, device=dev, dtype=F16)
    r = torch.randn(rows, D, generator=g, device=dev, dtype=F16)
    y, s, c = ops.rms_norm(x, residual=r, out_dtype=E4M3)
    z, s2 = ops.rms_norm(x, residual=r)
    assert torch.equal(s, s2)
    at = torch.cat([torch.arange(5, device=dev), torch.arange(2**27 - 5, min(2**27 + 5, rows), device=dev),
                    torch.arange(rows - 5, rows, device=dev), torch.randint(0, rows, (10000,), generator=g, device=dev)])
    ws, s_bound, wy, bound = ref.rms_norm(x[at], None, r[at], 1e-6)
    assert ((s[at].double() - ws).abs() <= s_bound).all()
    assert ((z[at].double() - wy).abs() <= bound + ref.half_step(wy, F16)).all()
    off = (y[at].double() * c[at].double()[:, None] - wy).abs()
    assert (off <= (wy.abs() * 2.0**-4 + ref.e4m3_scale(wy)[:, None] * 2.0**-10) * (1 + 2.0**-10)).all()
    want = ((x.float() + r.float()) if D == 1 else None)
    if D == 1:  # every row: the sign of the sum, to the rounding of 1 / sqrt(1 + eps / s^2)
        big = want.abs() > 0.125
        assert torch.equal(z[big].sign(), want[big].half().sign()) and (z[big].abs().float() - 1).abs().max() <= 2.0**-10
