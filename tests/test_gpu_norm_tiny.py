"""e4m3 rows whose largest value is so small that its quotient by 448 has few bits left, or none."""
import pytest
import torch

from sparsesnn_amd import ops

pytestmark = pytest.mark.gpu
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("D", [16, 384, 3001, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_tiny_values(dev, D, dtype):
    """Each row's y is its weight's, scaled down to 2^-149 ..; codes and scales have to give it back."""
    exponents = [-100, -117, -118, -119, -120, -126, -130, -135, -140, -141, -142, -145, -149]
    g = torch.Generator(device=dev).manual_seed(D)
    x = torch.randn(len(exponents), D, generator=g, device=dev, dtype=torch.float64)
    x /= x.abs().amax(-1, keepdim=True)
    x = (x * 2.0 ** torch.tensor(exponents, device=dev, dtype=torch.float64)[:, None]).to(dtype)
    # the squares vanish beside eps = 1, so that y = x
    q, _, c = ops.rms_norm(x, eps=1.0, out_dtype=E4M3)
    y = x.double()
    assert q.float().isfinite().all() and c.isfinite().all() and (c > 0).all()
    # half a step of the code, at least half of the smallest one; the scale is off by 2^-24 of itself where it is a
    # normal number; y by two more roundings or by half the smallest 32-bit value
    step = torch.clamp(y.abs() * 2.0**-4, min=0) + c.double()[:, None] * 2.0**-10
    bound = step * (1 + 2.0**-16) + y.abs() * 2.0**-21 + 2.0**-149
    assert ((q.double() * c.double()[:, None] - y).abs() <= bound).all()
    large = y.abs().amax(-1) >= 448 * 2.0**-126
    assert torch.allclose(c[large].double(), y.abs().amax(-1)[large] / 448, rtol=2.0**-22, atol=0)
