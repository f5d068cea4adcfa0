"""The linear operator's kernels at sizes that reach each of them, and their edges: few rows, 64-wide tiles
in one and in several parts, 128- and 256-wide tiles, operands that cannot be copied in 16-byte pieces."""
import ctypes

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import _lib, ops
from tests.test_gpu_token_ops import _gen, _linear_case, _randn, _within

pytestmark = pytest.mark.gpu
F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _run(dev, M, N, K, dtype, act, odt, bias=True, residual=True):
    g = _gen(dev, M + 3 * N + 5 * K)
    x, w, xs, ws = _linear_case(g, M, N, K, dtype)
    b = _randn(g, N, scale=0.5) if bias else None
    r = _randn(g, M, N, dtype=odt) if residual else None
    got = ops.linear(x, w, b, activation=act, residual=r, x_scale=xs, weight_scale=ws, out_dtype=odt)
    _within(got, *ref.linear(x, w, b, act, r, xs, ws, odt))
    return x, w, xs, ws, b, r, got


@pytest.mark.parametrize("M,N,K", [(16, 70, 8200), (17, 4096, 4096), (65, 130, 8192), (40, 2000, 6160),
                                   (33, 64, 7000), (200, 500, 3200)])
@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_few_tiles_of_a_long_reduction(dev, M, N, K, dtype):
    odt = F16 if dtype == F16 else BF16
    args = _run(dev, M, N, K, dtype, "silu", odt)
    x, w, xs, ws, b, r, got = args
    for _ in range(3):  # the parts are joined in a fixed order
        again = ops.linear(x, w, b, activation="silu", residual=r, x_scale=xs, weight_scale=ws, out_dtype=odt)
        assert torch.equal(again, got)


def test_without_scratch_memory(dev):
    """The C entry without a workspace, or with one too small, computes the same sums in one part."""
    g = _gen(dev, 2)
    M, N, K = 40, 256, 8192
    x, w, _, _ = _linear_case(g, M, N, K, BF16)
    value, bound = ref.linear(x, w, None, "none", None, None, None, BF16)
    lib = _lib.load()
    desc = _lib.LinearDesc(M=M, x_stride=K, weight_stride=K, residual_stride=0, out_stride=N, N=N, K=K, in_type=3,
                           out_type=3, bias_type=0, activation=0)
    size = ctypes.c_size_t()
    assert lib.sengine_amd_linear_workspace(ctypes.byref(desc), ctypes.byref(size)) == 0 and size.value > 0
    small = torch.empty(1024, dtype=torch.uint8, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    for ws, n in ((None, 0), (small.data_ptr(), 1024)):
        out = torch.full((M, N), 7.0, dtype=BF16, device=dev)
        assert lib.sengine_amd_linear_ws(ctypes.byref(desc), x.data_ptr(), w.data_ptr(), None, None, None, None,
                                         out.data_ptr(), ws, n, stream) == 0
        _within(out, value, bound)


@pytest.mark.parametrize("M,N,K", [(2048, 2048, 64), (2050, 2049, 200), (40000, 72, 40), (1111, 5001, 336)])
@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_middle_tiles(dev, M, N, K, dtype):
    if dtype == E4M3:
        K = K // 16 * 16
    odt = {F16: F16, BF16: BF16, E4M3: F32}[dtype]
    _run(dev, M, N, K, dtype, "gelu", odt)


@pytest.mark.parametrize("M,N,K", [(4096, 4096, 1024), (4100, 4099, 1096), (70000, 264, 1600), (4096, 4104, 1168)])
@pytest.mark.parametrize("dtype,odt", [(F16, F16), (BF16, F32), (E4M3, BF16), (E4M3, F16)])
@pytest.mark.parametrize("residual", [False, True])
def test_large_tiles(dev, M, N, K, dtype, odt, residual):
    if dtype == E4M3:
        K = K // 16 * 16
    _run(dev, M, N, K, dtype, "gelu_tanh" if residual else "relu", odt, bias=residual, residual=residual)


@pytest.mark.parametrize("M,N,K", [(40, 300, 1001), (300, 200, 4099), (2000, 2100, 131)])
@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_rows_that_cannot_be_copied(dev, M, N, K, dtype):
    _run(dev, M, N, K, dtype, "none", F16 if dtype == F16 else BF16)


def test_broadcast_rows_on_tiles(dev):
    """One token row for all, and one weight row for all (strides of zero)."""
    g = _gen(dev, 4)
    x, w, _, _ = _linear_case(g, 300, 512, 512, BF16)
    got = ops.linear(x[:1].expand(3000, 512), w)
    assert (got == got[:1]).all()
    _within(got[:1], *ref.linear(x[:1], w, None, "none", None, None, None, BF16))
    got = ops.linear(x, w[:1].expand(2048, 512))
    assert (got == got[:, :1]).all()


def test_not_numbers_on_large_tiles(dev):
    """NaN and infinity next to a reduction's tail reach their outputs and no others."""
    g = _gen(dev, 6)
    x, w, _, _ = _linear_case(g, 4096, 4096, 1096, F16)
    x[7], w[100, 1090] = 1.0, float("inf")
    x[8, 1095] = float("nan")
    y = ops.linear(x, w)
    assert y[8].isnan().all()
    assert y[7, 100] == float("inf")
    rows = torch.arange(4096, device=dev) != 8
    cols = torch.arange(4096, device=dev) != 100
    assert y[rows][:, cols].isfinite().all()
