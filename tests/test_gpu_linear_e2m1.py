"""The linear operator with 4-bit weights against its definition in 64 bits: every code, groups that end inside a tile,
few and many token rows, strides and alignments, values that are no numbers, and the quantizer."""
import ctypes
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import _lib, ops
from sparsesnn_amd.token_reader import e2m1_groups
from tests.test_gpu_token_ops import _gen, _randn, _within

pytestmark = pytest.mark.gpu
F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _case(g, M, N, K, group, dtype):
    """x and a weight of all codes, with scales over e4m3's whole range."""
    x = _randn(g, M, K, dtype=dtype)
    weight = torch.randint(0, 256, (N, K // 2), generator=g, device=x.device, dtype=torch.uint8)
    scale = torch.exp2(torch.randint(-9, 8, (N, -(-K // group)), generator=g, device=x.device).float())
    scale = (scale * (1 + torch.rand(scale.shape, generator=g, device=x.device) * 0.7)).to(E4M3)
    row = torch.exp(_randn(g, N)) / (100 * math.sqrt(max(K, 1)))
    return x, weight, scale, row


SIZES = [(1, 1, 2, 32), (1, 16, 32, 32), (2, 3, 30, 32), (4, 1536, 384, 32), (3, 40, 96, 64), (5, 17, 130, 32),
         (7, 33, 128, 128), (16, 100, 1554, 64), (17, 64, 256, 128), (29, 1000, 1554, 64), (33, 130, 4096, 32),
         (48, 24, 200, 64), (64, 257, 640, 128), (65, 40, 100, 32), (100, 200, 512, 64), (300, 130, 1030, 128),
         (700, 520, 2048, 32), (2100, 1100, 384, 64), (1030, 600, 1030, 32), (65, 8200, 96, 128), (9000, 40, 100, 32), (1, 1000, 8192, 32), (16, 50, 0, 32), (80, 50, 0, 64)]


@pytest.mark.parametrize("M,N,K,group", SIZES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear_e2m1(dev, M, N, K, group, dtype):
    g = _gen(dev, M * 7 + N * 5 + K)
    x, w, s, r = _case(g, M, N, K, group, dtype)
    b, res = _randn(g, N, scale=0.5), _randn(g, M, N, dtype=dtype)
    for act, row, bias, residual in (("none", r, None, None), ("gelu", r, b.to(dtype), None), ("silu", r, b, res),
                                     ("none", None, None, None)):
        if row is None:
            x = (x / (64 * math.sqrt(max(K, 1)))).to(dtype)
        got = ops.linear_e2m1(x, w, s, row, bias, activation=act, residual=residual)
        assert got.shape == (M, N) and got.dtype == dtype
        _within(got, *ref.linear_e2m1(x, w, s, row, bias, act, residual, dtype))


@pytest.mark.parametrize("M", [1, 20, 50, 200])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_types_of_output_and_bias(dev, M, act):
    g = _gen(dev, M)
    x, w, s, r = _case(g, M, 72, 288, 32, BF16)
    for odt in (F16, BF16, F32):
        for bdt in (F16, BF16, F32):
            b, res = _randn(g, 72, dtype=bdt), _randn(g, M, 72, dtype=odt)
            got = ops.linear_e2m1(x, w, s, r, b, act, residual=res, out_dtype=odt)
            _within(got, *ref.linear_e2m1(x, w, s, r, b, act, res, odt))


@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("K,group", [(384, 32), (100, 32), (1540, 128)])
def test_strides_and_alignment(dev, M, K, group):
    g = _gen(dev, M + K)
    N = 104
    x, w, s, r = _case(g, M, N, K, group, F16)
    res = _randn(g, M, N, dtype=F16)
    want = ref.linear_e2m1(x, w, s, r, None, "none", res, F16)
    _within(ops.linear_e2m1(x, w, s, r, residual=res), *want)

    def inside(t, pad, at):  # the same values as a slice of wider rows
        wide = torch.full((t.shape[0], t.shape[1] + pad), 9.0, device=dev).to(t.dtype)
        wide[:, at:at + t.shape[1]] = t
        return wide[:, at:at + t.shape[1]]

    for pad, at in ((16, 16), (32, 8), (7, 3)):
        out = torch.zeros(M, N + pad, dtype=F16, device=dev)
        got = ops.linear_e2m1(inside(x, pad, at), inside(w, pad, at), inside(s, pad, at), r, residual=inside(res, pad, at),
                              out=out[:, at:at + N])
        _within(got, *want)
        out[:, at:at + N] = 0
        assert (out == 0).all()
    acc = res.clone()
    assert ops.linear_e2m1(x, w, s, r, residual=acc, out=acc) is acc
    _within(acc, *want)


def test_extra_dims_bytes_of_torchs_type_and_empty(dev):
    g = _gen(dev, 9)
    x, w, s, r = _case(g, 24, 40, 64, 32, F16)
    want = ref.linear_e2m1(x, w, s, r, None, "none", None, F16)
    got = ops.linear_e2m1(x.view(2, 3, 4, 64), w, s, r)
    assert got.shape == (2, 3, 4, 40)
    _within(got.view(24, 40), *want)
    if hasattr(torch, "float4_e2m1fn_x2"):
        assert torch.equal(ops.linear_e2m1(x, w.view(torch.float4_e2m1fn_x2), s, r), got.view(24, 40))
    for n in (5, 300):
        same = ops.linear_e2m1(x[:1].expand(n, 64), w, s, r)  # one row for all
        _within(same, *(t.expand(n, 40) for t in ref.linear_e2m1(x[:1], w, s, r, None, "none", None, F16)))
    assert ops.linear_e2m1(x[:0], w, s, r).shape == (0, 40)


@pytest.mark.parametrize("M", [2, 40, 300])
def test_not_numbers(dev, M):
    """NaN and infinity reach the outputs they belong to and no others."""
    g = _gen(dev, M)
    x, w, s, r = _case(g, M, 70, 200, 32, F16)
    x[0, 5] = math.nan
    s.view(torch.uint8)[3, 2] = 0x7F  # NaN
    r[9] = math.inf
    y = ops.linear_e2m1(x, w, s, r)
    assert y[0].isnan().all() and y[1:, 3].isnan().all() and not y[1:, 9].isfinite().any()
    keep = [n for n in range(70) if n not in (3, 9)]
    assert y[1:, keep].isfinite().all()


@pytest.mark.parametrize("M,K", [(8200, 130), (16000, 256)])
def test_many_rows_without_scratch_memory(dev, M, K):
    """The C entry without a workspace, or with one that is too small, reads the codes for every 64 rows."""
    g = _gen(dev, M)
    x, w, s, r = _case(g, M, 50, K, 64, BF16)
    want = ref.linear_e2m1(x, w, s, r, None, "none", None, BF16)
    d = _lib.LinearE2m1Desc(M=M, x_stride=K, weight_stride=K // 2, scale_stride=s.shape[1], residual_stride=0, out_stride=50,
                            N=50, K=K, group=64, in_type=3, out_type=3, bias_type=0, activation=0)
    lib, n = _lib.load(), ctypes.c_size_t()
    assert lib.sengine_amd_linear_e2m1_workspace(ctypes.byref(d), ctypes.byref(n)) == 0 and n.value > 0
    scratch = torch.full((n.value,), 255, dtype=torch.uint8, device=dev)
    for size in (0, 16, n.value):
        out = torch.full((M, 50), -7.0, dtype=BF16, device=dev)
        rc = lib.sengine_amd_linear_e2m1_ws(ctypes.byref(d), x.data_ptr(), w.data_ptr(), s.data_ptr(), r.data_ptr(), None,
                                            None, out.data_ptr(), scratch.data_ptr() if size else None, size,
                                            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        _within(out, *want)
    out = torch.empty((M, 50), dtype=BF16, device=dev)
    assert lib.sengine_amd_linear_e2m1(ctypes.byref(d), x.data_ptr(), w.data_ptr(), s.data_ptr(), r.data_ptr(), None, None,
                                       out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    _within(out, *want)


@pytest.mark.parametrize("K,group", [(2, 32), (96, 32), (130, 64), (384, 128)])
def test_quantizer(dev, K, group):
    g = _gen(dev, K)
    w = _randn(g, 9, K) * torch.exp(3 * _randn(g, 9, 1))
    w[4] = 0
    w[5, : min(K, group)] = 0
    codes, scale, row = e2m1_groups(w, group)
    assert codes.shape == (9, K // 2) and scale.shape == (9, -(-K // group)) and row.shape == (9,)
    got = ref.e2m1_weight(codes, scale, K) * row.double()[:, None]
    # the nearest code to value / scale: off by half of the widest step (1: between 4 and 6) times the scale; a scale is
    # off by half an e4m3 step, 2^-4, so that the largest values of a group may lie that much past the last code
    s = torch.repeat_interleave(scale.double(), group, 1)[:, :K] * row.double()[:, None]
    assert ((got - w.double()).abs() <= s * (1 + 2.0**-20)).all()
    assert (got[4] == 0).all() and row[4] == 1 and (got[5, : min(K, group)] == 0).all()
    top = w.abs().amax(-1)
    assert ((got.abs().amax(-1) - top.double()).abs() <= top * 2.0**-3).all()
