"""Sizes that a descriptor's 32-bit fields cannot hold, refused by the torch wrappers before they are cut (no kernel is
launched; the tensors have no memory)."""
import pytest
import torch

from sparsesnn_amd import ops

F16, E4M3 = torch.float16, torch.float8_e4m3fn
BIG = 2**32


class OnDevice(torch.Tensor):
    is_cuda = True


def _t(*shape, dtype=F16):
    return torch.empty(*shape, dtype=dtype, device="meta").as_subclass(OnDevice)


@pytest.mark.parametrize("D", [2**31, BIG + 8, 3 * BIG + 384])
def test_norm(D):
    for dtype in (None, E4M3):
        with pytest.raises(ops.SEngineError, match="D"):
            ops._rms_norm_plan(None, _t(2, D), None, None, 1e-6, dtype, None, None, None)
    assert ops._rms_norm_plan(None, _t(BIG // 2, 64), None, None, 1e-6, None, None, None, None)


@pytest.mark.parametrize("M,N,K", [(3, BIG + 16, 8), (3, 16, BIG + 8), (40, 2**31, 8), (40, 8, 2**31)])
def test_linear(M, N, K):
    for dtype in (F16, E4M3):
        with pytest.raises(ops.SEngineError, match="N and K"):
            ops._linear_plan(None, _t(M, K, dtype=dtype), _t(N, K, dtype=dtype), None, "none", None, None, None, None, None)
    assert ops._linear_plan(None, _t(BIG, 8), _t(16, 8), None, "none", None, None, None, None, None)


@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv", [(BIG + 1, 1, 4, 2, 2), (1, BIG + 3, 4, 2, 2), (1, 1, BIG + 5, 2, 2),
                                            (1, 1, 4, BIG + 2, 2), (1, 1, 4, BIG + 2, BIG + 1), (1, 1, 2**31, 1, 1)])
def test_cross_attention(B, Lq, Lk, Hq, Hkv):
    q, k = _t(B, Lq, Hq, 64), _t(B, Lk, Hkv, 64)
    with pytest.raises(ops.SEngineError, match="2\\*\\*31"):
        ops._cross_plan(None, q, k, k, None, None, None, None)


def test_cross_attention_of_wide_heads():
    q = _t(1, 2, 1, BIG + 64)
    with pytest.raises(ops.SEngineError, match="2\\*\\*31"):
        ops._cross_plan(None, q, q, q, None, None, None, None)
