"""Sizes within the entries' limits whose launch would pass 2^32 threads, an error of the launch on the host (without a
GPU the error would be another one: no launch is tried)."""
import ctypes

import pytest

from sparsesnn_amd import _lib

P, INVALID_CONFIGURATION = 0x1000, 9
S3 = ctypes.c_int64 * 3


@pytest.mark.parametrize("M,N,K", [(1, 2**27, 8), (16, 2**31 - 256, 8), (17, 2**30, 7), (2**30, 2**12, 1032)])
def test_linear(M, N, K):
    d = _lib.LinearDesc(M=M, x_stride=K, weight_stride=K, residual_stride=0, out_stride=N, N=N, K=K, in_type=3, out_type=3,
                        bias_type=0, activation=0)
    rc = _lib.load().sengine_amd_linear(ctypes.byref(d), P, P, None, None, None, None, P, None)
    assert rc == INVALID_CONFIGURATION


@pytest.mark.parametrize("B,Lq,H,aligned", [(2**24, 1, 8, True), (2**20, 1, 64, False), (2**23, 1, 8, False),
                                            (1, 2**30 + 1, 1, False)])
def test_cross_attention(B, Lq, H, aligned):
    d = _lib.CrossDesc(B=B, Lq=Lq, Lk=5, Hq=H, Hkv=H, d=64, type=1, scale=0.1)
    for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
        setattr(d, name, S3(Lq * H * 64, H * 64, 64))
    q = P if aligned else P + 2
    rc = _lib.load().sengine_amd_cross_attention(ctypes.byref(d), q, P, P, None, None, P, None)
    assert rc == INVALID_CONFIGURATION
