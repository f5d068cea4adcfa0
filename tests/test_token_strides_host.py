"""Which rows the linear operator's tile kernels take, as the scratch memory that they ask for shows it (on the host)."""
import ctypes

import pytest

from sparsesnn_amd import _lib


def _size(x_stride, weight_stride):
    d = _lib.LinearDesc(M=32, x_stride=x_stride, weight_stride=weight_stride, residual_stride=0, out_stride=4096, N=4096,
                        K=8192, in_type=3, out_type=3, bias_type=0, activation=0)
    n = ctypes.c_size_t(7)
    assert _lib.load().sengine_amd_linear_workspace(ctypes.byref(d), ctypes.byref(n)) == 0
    return n.value


def test_rows_in_order():
    for a, b in ((8192, 8192), (0, 8192), (8192, 0), (16384, 9216), (2**21 - 8, 8192)):
        assert _size(a, b) > 0


@pytest.mark.parametrize("x_stride,weight_stride", [(-8192, 8192), (8192, -8192), (-8192, -8192), (-16, 8192),
                                                    (2**21, 8192), (8192, 2**21), (-2**40, 8192)])
def test_rows_backwards_or_far_apart(x_stride, weight_stride):
    """Their offsets are not those of a tile's copies (32 bits, from its first row on)."""
    assert _size(x_stride, weight_stride) == 0
