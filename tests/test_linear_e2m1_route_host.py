"""Which calls of the linear operator with 4-bit weights ask for memory to widen the weight in (no kernel is launched)."""
import ctypes

import pytest

from sparsesnn_amd import _lib


def _bytes(M, N, K, x_stride):
    d = _lib.LinearE2m1Desc(M=M, x_stride=x_stride, weight_stride=K // 2, scale_stride=-(-K // 32), residual_stride=0,
                            out_stride=N, N=N, K=K, group=32, in_type=1, out_type=1, bias_type=0, activation=0)
    n = ctypes.c_size_t(7)
    assert _lib.load().sengine_amd_linear_e2m1_workspace(ctypes.byref(d), ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("K,x_stride", [(8190, 8190), (8192, 8196), (8192, 8199), (8190, 8192)])
def test_rows_of_x_that_are_no_whole_pieces(K, x_stride):
    """Up to 128 rows of them are multiplied with the codes; the tiles of a widened weight do not take them."""
    for M in (65, 70, 128):
        assert _bytes(M, 8192, K, x_stride) == 0
    for M in (129, 256, 4096):
        assert _bytes(M, 8192, K, x_stride) >= 8192 * 8192 * 2


def test_rows_of_whole_pieces():
    assert _bytes(64, 8192, 8192, 8192) == 0 and _bytes(128, 1000, 8192, 8192) == 0
    for M, x_stride in ((65, 8192), (128, 8200), (129, 8192)):
        assert _bytes(M, 8192, 8192, x_stride) >= 8192 * 8192 * 2
