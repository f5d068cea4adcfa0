"""Cross attention's outputs that would be written twice, refused on the host."""
import ctypes

import pytest

from sparsesnn_amd import _lib

P = 0x1000
S3 = ctypes.c_int64 * 3


def _call(sizes, out_stride):
    d = _lib.CrossDesc(B=2, Lq=3, Lk=5, Hq=4, Hkv=2, d=64, type=1, scale=0.1)
    for k, v in sizes.items():
        setattr(d, k, v)
    for name in ("q_stride", "k_stride", "v_stride"):
        setattr(d, name, S3(768, 256, 64))
    d.out_stride = S3(*out_stride)
    lib = _lib.load()
    rc = lib.sengine_amd_cross_attention(ctypes.byref(d), P, P, P, None, None, P, None)
    return rc, lib.sengine_amd_last_error().decode()


@pytest.mark.parametrize("sizes,out_stride", [
    ({}, (0, 256, 64)), ({}, (768, 0, 64)), ({}, (768, 256, 0)), ({}, (768, 256, 56)), ({}, (768, 256, -56)),
    ({}, (8, 256, 64)), (dict(B=1), (0, 256, 32)), (dict(Lq=1, Hq=2), (63, 0, 64))])
def test_rows_that_overlap(sizes, out_stride):
    rc, text = _call(sizes, out_stride)
    assert rc == -2 and "overlap" in text
