"""What the token operators' entries with scratch memory refuse and ask for, checked on the host."""
import ctypes

import pytest

from sparsesnn_amd import _lib

P = 0x1000  # a pointer that is only compared and checked for alignment


def _linear(**kw):
    f = dict(M=32, x_stride=8192, weight_stride=8192, residual_stride=0, out_stride=4096, N=4096, K=8192, in_type=3,
             out_type=3, bias_type=0, activation=0)
    f.update(kw)
    return _lib.LinearDesc(**f)


def _cross(**kw):
    f = dict(B=1, Lq=1, Lk=16384, Hq=4, Hkv=2, d=64, type=1, scale=0.1)
    f.update(kw)
    return _lib.CrossDesc(**f)


def _size(name, desc):
    n = ctypes.c_size_t(7)
    assert getattr(_lib.load(), name)(ctypes.byref(desc), ctypes.byref(n)) == 0
    return n.value


def test_linear_scratch_memory():
    name = "sengine_amd_linear_workspace"
    size = _size(name, _linear())
    assert size > 0 and size % (64 * 64 * 4) == 0
    # one part: few rows, many tiles, a short reduction, rows that are not whole pieces, nothing to do
    for kw in (dict(M=16), dict(M=8192), dict(K=512), dict(x_stride=8193), dict(M=0), dict(K=0)):
        assert _size(name, _linear(**kw)) == 0
    lib, n = _lib.load(), ctypes.c_size_t()
    assert lib.sengine_amd_linear_workspace(None, ctypes.byref(n)) == -1
    assert lib.sengine_amd_linear_workspace(ctypes.byref(_linear()), None) == -1
    assert lib.sengine_amd_linear_ws(ctypes.byref(_linear()), P, P, None, None, None, None, P, P + 8, size, None) == -2
    assert lib.sengine_amd_linear_ws(None, P, P, None, None, None, None, P, P, size, None) == -1


def test_cross_attention_scratch_memory():
    name = "sengine_amd_cross_attention_workspace"
    size = _size(name, _cross())
    assert size > 0 and size % ((64 + 2) * 4 * 4) == 0
    for kw in (dict(Lk=300), dict(B=600), dict(Lq=0), dict(Lk=0), dict(B=0)):
        assert _size(name, _cross(**kw)) == 0
    lib, n = _lib.load(), ctypes.c_size_t()
    assert lib.sengine_amd_cross_attention_workspace(None, ctypes.byref(n)) == -1
    assert lib.sengine_amd_cross_attention_workspace(ctypes.byref(_cross()), None) == -1
    call = lib.sengine_amd_cross_attention_ws
    assert call(ctypes.byref(_cross()), P, P, P, None, None, P, P + 4, size, None) == -2
    assert call(ctypes.byref(_cross(Lk=2**30)), P, P, P, None, None, P, P, size, None) == -2
    assert call(None, P, P, P, None, None, P, P, size, None) == -1


@pytest.mark.parametrize("kw", [dict(d=60), dict(Hq=3), dict(type=2)])
def test_cross_attention_with_scratch_memory_refuses(kw):
    call = _lib.load().sengine_amd_cross_attention_ws
    assert call(ctypes.byref(_cross(**kw)), P, P, P, None, None, P, P, 1 << 20, None) == -2
