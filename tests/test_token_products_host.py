"""Sizes whose products pass 64 bits (on the host): refused by the entries, and no scratch memory is asked for.  In a
process of their own, which a division by zero would end."""
import subprocess
import sys

import pytest

CODE = """
import ctypes, sys
from sparsesnn_amd import _lib

lib, n, P = _lib.load(), ctypes.c_size_t(7), 0x1000
kind, sizes = sys.argv[1], dict(a.split("=") for a in sys.argv[2:])
sizes = {k: int(v) for k, v in sizes.items()}
if kind == "linear":
    d = _lib.LinearDesc(**{**dict(M=3, x_stride=8192, weight_stride=8192, residual_stride=0, out_stride=2**31 - 1, N=64,
                                  K=8192, in_type=3, out_type=3, bias_type=0, activation=0), **sizes})
    rc = lib.sengine_amd_linear(ctypes.byref(d), P, P, None, None, None, None, P, None)
    rw = lib.sengine_amd_linear_workspace(ctypes.byref(d), ctypes.byref(n))
else:
    d = _lib.CrossDesc(**{**dict(B=1, Lq=1, Lk=2000, Hq=4, Hkv=4, d=64, type=1, scale=0.1), **sizes})
    rc = lib.sengine_amd_cross_attention(ctypes.byref(d), P, P, P, None, None, P, None)
    rw = lib.sengine_amd_cross_attention_workspace(ctypes.byref(d), ctypes.byref(n))
print(rc, rw, n.value)
"""


@pytest.mark.parametrize("kind,sizes", [
    ("linear", dict(M=2**62, N=2**20)), ("linear", dict(M=2**62, N=2**20, K=8191)), ("linear", dict(M=2**63 - 1)),
    ("linear", dict(N=2**31 - 1)), ("linear", dict(N=2**31 - 255, K=8191)), ("linear", dict(M=2**37, N=64)),
    ("cross", dict(B=2**30, Lq=2**30, Hq=2**20, Hkv=2**20)), ("cross", dict(B=2**30, Lq=2**30, Hq=16, Hkv=16)),
    ("cross", dict(B=2**31 - 1, Lq=2**31 - 1, Hq=2**31 - 1, Hkv=1)), ("cross", dict(Lk=2**30)), ("cross", dict(d=136))])
def test_refused(kind, sizes):
    done = subprocess.run([sys.executable, "-c", CODE, kind, *(f"{k}={v}" for k, v in sizes.items())],
                          capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    assert done.stdout.split() == ["-2", "0", "0"]
