"""What the token operators refuse, checked on the host: the C entries' descriptors, and the torch
wrappers' tensors (no kernel is launched here)."""
import ctypes

import pytest
import torch

from sparsesnn_amd import _lib, ops

P = 0x1000  # a pointer that is only compared with null


def _rc(name, desc, *args):
    rc = getattr(_lib.load(), name)(ctypes.byref(desc) if desc is not None else None, *args)
    return rc, _lib.load().sengine_amd_last_error().decode()


def _norm(**kw):
    f = dict(rows=4, x_stride=384, residual_stride=384, out_stride=384, stream_stride=384, D=384, in_type=1,
             weight_type=1, out_type=1, eps=1e-6)
    f.update(kw)
    return _lib.RmsNormDesc(**f)


@pytest.mark.parametrize("kw,word", [
    (dict(D=0), "D"), (dict(D=32769), "D"), (dict(rows=-1), "rows"), (dict(rows=2**31), "rows"),
    (dict(in_type=0), "fp16"), (dict(in_type=4), "fp16"), (dict(out_type=2), "x's type"),
    (dict(weight_type=3), "weight"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(out_stride=383), "overlap"), (dict(stream_stride=0), "overlap"), (dict(out_type=4), "scale")])
def test_rms_norm_refuses(kw, word):
    rc, text = _rc("sengine_amd_rms_norm", _norm(**kw), P, P, P, P, P, None, None)
    assert rc < 0 and word in text


def test_rms_norm_null_pointers_and_no_rows():
    assert _rc("sengine_amd_rms_norm", None, P, P, P, P, P, P, None)[0] == -1
    assert _rc("sengine_amd_rms_norm", _norm(), None, P, P, P, P, P, None)[0] == -1
    assert _rc("sengine_amd_rms_norm", _norm(), P, P, P, None, P, P, None)[0] == -1
    assert _rc("sengine_amd_rms_norm", _norm(rows=0), None, None, None, None, None, None, None)[0] == 0


def _linear(**kw):
    f = dict(M=4, x_stride=64, weight_stride=64, residual_stride=32, out_stride=32, N=32, K=64, in_type=1, out_type=1,
             bias_type=1, activation=0)
    f.update(kw)
    return _lib.LinearDesc(**f)


@pytest.mark.parametrize("kw,word", [
    (dict(M=-1), "M"), (dict(N=0), "N"), (dict(K=-1), "K"), (dict(in_type=2), "e4m3"), (dict(in_type=0), "e4m3"),
    (dict(out_type=4), "output"), (dict(out_type=0), "output"), (dict(bias_type=4), "bias"),
    (dict(activation=5), "activation"), (dict(activation=-1), "activation"), (dict(out_stride=31), "overlap"),
    (dict(M=2**40), "large"), (dict(K=2**30), "large")])
def test_linear_refuses(kw, word):
    rc, text = _rc("sengine_amd_linear", _linear(**kw), P, P, None, None, P, P, P, None)
    assert rc < 0 and word in text


def test_linear_null_pointers_scales_and_no_rows():
    assert _rc("sengine_amd_linear", None, P, P, None, None, P, P, P, None)[0] == -1
    assert _rc("sengine_amd_linear", _linear(), None, P, None, None, P, P, P, None)[0] == -1
    assert _rc("sengine_amd_linear", _linear(), P, None, None, None, P, P, P, None)[0] == -1
    assert _rc("sengine_amd_linear", _linear(), P, P, None, None, P, P, None, None)[0] == -1
    assert _rc("sengine_amd_linear", _linear(), P, P, P, None, P, P, P, None)[0] == -2
    assert _rc("sengine_amd_linear", _linear(M=0), None, None, None, None, None, None, None, None)[0] == 0


def _cross(**kw):
    f = dict(B=2, Lq=3, Lk=5, Hq=4, Hkv=2, d=64, type=1, scale=0.1)
    f.update(kw)
    return _lib.CrossDesc(**f)


@pytest.mark.parametrize("kw,word", [
    (dict(B=-1), "B"), (dict(Lq=-1), "Lq"), (dict(Lk=-1), "Lk"), (dict(Hq=0), "heads"), (dict(Hkv=0), "heads"),
    (dict(Hkv=3), "multiple"), (dict(d=0), "head size"), (dict(d=12), "head size"), (dict(d=136), "head size"),
    (dict(type=2), "fp16"), (dict(type=4), "fp16"), (dict(B=2**20, Lq=2**10), "too many")])
def test_cross_attention_refuses(kw, word):
    rc, text = _rc("sengine_amd_cross_attention", _cross(**kw), P, P, P, None, None, P, None)
    assert rc < 0 and word in text


def test_cross_attention_null_pointers_and_no_queries():
    name = "sengine_amd_cross_attention"
    assert _rc(name, None, P, P, P, None, None, P, None)[0] == -1
    for at in (0, 1, 2, 5):
        args = [P, P, P, None, None, P, None]
        args[at] = None
        assert _rc(name, _cross(), *args)[0] == -1
    assert _rc(name, _cross(B=0), *[None] * 7)[0] == 0
    assert _rc(name, _cross(Lq=0), *[None] * 7)[0] == 0


def test_wrappers_refuse_host_tensors_and_others():
    x = torch.zeros(4, 64, dtype=torch.float16)
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    for call in (lambda: ops.rms_norm(x), lambda: ops.linear(x, x), lambda: ops.cross_attention(q, q, q)):
        with pytest.raises(ops.SEngineError, match="HIP device"):
            call()
    for call in (lambda: ops.rms_norm(3), lambda: ops.linear([1], x), lambda: ops.cross_attention(None, q, q)):
        with pytest.raises(TypeError):
            call()


def test_rows_of_a_strided_tensor():
    t = torch.zeros(4, 6, 32)
    assert ops._token_rows(t, "t") == (24, 32)
    assert ops._token_rows(t[:, :, :8], "t") == (24, 32)
    assert ops._token_rows(t[:, :1, :8], "t") == (4, 192)
    assert ops._token_rows(t[:1, :1, :8], "t")[0] == 1
    assert ops._token_rows(t[0, :1].expand(5, 32), "t") == (5, 0)
    for bad in (t[:, :3], t.transpose(0, 1), t[..., ::2], t.transpose(1, 2)):
        with pytest.raises(ops.SEngineError):
            ops._token_rows(bad, "t")
