"""What rotary and the linear operator with 4-bit weights refuse, checked on the host (no kernel is launched)."""
import ctypes

import pytest
import torch

from sparsesnn_amd import _lib, ops
from sparsesnn_amd.token_reader import e2m1_groups
from tests.test_token_sizes_host import OnDevice

P = 0x1000  # a pointer that is only compared
S3 = ctypes.c_int64 * 3
F16, E4M3, U8 = torch.float16, torch.float8_e4m3fn, torch.uint8


def _t(*shape, dtype=F16):
    return torch.empty(*shape, dtype=dtype, device="meta").as_subclass(OnDevice)


def _rc(name, desc, *args):
    rc = getattr(_lib.load(), name)(ctypes.byref(desc) if desc is not None else None, *args)
    return rc, _lib.load().sengine_amd_last_error().decode()


def _linear(**kw):
    f = dict(M=4, x_stride=64, weight_stride=32, scale_stride=2, residual_stride=32, out_stride=32, N=32, K=64, group=32,
             in_type=1, out_type=1, bias_type=1, activation=0)
    f.update(kw)
    return _lib.LinearE2m1Desc(**f)


@pytest.mark.parametrize("kw,word", [
    (dict(M=-1), "M"), (dict(N=0), "N"), (dict(K=-2), "K"), (dict(K=63), "even"), (dict(group=16), "groups"),
    (dict(group=0), "groups"), (dict(in_type=2), "fp16"), (dict(in_type=4), "fp16"), (dict(out_type=4), "output"),
    (dict(bias_type=4), "bias"), (dict(activation=5), "activation"), (dict(out_stride=31), "overlap"),
    (dict(M=2**40), "large"), (dict(K=2**30), "large"), (dict(N=2**31 - 1), "large"), (dict(M=2**63 - 1), "large"),
    (dict(M=2**37, N=2**30), "large")])
def test_linear_e2m1_refuses(kw, word):
    rc, text = _rc("sengine_amd_linear_e2m1", _linear(**kw), P, P, P, P, P, P, P, None)
    assert rc == -2 and word in text
    n = ctypes.c_size_t(7)
    if "large" in word:
        assert _lib.load().sengine_amd_linear_e2m1_workspace(ctypes.byref(_linear(**kw)), ctypes.byref(n)) == 0 and n.value == 0


def test_linear_e2m1_null_pointers_no_rows_and_scratch_memory():
    name = "sengine_amd_linear_e2m1"
    assert _rc(name, None, P, P, P, P, P, P, P, None)[0] == -1
    for i in (0, 1, 2, 6):
        args = [P] * 7
        args[i] = None
        assert _rc(name, _linear(), *args, None)[0] == -1
    assert _rc(name, _linear(M=0), *[None] * 8)[0] == 0
    assert _rc(name + "_ws", _linear(), *[P] * 7, P + 8, 100, None)[0] == -2
    lib, n = _lib.load(), ctypes.c_size_t(7)
    size = lambda **kw: (lib.sengine_amd_linear_e2m1_workspace(ctypes.byref(_linear(**kw)), ctypes.byref(n)), n.value)
    assert size() == (0, 0) and size(M=0) == (0, 0) and size(M=3000, K=0) == (0, 0)
    rc, got = size(M=30000, N=100, K=66)
    assert rc == 0 and got >= 100 * 72 * 2
    assert lib.sengine_amd_linear_e2m1_workspace(None, ctypes.byref(n)) == -1
    assert lib.sengine_amd_linear_e2m1_workspace(ctypes.byref(_linear()), None) == -1


def _rotary(**kw):
    d = _lib.RotaryDesc(B=2, L=3, Hq=4, Hk=2, d=48, axes=3, sections=(ctypes.c_int32 * 4)(8, 8, 8, 0), type=1)
    d.q_stride = d.out_q_stride = S3(576, 192, 48)
    d.k_stride = d.out_k_stride = S3(288, 96, 48)
    for k, v in kw.items():
        setattr(d, k, (ctypes.c_int32 * 4)(*v) if k == "sections" else S3(*v) if "stride" in k else v)
    return d


@pytest.mark.parametrize("kw,word", [
    (dict(B=-1), "B"), (dict(L=-1), "L"), (dict(Hq=0), "Hq"), (dict(Hk=-1), "Hk"), (dict(d=0), "d >="), (dict(axes=0), "axes"),
    (dict(axes=5), "axes"), (dict(sections=(8, -8, 8, 0)), "section"), (dict(sections=(8, 8, 9, 0)), "pairs"),
    (dict(sections=(0, 0, 0, 0)), "pairs"), (dict(sections=(2**31 - 1,) * 4, axes=4), "pairs"), (dict(type=4), "fp16"),
    (dict(d=1025), "1024"), (dict(Hq=1365), "65536"), (dict(Hq=2**31 - 1), "65536"),
    (dict(out_q_stride=(576, 192, 47)), "overlap"), (dict(out_k_stride=(0, 96, 48)), "overlap"),
    (dict(out_q_stride=(576, -47, 48)), "overlap")])
def test_rotary_refuses(kw, word):
    rc, text = _rc("sengine_amd_rotary", _rotary(**kw), P, P, P, P, P, P, None)
    assert rc == -2 and word in text


def test_rotary_null_pointers_and_no_tokens():
    assert _rc("sengine_amd_rotary", None, *[P] * 6, None)[0] == -1
    for i in range(6):
        args = [P] * 6
        args[i] = None
        assert _rc("sengine_amd_rotary", _rotary(), *args, None)[0] == -1
    for kw in (dict(B=0), dict(L=0)):
        assert _rc("sengine_amd_rotary", _rotary(**kw), *[None] * 7)[0] == 0
    assert _rc("sengine_amd_rotary", _rotary(B=2**31 - 1, L=2**31 - 1), *[P] * 6, None)[0] == 9  # past 2^32 threads


def _plan(x, w, s, **kw):
    a = dict(row_scale=None, bias=None, activation="none", residual=None, out_dtype=None, out=None)
    a.update(kw)
    return ops._linear_e2m1_plan(None, x, w, s, **a)


def test_linear_e2m1_checks_its_tensors():
    x, w, s = _t(5, 130), _t(40, 65, dtype=U8), _t(40, 5, dtype=E4M3)
    assert _plan(x, w, s)[0]._obj.group == 32
    assert _plan(x, w, _t(40, 3, dtype=E4M3))[0]._obj.group == 64
    assert _plan(x, w, _t(40, 2, dtype=E4M3))[0]._obj.group == 128
    for bad, word in (((_t(5, 130, dtype=torch.float32), w, s), "dtype"), ((x, _t(40, 64, dtype=U8), s), "weight"),
                      ((x, _t(40, 65, dtype=E4M3), s), "weight"), ((x, w, _t(40, 4, dtype=E4M3)), "group_scale"),
                      ((x, w, _t(39, 5, dtype=E4M3)), "group_scale"), ((x, w, _t(40, 5)), "group_scale"),
                      ((torch.empty(5, 130, dtype=F16), w, s), "HIP device"), ((x, w[:, ::2], s), "weight")):
        with pytest.raises(ops.SEngineError, match=word):
            _plan(*bad)
    for kw, word in ((dict(row_scale=_t(40)), "row_scale"), (dict(row_scale=_t(39, dtype=torch.float32)), "row_scale"),
                     (dict(bias=_t(41)), "bias"), (dict(residual=_t(5, 41)), "residual"),
                     (dict(residual=_t(5, 40, dtype=torch.bfloat16)), "residual"), (dict(out_dtype=E4M3), "out_dtype"),
                     (dict(out=_t(5, 40, dtype=torch.bfloat16)), "out")):
        with pytest.raises(ops.SEngineError, match=word):
            _plan(x, w, s, **kw)
    with pytest.raises(ValueError, match="activation"):
        _plan(x, w, s, activation="tanh")
    with pytest.raises(ops.SEngineError, match="N and K"):
        _plan(_t(3, 2**32 + 64), _t(4, 2**31 + 32, dtype=U8), s)


def test_rotary_checks_its_tensors():
    q, k, pos = _t(2, 5, 4, 48), _t(2, 5, 2, 48), _t(2, 5, 3, dtype=torch.int32)
    f = _t(24, dtype=torch.float32)
    plan = lambda *a, out_q=None, out_k=None: ops._rotary_plan(None, *a, False, out_q, out_k)
    assert plan(q, k, pos, f, (8, 8, 8)) and plan(q, None, _t(5, 3, dtype=torch.float32), f, (8, 8, 8))
    for args, word in (
            ((q, _t(2, 5, 2, 40), pos, f, (8, 8, 8)), "k:"), ((q, _t(2, 4, 2, 48), pos, f, (8, 8, 8)), "k:"),
            ((q[0], k, pos, f, (8, 8, 8)), "q:"), ((q, k, _t(2, 5, 2, dtype=torch.int32), f, (8, 8, 8)), "positions"),
            ((q, k, _t(2, 5, 3, dtype=torch.int64), f, (8, 8, 8)), "positions"), ((q, k, pos, f, ()), "sections"),
            ((q, k, pos, f, (8, 8, 4, 2, 2)), "sections"), ((q, k, pos, f, (8, 8.0, 8)), "sections"),
            ((q, k, pos, f, (8, 8, -1)), "sections"), ((q, k, pos, _t(23, dtype=torch.float32), (8, 8, 8)), "frequencies"),
            ((q, k, pos, _t(24), (8, 8, 8)), "frequencies"), ((q.transpose(2, 3), None, pos, f, (1, 1, 0)), "frequencies"),
            ((_t(2, 5, 48, 4).transpose(2, 3), None, pos, f, (8, 8, 8)), "side by side"),
            ((q, k, _t(3, 2, 5, dtype=torch.int32).permute(1, 2, 0), f, (8, 8, 8)), "positions")):
        with pytest.raises(ops.SEngineError, match=word):
            plan(*args)
    with pytest.raises(ops.SEngineError, match="out_k"):
        plan(q, None, pos, f, (8, 8, 8), out_k=k)
    with pytest.raises(ops.SEngineError, match="out_q"):
        plan(q, k, pos, f, (8, 8, 8), out_q=k)
    with pytest.raises(ops.SEngineError, match="2\\*\\*31"):
        plan(_t(2**31, 1, 1, 48), None, _t(1, 3, dtype=torch.int32), f, (8, 8, 8))


def test_quantizer_refuses():
    for w, g in ((torch.zeros(3, 5), 32), (torch.zeros(3), 32), (torch.zeros(3, 4), 16)):
        with pytest.raises(ops.SEngineError, match="e2m1_groups"):
            e2m1_groups(w, g)
