"""What decaying linear attention refuses and which scratch memory it asks for, checked on the host (no kernel is
launched)."""
import ctypes

import pytest
import torch

from sparsesnn_amd import _lib, ops
from tests.test_linear_e2m1_host import OnDevice, _rc, _t

P = 0x1000
S3, S2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
F16, F32, I32 = torch.float16, torch.float32, torch.int32


def _desc(**kw):
    f = dict(B=2, L=300, H=4, dk=64, dv=48, type=1, scale=0.1)
    f.update({k: v for k, v in kw.items() if "stride" not in k})
    d = _lib.DecayDesc(**f)
    B, L, H, dk, dv = (max(f[k], 1) for k in ("B", "L", "H", "dk", "dv"))
    d.q_stride = d.k_stride = S3(L * H * dk, H * dk, dk)
    d.v_stride = d.out_stride = S3(L * H * dv, H * dv, dv)
    d.state_stride = d.state_out_stride = S2(H * dk * dv, dk * dv)
    for k, v in kw.items():
        if "stride" in k:
            setattr(d, k, (S2 if "state" in k else S3)(*v))
    return d


@pytest.mark.parametrize("kw,word", [
    (dict(B=-1), "B"), (dict(L=-1), "L"), (dict(H=0), "H"), (dict(dk=4), "dk"), (dict(dk=60), "dk"), (dict(dk=136), "dk"),
    (dict(dv=12), "dv"), (dict(dv=264), "dv"), (dict(type=2), "fp16"), (dict(type=4), "fp16"), (dict(L=2**31 - 1), "large"),
    (dict(B=2**30, H=2), "large"), (dict(out_stride=(300 * 192, 192, 40)), "overlap"),
    (dict(out_stride=(0, 192, 48)), "overlap"), (dict(out_stride=(300 * 192, 0, 48)), "overlap"),
    (dict(state_out_stride=(0, 64 * 48)), "overlap"), (dict(state_out_stride=(4 * 64 * 48, 64 * 40)), "overlap"),
    (dict(q_stride=(300 * 256, 257, 64)), "16 bytes"), (dict(v_stride=(300 * 192, 192, 52)), "16 bytes"),
    (dict(state_stride=(4 * 64 * 48, 64 * 48 + 2)), "16 bytes")])
def test_refuses(kw, word):
    rc, text = _rc("sengine_amd_decay_attention", _desc(**kw), P, P, P, P, P, P, P, P, None)
    assert rc == -2 and word in text


def test_null_pointers_alignment_and_nothing_to_do():
    name = "sengine_amd_decay_attention"
    assert _rc(name, None, *[P] * 8, None)[0] == -1
    for i in (0, 1, 2, 3, 6):  # state, lengths and the last state may be absent
        args = [P] * 8
        args[i] = None
        assert _rc(name, _desc(), *args, None)[0] == -1
    for i in (0, 1, 2, 4, 6, 7):
        args = [P] * 8
        args[i] = P + 8
        assert _rc(name, _desc(), *args, None)[0] == -2
    assert _rc(name, _desc(B=0), *[None] * 9)[0] == 0
    assert _rc(name + "_ws", _desc(), *[P] * 8, P + 8, 100, None)[0] == -2
    assert _rc(name, _desc(B=2**22, H=256, L=4), *[P] * 8, None)[0] == 9  # past 2^32 threads
    assert _rc(name, _desc(B=2**22, H=256, L=40), *[P] * 8, None)[0] == 9


def test_scratch_memory():
    lib, n = _lib.load(), ctypes.c_size_t(7)

    def size(**kw):
        assert lib.sengine_amd_decay_attention_workspace(ctypes.byref(_desc(**kw)), ctypes.byref(n)) == 0
        return n.value

    assert size(B=1, H=2, L=20000) > 0 and size(B=1, H=2, L=20000) % (2 * 64 * 48 * 4) == 0
    # one token, few tokens, many heads, nothing to do, refused
    for kw in (dict(L=1), dict(L=100), dict(B=512, H=16, L=20000), dict(L=0), dict(B=0), dict(dk=60), dict(L=-5),
               dict(B=2**30, H=2**30, L=20000)):
        assert size(**kw) == 0
    assert lib.sengine_amd_decay_attention_workspace(None, ctypes.byref(n)) == -1
    assert lib.sengine_amd_decay_attention_workspace(ctypes.byref(_desc()), None) == -1


def test_checks_its_tensors():
    q, v, g = _t(2, 5, 4, 64), _t(2, 5, 4, 48), _t(4, dtype=F32)
    s, n = _t(2, 4, 64, 48, dtype=F32), _t(2, dtype=I32)

    def plan(q=q, k=q, v=v, g=g, state=None, lengths=None, out=None, state_out=None):
        return ops._decay_plan(None, q, k, v, g, state, lengths, None, out, state_out)

    assert plan(state=s, lengths=n, out=v, state_out=s)[1:3] == (0, (2, 4, 64, 48))
    for kw, word in (
            (dict(q=_t(2, 5, 4, 64, dtype=F32)), "dtype"), (dict(k=_t(2, 5, 4, 64, dtype=torch.bfloat16)), "k:"),
            (dict(k=_t(2, 6, 4, 64)), "decay_attention"), (dict(v=_t(2, 5, 3, 48)), "decay_attention"),
            (dict(v=_t(2, 5, 48)), "decay_attention"), (dict(g=_t(4)), "decay"), (dict(g=_t(5, dtype=F32)), "decay"),
            (dict(lengths=_t(3, dtype=I32)), "lengths"), (dict(lengths=_t(2, dtype=torch.int64)), "lengths"),
            (dict(state=_t(2, 4, 64, 48)), "state"), (dict(state=_t(2, 4, 48, 64, dtype=F32)), "state"),
            (dict(state=_t(2, 4, 48, 64, dtype=F32).transpose(2, 3)), "contiguous"),
            (dict(state_out=_t(2, 4, 64, 56, dtype=F32)[..., :48]), "contiguous"), (dict(out=_t(2, 5, 4, 64)), "out"),
            (dict(v=_t(2, 5, 4, 52)[..., :48]), "16 bytes"), (dict(q=_t(2, 4, 64, 5).permute(0, 3, 1, 2)), "side by side"),
            (dict(q=torch.empty(2, 5, 4, 64, dtype=F16)), "HIP device")):
        with pytest.raises(ops.SEngineError, match=word):
            plan(**kw)
    big = _t(1, 2**31, 1, 64)
    with pytest.raises(ops.SEngineError, match="2\\*\\*31"):
        plan(q=big, k=big, v=big, g=_t(1, dtype=F32))
    assert isinstance(q, OnDevice)
