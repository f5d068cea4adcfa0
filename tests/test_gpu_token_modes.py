"""Forward-mode differentiation and tracing: the token operators would leave out a tangent, or a recording would leave
out the operator, so they refuse."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _linear_case, _qkv, _randn

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _calls(dev):
    g = _gen(dev, 1)
    x, w, _, _ = _linear_case(g, 20, 32, 64, F16)
    norm_w = _randn(g, 64, dtype=F16)
    q, k, v = _qkv(g, 1, 3, 40, 2, 2, 32, F16)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return [(lambda *t: ops.rms_norm(*t), (x, norm_w, x.clone())),
            (lambda a, b, c, r: ops.linear(a, b, c, residual=r), (x, w, _randn(g, 32, dtype=F16), x[:, :32].contiguous())),
            (lambda *t: ops.cross_attention(*t), (q, k, v))]


def test_a_tangent_is_refused(dev):
    for f, args in _calls(dev):
        want = f(*args)
        with fwd.dual_level():
            for i in range(len(args)):
                dual = [*args]
                dual[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                for _ in range(2):
                    with pytest.raises(ops.SEngineError, match="tangent"):
                        f(*dual)
            got = f(*args)  # no tangent: as ever
        pair = lambda t: t if isinstance(t, tuple) else (t,)
        assert all(torch.equal(a, b) for a, b in zip(pair(got), pair(want)))


def test_a_recording_is_refused(dev):
    for f, args in _calls(dev):
        f(*args)
        with pytest.raises(ops.SEngineError, match="record"):
            torch.jit.trace(f, args, check_trace=False)
        with pytest.raises(ops.SEngineError, match="record"):
            make_fx(f)(*args)
        f(*args)
