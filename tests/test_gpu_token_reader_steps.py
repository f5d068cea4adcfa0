"""TokenReader step by step: every operator's result on the way against its formula on what the network has there."""
import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import token_reader as tr
from tests.test_gpu_token_ops import _check_norm, _within

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Lq,N", [(1, 196), (64, 300)])
def test_every_step(dev, monkeypatch, eight_bit, dtype, Lq, N):
    """What each operator gives on the way is within the oracle's bounds of its formula on the tensors and weights that
    the network has at that place: a bias left out or a wrong scale of one row does not pass."""
    given = []

    def recorded(name):
        f = getattr(tr.ops, name)

        def call(*args, **kw):
            out = f(*args, **kw)
            given.append((name, [None if t is None else t.clone() for t in (out if isinstance(out, tuple) else (out,))]))
            return out

        monkeypatch.setattr(tr.ops, name, call)

    params = tr.random_reader_params(1, embed=96, depth=2, num_classes=70, queries=Lq)
    reader = tr.TokenReader(params, heads=2, dtype=dtype, eight_bit=eight_bit, device=dev)
    p = {k: v.to(dev, dtype) for k, v in params.items()}
    g = torch.Generator(device=dev).manual_seed(Lq)
    tokens = torch.randint(0, 6, (3, N, 96), generator=g, device=dev).to(dtype)
    mask = torch.rand(3, N, generator=g, device=dev) > 0.2
    for name in ("rms_norm", "linear", "cross_attention"):
        recorded(name)
    logits = reader.read(reader.encode(tokens), key_mask=mask)
    steps = iter(given)

    def norm(x, weight, residual=None, out_dtype=None):
        name, got = next(steps)
        assert name == "rms_norm"
        _check_norm(x, p[weight + ".weight"], residual, 1e-6, out_dtype, got)
        return got

    def linear(x, layer, act="none", residual=None, scale=None, out_dtype=dtype):
        name, (got,) = next(steps)
        assert name == "linear" and got.dtype == out_dtype
        w, ws = p[layer + ".weight"], None
        if scale is not None:
            w = params[layer + ".weight"].to(dev)
            ws = w.abs().amax(-1) / 448
            w = (w / ws[:, None]).to(torch.float8_e4m3fn)
        _within(got, *ref.linear(x, w, p[layer + ".bias"], act, residual, scale, ws, out_dtype))
        return got

    kv = []
    for i in range(2):
        y = norm(tokens, f"block.{i}.norm_kv")[0]
        kv.append(linear(y, f"block.{i}.kv").view(3, N, 2, 2, 48))
    x = p["queries"].expand(3, -1, -1)
    for i in range(2):
        pre = f"block.{i}."
        q = linear(norm(x, pre + "norm1")[0], pre + "q").view(3, Lq, 2, 48)
        name, (o,) = next(steps)
        assert name == "cross_attention"
        _within(o, *ref.cross_attention(q, kv[i][:, :, 0], kv[i][:, :, 1], None, None, mask))
        a = linear(o.view(3, Lq, 96), pre + "out")
        y, x, *scale = norm(a, pre + "norm2", x, torch.float8_e4m3fn if eight_bit else None)
        h = linear(y, pre + "fc1", "gelu", scale=scale[0] if eight_bit else None)
        x = linear(h, pre + "fc2", residual=x)
    want = linear(norm(x, "norm")[0], "head", out_dtype=torch.float32)
    assert next(steps, None) is None and torch.equal(logits, want)
