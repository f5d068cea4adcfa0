"""Token operators on tensors of a device that is not the current one: every launch of a reader makes it so."""
import contextlib

import pytest
import torch

from sparsesnn_amd import ops
from sparsesnn_amd.token_reader import TokenReader, random_reader_params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("four_bit", [False, True])
def test_every_launch_of_a_reader(dev, monkeypatch, four_bit):
    params = random_reader_params(2, embed=64, depth=2, num_classes=20, queries=3, mixer_heads=2)
    reader = TokenReader(params, heads=2, four_bit=four_bit, sections=(8, 8), device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    tokens = torch.randn(2, 30, 64, generator=g, device=dev).half()
    where, here = (torch.arange(n, dtype=torch.int32, device=dev)[:, None].expand(n, 2).contiguous() for n in (30, 3))

    def run():
        return reader.read(reader.encode(tokens, where), positions=here, state=reader.start(2))

    want = run()
    entered, launched = [], []

    @contextlib.contextmanager
    def device(d):
        entered.append(d)
        yield
        assert entered[-1] == d

    lib, load = ops._lib.load(), ops._lib.load
    names = [n for n in ops._lib.SIGNATURES if n.startswith("sengine_amd_") and not n.endswith("_workspace")]

    class Counted:
        def __getattr__(self, name):
            f = getattr(lib, name)
            if name not in names:
                return f

            def call(*args):
                launched.append((name, len(entered)))
                return f(*args)

            return call

    monkeypatch.setattr(ops._lib, "load", lambda: Counted())
    monkeypatch.setattr(ops, "_current_device", lambda: dev.index + 1)
    monkeypatch.setattr(torch.cuda, "device", device)
    got = run()
    monkeypatch.setattr(ops._lib, "load", load)
    assert torch.equal(got, want)
    assert {n.removeprefix("sengine_amd_").removesuffix("_ws") for n, _ in launched} >= {
        "rms_norm", "linear", "cross_attention", "rotary", "decay_attention"}
    # each in a context of its own
    assert [n for _, n in launched] == list(range(1, len(launched) + 1)) and set(entered) == {dev}
