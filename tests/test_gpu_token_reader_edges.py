"""TokenReader of parameters that require gradients, and of nothing."""
import pytest
import torch

from sparsesnn_amd import token_reader as tr

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("eight_bit", [False, True])
def test_parameters_that_require_gradients(dev, eight_bit):
    p = tr.random_reader_params(3, embed=64, depth=2, num_classes=10, queries=2)
    tokens = torch.randint(0, 6, (2, 50, 64), device=dev).to(F16)
    want = tr.TokenReader(p, heads=4, eight_bit=eight_bit, device=dev)
    got = tr.TokenReader({k: torch.nn.Parameter(v) for k, v in p.items()}, heads=4, eight_bit=eight_bit, device=dev)
    assert torch.equal(got.read(got.encode(tokens)), want.read(want.encode(tokens)))


@pytest.mark.parametrize("eight_bit", [False, True])
def test_no_sequences_no_queries_no_tokens(dev, eight_bit):
    p = tr.random_reader_params(4, embed=64, depth=2, num_classes=10, queries=3)
    reader = tr.TokenReader(p, heads=4, eight_bit=eight_bit, device=dev)
    none = reader.encode(torch.zeros(0, 50, 64, dtype=F16, device=dev))
    assert reader.read(none).shape == (0, 3, 10)
    some = reader.encode(torch.ones(2, 50, 64, dtype=F16, device=dev))
    assert reader.read(some, torch.zeros(2, 0, 64, dtype=F16, device=dev)).shape == (2, 0, 10)
    empty = reader.encode(torch.zeros(2, 0, 64, dtype=F16, device=dev))
    got = reader.read(empty)
    nothing = torch.zeros(2, dtype=torch.int32, device=dev)  # the same as tokens that do not count
    assert got.isfinite().all() and torch.equal(got, reader.read(some, key_lengths=nothing))
