"""What a reader makes by itself has its own types, whatever torch's default type is."""
import contextlib

import pytest
import torch

from sparsesnn_amd.token_reader import TokenReader, e2m1_groups, random_reader_params


@contextlib.contextmanager
def _default(dtype):
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        yield
    finally:
        torch.set_default_dtype(before)


@pytest.mark.parametrize("default", [torch.float64, torch.float16])
def test_states(default):
    params = random_reader_params(embed=64, depth=2, mixer_heads=2)
    reader = TokenReader(params, heads=2, device="cpu")
    with _default(default):
        state = reader.start(3)
    assert [(s.dtype, tuple(s.shape)) for s in state] == [(torch.float32, (3, 2, 32, 32))] * 2


@pytest.mark.parametrize("default", [torch.float64, torch.float16])
@pytest.mark.parametrize("K", [0, 130])
def test_weights_in_four_bits(default, K):
    w = torch.randn(9, K, generator=torch.Generator().manual_seed(1))
    want = e2m1_groups(w)
    with _default(default):
        got = e2m1_groups(w)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("default", [torch.float64, torch.float16])
def test_readers(default):
    params = random_reader_params(embed=64, depth=1, mixer_heads=2)
    make = lambda four: TokenReader(params, heads=2, device="cpu", four_bit=four, sections=(8, 0, 5))
    for four in (False, True):
        want = make(four)
        with _default(default):
            got = make(four)
        assert got.frequencies.dtype == torch.float32 and torch.equal(got.frequencies, want.frequencies)
        assert got.decay[0].dtype == torch.float32 and torch.equal(got.decay[0], want.decay[0])
        for k in want.four:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got.four[k], want.four[k]))
