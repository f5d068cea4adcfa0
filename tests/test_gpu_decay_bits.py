"""Decaying linear attention keeps its state's 32 bits: where only early tokens are left in the last state, and where an
output is the difference of state values that almost cancel."""
import pytest
import torch

from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _randn

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
U = 2.0**-24


@pytest.mark.parametrize("B,H,L,dk,dv", [(1, 4, 384, 16, 128), (2, 3, 200, 64, 48), (1, 4, 1500, 128, 64),
                                         (8, 40, 300, 32, 256)])
@pytest.mark.parametrize("back", [130, 190])
def test_a_state_of_early_tokens(dev, B, H, L, dk, dv, back):
    """One token that counts, `back` tokens before the end: every value of the last state is a single product k v g^back."""
    g = _gen(dev, L + back)
    k, v = torch.zeros(B, L, H, dk, dtype=BF16, device=dev), _randn(g, B, L, H, dv, dtype=BF16)
    at = L - 1 - back
    k[:, at] = _randn(g, B, H, dk, dtype=BF16)
    decay = torch.exp2(-torch.rand(H, generator=g, device=dev) * 0.09 - 0.035)
    _, s = ops.decay_attention(torch.zeros_like(k), k, v, decay)
    age = decay.double() ** back
    want = k[:, at].double()[..., :, None] * v[:, at].double()[..., None, :] * age[:, None, None]
    # Products of 16-bit values are exact.  The power of the decay is a product of one a chunk of 64 tokens, of which
    # each is off by a unit (2 U) and its exponent by a unit of the logarithm, 2 U, and a product's U of itself, and each
    # is rounded when it is multiplied; the product with v rounds once, and its three parts are added in 24 bits, each
    # sum off by 2 U at the most.
    powers = 2 + back // 64
    rel = 3 * U * back * -torch.log(decay.double()) + powers * 3 * U + U + 3 * 2 * U
    assert float(rel.max()) < 2.0**-17  # what two parts of eight bits leave out of some values
    assert ((s.double() - want).abs() <= want.abs() * rel[:, None, None]).all()


@pytest.mark.parametrize("L,H,dk,dv", [(64, 2, 16, 128), (100, 3, 64, 48), (130, 2, 128, 64), (64, 70, 32, 256)])
def test_outputs_of_states_that_almost_cancel(dev, L, H, dk, dv):
    """q takes the difference of two rows of the state that are 2^-15 apart, and no key counts."""
    g = _gen(dev, L + dv)
    q, k, v = (torch.zeros(1, L, H, n, dtype=BF16, device=dev) for n in (dk, dk, dv))
    q[..., 3], q[..., dk - 2] = 1.0, -1.0
    state = _randn(g, 1, H, dk, dv)
    state[:, :, dk - 2] = state[:, :, 3] * (1 + (1 + torch.rand(1, H, dv, generator=g, device=dev)) * 2.0**-15)
    o, s = ops.decay_attention(q, k, v, torch.ones(H, device=dev), state=state, scale=1.0)
    assert torch.equal(s, state)
    big = state[:, :, 3].double().abs()
    want = state[:, :, 3].double() - state[:, :, dk - 2].double()
    # a value is three parts of eight bits; the six are added in 24 bits, each sum off by 2 U of it at the most, and the
    # output rounds by 2^-8 of itself at the most
    bound = big * (6 * 2 * U) + want.abs() * (2.0**-8 + 4 * U)
    assert ((o.double() - want[:, None]).abs() <= bound[:, None]).all()


@pytest.mark.parametrize("L,H,dk,dv", [(64, 40, 16, 48), (50, 8, 64, 128), (30, 300, 32, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, BF16])
def test_weights_within_a_chunk_that_almost_cancel(dev, L, H, dk, dv, dtype):
    """Two tokens whose weighted values are alike but for their sign and last bits: every part of both counts."""
    g = _gen(dev, L + H)
    q, k, v = (torch.zeros(1, L, H, n, dtype=dtype, device=dev) for n in (dk, dk, dv))
    a = 1 + torch.rand(H, generator=g, device=dev).to(dtype)
    q[..., 2], q[..., dk - 1] = 1.0, a
    k[:, 1, :, 2], k[:, 6, :, dk - 1] = 1.0, 1.0
    v[:, 6] = _randn(g, 1, H, dv, dtype=dtype)
    v[:, 1] = (-a.double()[:, None] * v[:, 6].double()).to(dtype)
    o, _ = ops.decay_attention(q, k, v, torch.ones(H, device=dev), scale=1024.0)
    size = (a.double()[:, None] * v[:, 6].double()).abs() * 1024
    want = (v[:, 1].double() + a.double()[:, None] * v[:, 6].double()) * 1024
    # the weights, 1 and a, have 11 bits at the most: their parts are exact, as are those of the values; up to eight products
    # of parts are added in 24 bits, each sum off by 2 U of up to twice the size; an output rounds by half a step
    step = torch.finfo(dtype).eps / 2
    bound = size * (8 * 2 * 2 * U) + want.abs() * (step + 4 * U) + torch.finfo(dtype).smallest_normal * step
    assert ((o[:, 6:].double() - want[:, None]).abs() <= bound[:, None]).all()
