"""Rotary positions against their definition in 64 bits: sections, orders of the pairs, types, piece sizes, strides, far
positions, outputs in place."""
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops
from tests.test_gpu_token_ops import _gen, _randn, _within

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _freq(dev, sections):
    return torch.cat([10000.0 ** -(torch.arange(n) / max(n, 1)) for n in sections]).float().to(dev)


def _check(x, got, positions, freq, sections, interleaved):
    assert got.dtype == x.dtype and got.shape == x.shape
    _within(got, *ref.rotary(x, positions, freq, sections, interleaved))


@pytest.mark.parametrize("d,sections", [
    (2, (1,)), (5, (2,)), (16, (8,)), (16, (3, 5)), (48, (8, 8, 8)), (48, (4, 0, 8)), (40, (20,)), (40, (5, 5)),
    (80, (7, 13, 20)), (128, (16, 24, 24)), (128, (16, 8, 4, 4)), (130, (65,)), (97, (1, 2, 3)), (1024, (512,))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rotary(dev, d, sections, interleaved, dtype):
    g = _gen(dev, d + sum(sections))
    freq = _freq(dev, sections)
    for B, L, Hq, Hk in ((1, 1, 1, 1), (2, 37, 3, 1), (3, 700, 2, 2)):
        qkv = _randn(g, B, L, Hq + 2 * Hk, d, dtype=dtype)
        q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
        pos = torch.randint(0, 3000, (B, L, len(sections)), generator=g, device=dev, dtype=torch.int32)
        yq, yk = ops.rotary(q, k, pos, freq, sections, interleaved)
        _check(q, yq, pos, freq, sections, interleaved)
        _check(k, yk, pos, freq, sections, interleaved)
        alone, none = ops.rotary(q, None, pos, freq, list(sections), interleaved)
        assert none is None and torch.equal(alone, yq)


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions(dev, interleaved):
    """Far, negative, fractional and shared positions; positions with strides."""
    g = _gen(dev, 1)
    q, k = _randn(g, 2, 50, 2, 48, dtype=F32), _randn(g, 2, 50, 1, 48, dtype=F32)
    freq, sections = _freq(dev, (8, 8, 8)), (8, 8, 8)
    far = torch.randint(-2**31, 2**31 - 1, (2, 50, 3), generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    far[0, :3] = torch.tensor([2**31 - 1, -2**31, 0], dtype=torch.int32, device=dev)
    real = torch.randn(2, 50, 3, generator=g, device=dev) * 1e4
    wide = torch.randint(0, 99, (2, 100, 5), generator=g, device=dev, dtype=torch.int32)
    for pos in (far, real, wide[:, ::2, 1:4], real[0], wide[1, ::2, :3]):
        for x, y in zip((q, k), ops.rotary(q, k, pos, freq, sections, interleaved)):
            _check(x, y, pos, freq, sections, interleaved)
    one = torch.arange(50, dtype=torch.int32, device=dev)
    for pos in (one[:, None], one[None, :, None].expand(2, 50, 1)):
        y, _ = ops.rotary(q, None, pos, freq, (24,), interleaved)
        _check(q, y, one[:, None], freq, (24,), interleaved)
    still, _ = ops.rotary(q, None, torch.zeros_like(far), freq, sections, interleaved)
    assert torch.equal(still, q)


@pytest.mark.parametrize("d,pairs", [(48, 24), (48, 16), (44, 11), (37, 18)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_in_place(dev, d, pairs, interleaved):
    g = _gen(dev, d)
    B, L, H = 2, 33, 3
    freq = _freq(dev, (pairs,))
    pos = torch.randint(0, 100, (B, L, 1), generator=g, device=dev, dtype=torch.int32)
    wide = _randn(g, B, L, H, d + 7, dtype=F16)
    heads_first = _randn(g, B, H, L, d, dtype=F16).transpose(1, 2)
    odd = wide[..., 3:3 + d]
    for q in (odd, heads_first, odd[:, :, :1].expand(B, L, H, d), odd[:1].expand(B, L, H, d)):
        y, yk = ops.rotary(q, heads_first, pos, freq, (pairs,), interleaved)
        _check(q, y, pos, freq, (pairs,), interleaved)
        _check(heads_first, yk, pos, freq, (pairs,), interleaved)
    want, want_k = ops.rotary(odd, heads_first, pos, freq, (pairs,), interleaved)
    outer = torch.full((B, L, H, d + 7), 5.0, dtype=F16, device=dev)
    into = outer[..., 3:3 + d]
    got, _ = ops.rotary(odd, None, pos, freq, (pairs,), interleaved, out_q=into)
    assert got is into and torch.equal(into, want) and (outer[..., :3] == 5).all() and (outer[..., 3 + d:] == 5).all()
    before, k = wide.clone(), heads_first.clone(memory_format=torch.preserve_format)
    got, got_k = ops.rotary(odd, k, pos, freq, (pairs,), interleaved, out_q=odd, out_k=k)
    assert torch.equal(got, want) and torch.equal(got_k, want_k)
    assert torch.equal(wide[..., :3], before[..., :3]) and torch.equal(wide[..., 3 + d:], before[..., 3 + d:])
    y, yk = ops.rotary(before[..., 3:3 + d], k.copy_(heads_first), pos, freq, (pairs,), interleaved, out_k=k)
    assert torch.equal(y, want) and torch.equal(yk, want_k)


def test_nothing_to_turn_and_not_numbers(dev):
    freq = _freq(dev, (8,))
    for shape in ((0, 4, 2, 16), (3, 0, 2, 16)):
        q = torch.empty(shape, dtype=F16, device=dev)
        y, yk = ops.rotary(q, q, torch.zeros(*shape[:2], 1, dtype=torch.int32, device=dev), freq, (8,))
        assert y.shape == shape and yk.shape == shape
    q = torch.ones(1, 3, 2, 20, dtype=F16, device=dev)
    q[0, 1, 0, 2] = math.nan
    q[0, 1, 1, 19] = math.inf
    pos = torch.ones(1, 3, 1, dtype=F32, device=dev)
    pos[0, 2] = math.nan
    y, _ = ops.rotary(q, None, pos, freq, (8,))
    assert y[0, 2, :, :16].isnan().all() and (y[0, 2, :, 16:] == 1).all()  # a turn by no number
    bad = y[0, 1].isnan()
    assert bad[0, 2] and bad[0, 10] and int(bad.sum()) == 2 and y[0, 1, 1, 19] == math.inf
    assert y[0, 0].isfinite().all()


def test_many_tokens(dev):
    """More tokens than a workgroup takes of the largest grids, and the last workgroup's few."""
    g = _gen(dev, 2)
    q = _randn(g, 1, 70_001, 1, 16, dtype=F16)
    pos = torch.arange(70_001, dtype=torch.int32, device=dev)[None, :, None]
    freq = _freq(dev, (8,))
    _check(q, ops.rotary(q, None, pos, freq, (8,))[0], pos, freq, (8,), False)
