"""Cross attention's kernels at sizes that reach each of them: rows of a group on one wave or many, neighbouring heads
copied as one row, keys in parts, masks longer than one list, and the kernel for any layout."""
import ctypes
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import _lib, ops
from tests.test_gpu_token_ops import _gen, _qkv, _within

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,d", [
    (1, 1, 5000, 4, 4, 64), (2, 3, 3000, 8, 2, 128), (3, 1, 2100, 16, 1, 80), (1, 16, 1500, 3, 3, 24),  # parts
    (2, 1, 700, 8, 8, 48), (1, 4, 3001, 16, 4, 16), (5, 2, 90, 12, 4, 32), (9, 16, 33, 4, 4, 48),  # merged heads
    (2, 64, 500, 8, 8, 48), (3, 20, 777, 8, 4, 32), (1, 40, 2000, 4, 4, 16), (40, 33, 65, 4, 4, 48),
    (1, 64, 3000, 2, 2, 128), (2, 100, 200, 6, 3, 96), (1, 128, 64, 2, 2, 40),  # 64 and 128 rows
    (2, 300, 400, 4, 4, 128), (1, 1000, 130, 3, 3, 64), (3, 129, 63, 8, 4, 16), (1, 513, 1030, 2, 1, 112)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_routes(dev, B, Lq, Lk, Hq, Hkv, d, dtype):
    g = _gen(dev, B * 7 + Lq + Lk + d)
    q, k, v = _qkv(g, B, Lq, Lk, Hq, Hkv, d, dtype)
    lengths = torch.randint(0, Lk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    mask = torch.rand(B, Lk, generator=g, device=dev) > 0.3
    for n, m in ((None, None), (lengths, None), (None, mask), (lengths, mask)):
        got = ops.cross_attention(q, k, v, key_lengths=n, key_mask=m)
        _within(got, *ref.cross_attention(q, k, v, None, n, m))
        assert torch.equal(got, ops.cross_attention(q, k, v, key_lengths=n, key_mask=m))


@pytest.mark.parametrize("Lq,Hkv,d", [(1, 4, 64), (2, 4, 48), (50, 4, 48), (300, 2, 128)])
def test_masks_longer_than_a_list(dev, Lq, Hkv, d):
    """Nine thousand keys: stretches with every key, with few, with none, and one key at the very end."""
    g = _gen(dev, Lq)
    Lk = 9001
    q, k, v = _qkv(g, 3, Lq, Lk, Hkv, Hkv, d, F16)
    mask = torch.ones(3, Lk, dtype=torch.bool, device=dev)
    mask[0, 4000:8500] = False
    mask[1] = torch.rand(Lk, generator=g, device=dev) > 0.99
    mask[2] = False
    mask[2, -1] = True
    junk = torch.where(mask[:, :, None, None], 0.0, math.nan).to(F16)
    k, v = k + junk, v + junk
    got = ops.cross_attention(q, k, v, key_mask=mask)
    _within(got, *ref.cross_attention(q, k, v, None, None, mask))
    _within(got[2], v[2, -1].double().expand_as(got[2]), ref.half_step(v[2, -1].double(), F16).expand_as(got[2]))


@pytest.mark.parametrize("Lq", [1, 30, 64, 200])
@pytest.mark.parametrize("d", [16, 32, 48, 64])
def test_heads_do_not_touch_each_other(dev, Lq, d):
    """One head's keys and values hold infinities and NaN: the others' results are the same bits as without."""
    g = _gen(dev, Lq + d)
    q, k, v = _qkv(g, 2, Lq, 130, 8, 8, d, F16)
    want = ops.cross_attention(q, k, v)
    kv = torch.stack([k, v], 2)
    for bad in (math.nan, math.inf):
        kv[:, :, 0, 3], kv[:, :, 1, 3] = bad, bad
        got = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1])
        keep = [h for h in range(8) if h != 3]
        assert torch.equal(got[:, :, keep], want[:, :, keep])
        assert got[:, :, 3].isnan().all()


@pytest.mark.parametrize("Lq,Lk", [(1, 4000), (40, 2000)])
def test_parts_whose_scores_lie_far_apart(dev, Lq, Lk):
    g = _gen(dev, 3)
    q, k, v = _qkv(g, 1, Lq, Lk, 2, 2, 64, BF16)
    k = k * torch.linspace(0.1, 12, Lk, device=dev)[:, None, None].to(BF16)
    for kk in (k, k.flip(1)):
        _within(ops.cross_attention(q * 3, kk, v), *ref.cross_attention(q * 3, kk, v))


def _call(q, k, v, out, ws=None, size=0, lengths=None, mask=None):
    s3 = ctypes.c_int64 * 3
    st = [s3(*t.stride()[:3]) for t in (q, k, v, out)]
    desc = _lib.CrossDesc(*st, 0 if mask is None else mask.stride(0), q.shape[0], q.shape[1], k.shape[1], q.shape[2],
                          k.shape[2], q.shape[3], 1 if q.dtype == F16 else 3, 1 / math.sqrt(q.shape[3]))
    need = ctypes.c_size_t()
    lib = _lib.load()
    assert lib.sengine_amd_cross_attention_workspace(ctypes.byref(desc), ctypes.byref(need)) == 0
    ptr = lambda t: None if t is None else t.data_ptr()
    rc = lib.sengine_amd_cross_attention_ws(ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(lengths),
                                            ptr(mask), out.data_ptr(), ws, size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return need.value


def test_without_scratch_memory(dev):
    g = _gen(dev, 8)
    q, k, v = _qkv(g, 1, 1, 6000, 4, 4, 64, F16)
    want = ref.cross_attention(q, k, v)
    small = torch.empty(256, dtype=torch.uint8, device=dev)
    for ws, n in ((None, 0), (small.data_ptr(), 256)):
        out = torch.full_like(q, 7.0)
        assert _call(q, k, v, out, ws, n) > 256
        _within(out, *want)


@pytest.mark.parametrize("d", [8, 48, 128])
def test_rows_at_any_address(dev, d):
    """The C entry takes rows at any element: those that are not 16-byte aligned go another way."""
    g = _gen(dev, d)
    wide = torch.randn(2, 50, 3, 2, d + 5, generator=g, device=dev).to(F16)
    q, k, v = (wide[:, :, i, :, 3:3 + d] for i in range(3))
    q = q[:, :9]
    n = torch.tensor([50, 7], dtype=torch.int32, device=dev)
    mask = torch.rand(2, 50, generator=g, device=dev) > 0.5
    out = torch.zeros(2, 9, 2, d + 1, dtype=F16, device=dev)[..., 1:]
    _call(q, k, v, out, lengths=n, mask=mask)
    _within(out, *ref.cross_attention(q, k, v, None, n, mask))


def test_far_apart_keys(dev):
    """Keys whose strides leave no room for 32-bit offsets inside a stretch."""
    g = _gen(dev, 1)
    wide = torch.zeros(40, 2, 300000, dtype=F16, device=dev)
    kv = torch.randn(1, 40, 2, 2, 16, generator=g, device=dev).to(F16)
    wide[:, :, :32] = kv.view(40, 2, 32)
    k, v = wide[:, 0, :32].view(1, 40, 2, 16), wide[:, 1, :32].view(1, 40, 2, 16)
    q = torch.randn(1, 5, 2, 16, generator=g, device=dev).to(F16)
    _within(ops.cross_attention(q, k, v), *ref.cross_attention(q, k, v))
