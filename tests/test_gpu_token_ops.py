"""The token operators (norm, linear, cross attention) against their definitions in 64 bits: odd
sizes, strides and alignments, rows and sequences that are empty, NaN and infinity where nothing
counts, outputs in place, streams and graphs.  The bounds are the oracle's."""
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import ops

pytestmark = pytest.mark.gpu
F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


def _within(got, value, bound):
    off = (got.double() - value).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (int(bad.sum()), float((off / bound).nan_to_num(math.inf).max()))


# ------------------------------------------------------------------------ norm

def _check_norm(x, weight, residual, eps, out_dtype, got):
    s, s_bound, y, y_bound = ref.rms_norm(x, weight, residual, eps)
    if residual is None:
        assert got[1] is None
    else:
        _within(got[1], s, s_bound)
    if out_dtype is None:
        assert got[0].dtype == x.dtype
        _within(got[0], y, y_bound + ref.half_step(y, x.dtype))
        return
    c = ref.e4m3_scale(y)
    rel = float((y_bound / y.abs()).nan_to_num(0).max()) + 4 * ref.U
    _within(got[2], c, c * rel)
    # codes are off by half a step of the value (or of the smallest code), the scale by its own error
    step = torch.clamp(y.abs() * 2.0**-4, min=0) + c[..., None] * 2.0**-10
    _within(got[0].double() * got[2].double()[..., None], y, step * (1 + 2.0**-16) + y.abs() * 4 * rel)


@pytest.mark.parametrize("rows,D", [(1, 1), (1, 384), (4, 384), (5, 8), (3, 13), (7, 128), (33, 520), (9, 1000),
                                    (6, 1001), (5, 2056), (3, 4099), (2, 8192), (2, 20000), (1, 32767), (2, 32768),
                                    (1000, 384)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("out_dtype", [None, E4M3])
def test_rms_norm(dev, rows, D, dtype, out_dtype):
    g = _gen(dev, rows * 40000 + D)
    x, r = _randn(g, rows, D, dtype=dtype), _randn(g, rows, D, dtype=dtype, scale=3.0)
    w = 1 + _randn(g, D, scale=0.3)
    for weight, residual in ((w.to(dtype), r), (None, None), (w, None)):
        _check_norm(x, weight, residual, 1e-6, out_dtype,
                    ops.rms_norm(x, weight, residual, eps=1e-6, out_dtype=out_dtype))


def test_rms_norm_strides_in_place_and_extra_dims(dev):
    g = _gen(dev, 5)
    wide = _randn(g, 3, 7, 500, dtype=F16)
    x, r = wide[..., 3:387], wide[..., 100:484].contiguous()  # rows that begin at odd elements
    w = 1 + _randn(g, 384, dtype=F16, scale=0.3)
    got = ops.rms_norm(x, w, r)
    assert got[0].shape == x.shape
    _check_norm(x, w, r, 1e-6, None, got)
    stream = r.clone()
    y, st = ops.rms_norm(x, w, stream, stream_out=stream)  # the stream updated in place
    assert st is stream and torch.equal(y, got[0]) and torch.equal(stream, got[1])
    x2 = x.contiguous()  # aligned rows are summed in another order: their own result is what is compared with
    want = ops.rms_norm(x2, w, r)[0]
    over = x2.clone()
    assert torch.equal(ops.rms_norm(over, w, r, out=over)[0], want)  # the output over the input
    rows = torch.empty(21, 800, dtype=F16, device=dev)[:, 8:392]
    assert ops.rms_norm(x.reshape(21, 384), w, r.view(21, 384), out=rows)[0] is rows
    assert torch.equal(rows, got[0].view(21, 384))
    row = x2[:1, :1].expand(3, 7, 384)  # one row for all
    _check_norm(row, w, r, 1e-6, E4M3, ops.rms_norm(row, w, r, out_dtype=E4M3))


@pytest.mark.parametrize("D", [384, 1001, 5000])
def test_rms_norm_rows_of_zeros_and_not_numbers(dev, D):
    x = torch.zeros(5, D, dtype=F16, device=dev)
    x[1] = 1.0
    x[2, D // 2] = math.nan
    x[3, 0] = math.inf
    x[4, -1] = 65504.0
    q, _, c = ops.rms_norm(x, eps=1e-6, out_dtype=E4M3)
    y, _ = ops.rms_norm(x, eps=1e-6)
    assert (q[0].float() == 0).all() and c[0] == 1 and (y[0] == 0).all()
    assert (q[1].float() == 448).all() and (y[1] == 1).all()
    assert y[2].isnan().all() and q[2].float().isnan().all() and c[2].isnan()
    assert y[3, 0].isnan() and (y[3, 1:] == 0).all() and q[3].float().isnan().all()  # infinity over infinity
    assert y[4, -1].float().item() == pytest.approx(math.sqrt(D), rel=2.0**-11) and (y[4, :-1] == 0).all()
    z, _ = ops.rms_norm(x[:1], eps=0.0)
    assert z.isnan().all()  # 0 / 0, as the formula has it


def test_rms_norm_empty(dev):
    x = torch.empty(0, 384, dtype=F16, device=dev)
    y, s, c = ops.rms_norm(x, residual=x, out_dtype=E4M3)
    assert y.shape == (0, 384) and s.shape == (0, 384) and c.shape == (0,)


# ------------------------------------------------------------------------ linear

def _codes(x):
    c = ref.e4m3_scale(x.float())
    return (x.float() / c[:, None]).to(E4M3), c


def _linear_case(g, M, N, K, dtype):
    x, w = _randn(g, M, K), _randn(g, N, K, scale=1 / math.sqrt(max(K, 1)))
    if dtype == E4M3:
        if K == 0:
            return x.to(E4M3), w.to(E4M3), torch.ones(M, device=x.device), torch.ones(N, device=x.device)
        (x, xs), (w, ws) = _codes(x), _codes(w)
        return x, w, xs, ws
    return x.to(dtype), w.to(dtype), None, None


@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 16, 32), (1, 1000, 384), (2, 3, 5), (4, 1536, 384), (7, 33, 200), (16, 64, 64), (17, 100, 1552),
    (31, 1001, 999), (33, 257, 136), (64, 384, 1536), (65, 63, 63), (100, 8, 4096), (129, 255, 320), (200, 400, 40),
    (257, 513, 264), (300, 520, 1024), (777, 1000, 77), (1500, 640, 384), (3000, 300, 48), (5, 40, 0),
    (2300, 2056, 160)])
@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_linear(dev, M, N, K, dtype):
    g = _gen(dev, M * 7 + N * 5 + K)
    x, w, xs, ws = _linear_case(g, M, N, K, dtype)
    odt = dtype if dtype != E4M3 else (F16, BF16, F32)[M % 3]
    b, r = _randn(g, N, scale=0.5), _randn(g, M, N, dtype=odt)
    for act, bias, res in (("none", None, None), ("gelu", b.to(odt), None), ("silu", b, r)):
        got = ops.linear(x, w, bias, activation=act, residual=res, x_scale=xs, weight_scale=ws, out_dtype=odt)
        assert got.shape == (M, N) and got.dtype == odt
        _within(got, *ref.linear(x, w, bias, act, res, xs, ws, odt))


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("odt", [F16, BF16, F32])
@pytest.mark.parametrize("M", [3, 150])
def test_linear_activations_and_types(dev, act, odt, M):
    g = _gen(dev, M)
    x, w, _, _ = _linear_case(g, M, 96, 128, BF16)
    x = x * 4  # into the flat ends of the activations
    for bdt in (F16, BF16, F32):
        b, r = _randn(g, 96, dtype=bdt), _randn(g, M, 96, dtype=odt)
        got = ops.linear(x, w, b, activation=act, residual=r, out_dtype=odt)
        _within(got, *ref.linear(x, w, b, act, r, None, None, odt))
    q, k = x.to(E4M3), w.to(E4M3)  # without scales
    _within(ops.linear(q, k, b, activation=act, out_dtype=odt), *ref.linear(q, k, b, act, None, None, None, odt))


@pytest.mark.parametrize("M", [1, 30, 300])
@pytest.mark.parametrize("dtype,K", [(F16, 384), (BF16, 100), (E4M3, 384), (E4M3, 1536)])
def test_linear_strides_and_alignment(dev, M, dtype, K):
    g = _gen(dev, M + K)
    N = 200
    x, w, xs, ws = _linear_case(g, M, N, K, dtype)
    odt = BF16 if dtype == E4M3 else dtype
    r = _randn(g, M, N, dtype=odt)
    want = ref.linear(x, w, None, "none", r, xs, ws, odt)
    _within(ops.linear(x, w, residual=r, x_scale=xs, weight_scale=ws, out_dtype=odt), *want)

    def inside(t, pad, at):  # the same values as a slice of wider rows
        wide = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=F32, device=dev).to(t.dtype)
        wide[:, at:at + t.shape[1]] = t
        return wide[:, at:at + t.shape[1]]

    for pad, at in ((16, 16), (32, 8), (7, 3)):
        out = torch.zeros(M, N + pad, dtype=odt, device=dev)
        got = ops.linear(inside(x, pad, at), inside(w, pad, at), residual=inside(r, pad, at), x_scale=xs,
                         weight_scale=ws, out_dtype=odt, out=out[:, at:at + N])
        _within(got, *want)
        out[:, at:at + N] = 0
        assert (out == 0).all()  # nothing beside the rows is written
    acc = r.clone()
    assert ops.linear(x, w, residual=acc, x_scale=xs, weight_scale=ws, out_dtype=odt, out=acc) is acc
    _within(acc, *want)


def test_linear_extra_dims_broadcast_rows_and_empty(dev):
    g = _gen(dev, 9)
    x, w, _, _ = _linear_case(g, 24, 40, 64, F16)
    got = ops.linear(x.view(2, 3, 4, 64), w)
    assert got.shape == (2, 3, 4, 40)
    _within(got.view(24, 40), *ref.linear(x, w, None, "none", None, None, None, F16))
    same = ops.linear(x[:1].expand(300, 64), w)  # one row for all
    assert (same == same[:1]).all()
    _within(same[:1], *ref.linear(x[:1], w, None, "none", None, None, None, F16))
    assert ops.linear(x[:0], w).shape == (0, 40)


@pytest.mark.parametrize("M", [2, 40, 300])
def test_linear_not_numbers(dev, M):
    """NaN and infinity reach the outputs they belong to and no others."""
    g = _gen(dev, M)
    x, w, _, _ = _linear_case(g, M, 70, 200, F16)
    x[0, 5], w[3, 7] = math.nan, math.inf
    w[3].abs_()
    y = ops.linear(x, w)
    assert y[0].isnan().all() and not y[1:, 3].isfinite().any()
    keep = [n for n in range(70) if n != 3]
    assert y[1:, keep].isfinite().all()


# ------------------------------------------------------------------------ cross attention

def _qkv(g, B, Lq, Lk, Hq, Hkv, d, dtype):
    kv = _randn(g, B, Lk, 2, Hkv, d, dtype=dtype)
    return _randn(g, B, Lq, Hq, d, dtype=dtype, scale=1.5), kv[:, :, 0], kv[:, :, 1]


CROSS = [  # B, Lq, Lk, Hq, Hkv, d
    (1, 1, 1, 1, 1, 8), (2, 1, 196, 8, 8, 48), (3, 1, 5, 4, 1, 16), (1, 1, 4000, 8, 2, 64), (2, 1, 1000, 16, 2, 128),
    (2, 3, 65, 6, 3, 40), (1, 5, 63, 4, 4, 32), (2, 16, 64, 2, 2, 24), (1, 17, 130, 8, 1, 80), (2, 33, 200, 4, 2, 48),
    (1, 64, 300, 3, 3, 96), (2, 100, 129, 4, 4, 128), (1, 130, 1, 2, 1, 64), (1, 257, 513, 2, 2, 112),
    (1, 300, 77, 4, 1, 56), (3, 2, 700, 32, 8, 128)]


@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,d", CROSS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_cross_attention(dev, B, Lq, Lk, Hq, Hkv, d, dtype):
    g = _gen(dev, B + Lq * 3 + Lk * 5 + d)
    q, k, v = _qkv(g, B, Lq, Lk, Hq, Hkv, d, dtype)
    _within(ops.cross_attention(q, k, v), *ref.cross_attention(q, k, v))
    lengths = torch.randint(0, Lk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    mask = torch.rand(B, Lk, generator=g, device=dev) > 0.4
    for n, m in ((lengths, None), (None, mask), (lengths, mask)):
        _within(ops.cross_attention(q, k, v, scale=0.2, key_lengths=n, key_mask=m),
                *ref.cross_attention(q, k, v, 0.2, n, m))


@pytest.mark.parametrize("Lq", [1, 20, 200])
@pytest.mark.parametrize("Lk", [1, 70, 1030])
def test_cross_attention_what_does_not_count_is_not_used(dev, Lq, Lk):
    """Keys and values that do not count hold NaN, infinities and the type's lowest values; one
    sequence has no keys by its length, one by its mask."""
    g = _gen(dev, Lq + Lk)
    B, H, d = 4, 3, 64
    q, k, v = _qkv(g, B, Lq, Lk, H, H, d, F16)
    lengths = torch.tensor([Lk, 0, Lk // 2, Lk + 9], dtype=torch.int32, device=dev)  # the last is clamped
    mask = torch.rand(B, Lk, generator=g, device=dev) > 0.3
    mask[3] = False
    counts = mask & (torch.arange(Lk, device=dev) < lengths[:, None])
    junk = torch.tensor([math.nan, math.inf, -math.inf, -65504.0], dtype=F16, device=dev)
    j = junk[torch.arange(Lk, device=dev) % 4]
    for t in (k, v):
        t.copy_(torch.where(counts[:, :, None, None], t, j[None, :, None, None]))
    got = ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask)
    assert (got[1] == 0).all() and (got[3] == 0).all()
    _within(got, *ref.cross_attention(q, k, v, None, lengths, mask))
    _within(ops.cross_attention(q[:3], k[:3], v[:3], key_lengths=counts[:3].sum(1).int() * 0),
            *ref.cross_attention(q[:3], k[:3], v[:3], None, torch.zeros(3, dtype=torch.int32)))


@pytest.mark.parametrize("Lq", [1, 40])
def test_cross_attention_large_scores(dev, Lq):
    """Scores far apart: the maximum moves by more than the exponential's range from tile to tile."""
    g = _gen(dev, 3)
    q, k, v = _qkv(g, 2, Lq, 600, 2, 2, 64, BF16)
    k = k * torch.linspace(0.1, 12, 600, device=dev)[:, None, None].to(BF16)
    q = q * 4
    _within(ops.cross_attention(q, k, v), *ref.cross_attention(q, k, v))
    _within(ops.cross_attention(q, -k.flip(1), v, scale=-0.5), *ref.cross_attention(q, -k.flip(1), v, -0.5))


@pytest.mark.parametrize("Lq,Lk", [(1, 300), (1, 3000), (50, 300)])
def test_cross_attention_strides(dev, Lq, Lk):
    """Heads first, states shared by the batch, an output inside a wider one, no keys at all."""
    g = _gen(dev, Lq)
    B, H, d = 3, 4, 48
    q, k, v = _qkv(g, B, Lq, Lk, H, H, d, F16)
    want = ref.cross_attention(q, k, v)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    _within(ops.cross_attention(*heads_first), *want)
    wide = torch.zeros(B, Lq, 3, H, d, dtype=F16, device=dev)
    out = ops.cross_attention(q, k, v, out=wide[:, :, 1])
    _within(out, *want)
    assert (wide[:, :, 0] == 0).all() and (wide[:, :, 2] == 0).all()
    shared = [t[:1].expand(B, Lk, H, d) for t in (k, v)]
    _within(ops.cross_attention(q, *shared), *ref.cross_attention(q, *shared))
    assert (ops.cross_attention(q, k[:, :0], v[:, :0]) == 0).all()
    assert ops.cross_attention(q[:, :0], k, v).shape == (B, 0, H, d)


# ------------------------------------------------------------------------ streams, graphs, repeats

def _all(x, w8, w, q, k, v, lengths):
    y, s, c = ops.rms_norm(x, residual=x, out_dtype=E4M3)
    a = ops.linear(y, w8, activation="gelu", x_scale=c, out_dtype=F16)
    b = ops.linear(x[:3], w, residual=x[:3])
    return [y.float(), s, c, a, b, ops.cross_attention(q, k, v, key_lengths=lengths),
            ops.cross_attention(q[:, :1], k, v, key_lengths=lengths)]


def test_token_ops_side_stream_and_graph(dev):
    """The same bits on another stream and in a graph replayed with eager work in between."""
    g = _gen(dev, 1)
    x, w = _randn(g, 300, 384, dtype=F16), _randn(g, 384, 384, dtype=F16, scale=0.05)
    q, k, v = _qkv(g, 2, 40, 900, 8, 8, 48, F16)
    n = torch.tensor([900, 123], dtype=torch.int32, device=dev)
    args = (x, w.to(E4M3), w, q, k, v, n)
    want = _all(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _all(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _all(*args)
    for i in range(3):
        x.copy_(x.roll(1, 0))
        q.copy_(q.flip(1))
        n.copy_(n.flip(0))
        want = _all(*args)
        for t in held:
            t.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i
