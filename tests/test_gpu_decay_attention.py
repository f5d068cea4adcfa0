"""Decaying linear attention against the recurrence in 64 bits: one token and many, chunks and segments that end anywhere,
narrow and wide heads, decays of 0 and 1, lengths, states, strides, values that are no numbers, scratch memory."""
import ctypes
import math

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import _lib, ops
from tests.test_gpu_token_ops import _gen, _randn, _within

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _case(g, B, L, H, dk, dv, dtype, qk=1.0):
    q, k = _randn(g, B, L, H, dk, dtype=dtype, scale=qk), _randn(g, B, L, H, dk, dtype=dtype, scale=qk)
    v = _randn(g, B, L, H, dv, dtype=dtype)
    decay = 1 - torch.exp2(-1 - 10 * torch.rand(H, generator=g, device=g.device))
    if H > 2:
        decay[0], decay[1] = 0.0, 1.0
    return q, k, v, decay, _randn(g, B, H, dk, dv)


def _check(got, want):
    assert got[0].isfinite().all() and got[1].dtype == F32
    _within(got[0], *want[0])
    _within(got[1], *want[1])


SIZES = [  # B, L, H, dk, dv
    (1, 1, 1, 8, 8), (4, 1, 8, 48, 48), (3, 2, 4, 64, 256), (2, 5, 3, 16, 24), (2, 16, 3, 128, 128), (1, 17, 2, 32, 32),
    (2, 33, 3, 40, 56), (1, 63, 4, 64, 64), (3, 64, 3, 48, 48), (2, 65, 3, 128, 64), (1, 127, 3, 96, 128),
    (2, 129, 4, 128, 256), (1, 200, 3, 24, 96), (3, 300, 5, 56, 8), (1, 511, 3, 80, 80), (1, 1030, 4, 64, 128),
    (1, 2500, 3, 32, 40), (1, 777, 1, 128, 128), (2, 1500, 2, 8, 256)]


@pytest.mark.parametrize("B,L,H,dk,dv", SIZES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decay_attention(dev, B, L, H, dk, dv, dtype):
    g = _gen(dev, B + 3 * L + dk + 7 * dv)
    q, k, v, decay, state = _case(g, B, L, H, dk, dv, dtype)
    got = ops.decay_attention(q, k, v, decay)
    assert got[0].shape == (B, L, H, dv) and got[0].dtype == dtype and got[1].shape == (B, H, dk, dv)
    _check(got, ref.decay_attention(q, k, v, decay))
    _check(ops.decay_attention(q, k, v, decay, state=state, scale=0.3),
           ref.decay_attention(q, k, v, decay, state, None, 0.3))


@pytest.mark.parametrize("B,L,H,dk,dv", [(1, 1500, 2, 64, 64), (3, 3000, 67, 128, 128), (4, 3000, 50, 64, 64)])
def test_state_in_place_of_segments(dev, B, L, H, dk, dv):
    """The last segment of a sequence writes the state that the first one reads, in any order: more of them than the chip
    holds at once, sequences that end in their first segment, and an empty one."""
    g = _gen(dev, L + H)
    q, k, v, decay, state = _case(g, B, L, H, dk, dv, BF16)
    lengths = torch.full((B,), L, dtype=torch.int32, device=dev)
    if B > 1:
        lengths[0], lengths[-1] = 40, 0
    want = ops.decay_attention(q, k, v, decay, state=state, lengths=lengths)
    for _ in range(3):
        held = state.clone()
        got = ops.decay_attention(q, k, v, decay, state=held, lengths=lengths, state_out=held)
        assert torch.equal(got[0], want[0]) and torch.equal(held, want[1])


@pytest.mark.parametrize("B,L,H,dk,dv", [(8, 70, 36, 128, 128), (2, 300, 40, 64, 200), (5, 130, 70, 96, 96),
                                         (4, 100, 70, 24, 72), (2, 2100, 24, 128, 128), (1, 1100, 40, 32, 88),
                                         (6, 777, 12, 64, 80), (1, 1100, 56, 32, 88)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_workgroups(dev, B, L, H, dk, dv, dtype):
    """About as many workgroups as the chip has CUs, and more, where waves are wider."""
    g = _gen(dev, B + 3 * L + dk + 7 * dv)
    q, k, v, decay, state = _case(g, B, L, H, dk, dv, dtype)
    _check(ops.decay_attention(q, k, v, decay, state=state), ref.decay_attention(q, k, v, decay, state))


@pytest.mark.parametrize("step", [0, 8, 16, 24])
def test_rows_that_overlap(dev, step):
    """Tokens whose rows begin `step` values apart: a row past the last token would lie within the last ones, and what is
    no number there belongs to other columns."""
    g = _gen(dev, step)
    L, d = 100, 24
    q, k, v, decay, _ = _case(g, 1, L, 1, d, d, BF16)
    spread = lambda t: torch.as_strided(t.flatten(), (1, L, 1, d), (0, step, 0, 1))
    k, v = spread(k), spread(v)
    _check(ops.decay_attention(q, k, v, decay), ref.decay_attention(q, k, v, decay))
    for t in (k, v):
        t[0, L - 1, 0, d - 1] = math.nan
        got, want = ops.decay_attention(q, k, v, decay), ops.decay_attention(q, k.contiguous(), v.contiguous(), decay)
        assert all(torch.equal(a.isnan(), b.isnan()) for a, b in zip(got, want))


@pytest.mark.parametrize("L", [1, 7, 100, 1000])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_lengths(dev, L, dtype):
    """Sequences that end anywhere, one empty, lengths that are clamped; what lies behind is not used."""
    g = _gen(dev, L)
    B, H, dk, dv = 6, 3, 48, 72
    q, k, v, decay, state = _case(g, B, L, H, dk, dv, dtype)
    lengths = torch.tensor([0, L, L // 2, L + 50, -3, max(1, L - 1)], dtype=torch.int32, device=dev)
    behind = torch.arange(L, device=dev) >= lengths[:, None]
    junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min], dtype=dtype, device=dev)
    for t in (q, k, v):
        t.copy_(torch.where(behind[..., None, None], junk[torch.arange(L, device=dev) % 4][:, None, None], t))
    got = ops.decay_attention(q, k, v, decay, state=state, lengths=lengths)
    assert (got[0][behind] == 0).all()
    assert torch.equal(got[1][0], state[0]) and torch.equal(got[1][4], state[4])
    _check(got, ref.decay_attention(q, k, v, decay, state, lengths))
    fresh = ops.decay_attention(q, k, v, decay, lengths=lengths)
    assert (fresh[1][0] == 0).all()
    _check(fresh, ref.decay_attention(q, k, v, decay, None, lengths))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_prompt_and_its_tokens(dev, dtype):
    """A prompt, then tokens one by one and a few at a time on its state, is the whole stream; the state in place."""
    g = _gen(dev, 4)
    B, L, H, dk, dv = 2, 200, 4, 64, 64
    q, k, v, decay, state = _case(g, B, L, H, dk, dv, dtype)
    want = ref.decay_attention(q, k, v, decay, state)
    outs, at, held = [], 0, state.clone()
    for n in (130, 1, 1, 3, 16, 17, 1, 31):
        piece = slice(at, at + n)
        o, s = ops.decay_attention(q[:, piece], k[:, piece], v[:, piece], decay, state=held, state_out=held)
        assert s is held
        outs.append(o)
        at += n
    assert at == L
    _check((torch.cat(outs, 1), held), want)


@pytest.mark.parametrize("L", [3, 150, 900])
def test_strides(dev, L):
    g = _gen(dev, L)
    B, H, d = 2, 3, 48
    q, k, v, decay, state = _case(g, B, L, H, d, d, F16)
    want = ops.decay_attention(q, k, v, decay, state=state)
    _check(want, ref.decay_attention(q, k, v, decay, state))
    qkv = torch.stack([q, k, v], 2)  # one product's output
    views = [qkv[:, :, i] for i in range(3)]
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    for a in (views, heads_first):
        got = ops.decay_attention(*a, decay, state=state)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.full((B, L, 2, H, d), 5.0, dtype=F16, device=dev)
    pool = torch.full((5, H, d, d), 6.0, device=dev)
    pool[1:4:2] = state
    o, s = ops.decay_attention(q, k, v, decay, state=pool[1:4:2], out=wide[:, :, 1], state_out=pool[1:4:2])
    assert torch.equal(o, want[0]) and torch.equal(s, want[1])
    assert (wide[:, :, 0] == 5).all() and (pool[0::2] == 6).all()
    one = ops.decay_attention(q[:1].expand(B, L, H, d), k[:1].expand(B, L, H, d), v[:1].expand(B, L, H, d), decay)
    assert torch.equal(one[0][0], one[0][1])
    _check(one, ref.decay_attention(*(t[:1].expand(B, L, H, d) for t in (q, k, v)), decay))


@pytest.mark.parametrize("L", [5, 64, 200])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_value_that_is_not_finite_leaves_earlier_tokens_alone(dev, L, dtype, value):
    g = _gen(dev, L)
    q, k, v, decay, state = _case(g, 1, L, 4, 32, 64, dtype)
    clean = ops.decay_attention(q, k, v, decay, state=state)
    at = (3 * L) // 4
    for name, t in (("v", v), ("k", k), ("q", q)):
        bad = t.clone()
        bad[0, at, 2, 5] = value
        args = {"q": q, "k": k, "v": v, name: bad}
        o, s = ops.decay_attention(args["q"], args["k"], args["v"], decay, state=state)
        assert torch.equal(o[:, :at], clean[0][:, :at]), name
        others = [0, 1, 3]
        assert torch.equal(o[:, :, others], clean[0][:, :, others]) and torch.equal(s[:, others], clean[1][:, others])
        if name == "q":
            assert not o[0, at, 2].isfinite().any() and torch.equal(s, clean[1])
            assert torch.equal(o[:, at + 1:], clean[0][:, at + 1:])
        elif name == "v":
            assert not o[0, at:, 2, 5].isfinite().any() and not s[0, 2, :, 5].isfinite().any()
            columns = [c for c in range(64) if c != 5]
            assert torch.equal(o[0, :, 2, columns], clean[0][0, :, 2, columns])
        else:
            assert not o[0, at, 2].isfinite().any() and not s[0, 2, 5].isfinite().any()


@pytest.mark.parametrize("L", [9, 300])
def test_far_values(dev, L):
    """States and weights past fp16's range, and below it."""
    g = _gen(dev, L)
    q, k, v, decay, state = _case(g, 2, L, 4, 64, 64, F16)
    decay[1] = 1.0
    for a, b, c, s in ((1e-3, 100.0, 60.0, 1e5), (0.02, 200.0, 2e-4, 1e-3), (1e-2, 1e-4, 1e3, 1.0), (30.0, 30.0, 0.01, 1e2),
                       (1e-3, 1e-3, 1e-1, 0.0)):
        args = ((q * a).to(F16), (k * b).to(F16), (v * c).to(F16))
        want = ref.decay_attention(*args, decay, state * s)
        assert float(want[0][0].abs().max()) < 65504
        _check(ops.decay_attention(*args, decay, state=state * s), want)
    big = v.clone()
    big[..., 0] = 60000.0  # columns of very different sizes
    big[..., 1] *= 1e-4
    _check(ops.decay_attention((q * 1e-3).to(F16), (k * 1e-2).to(F16), big, decay, state=state),
           ref.decay_attention((q * 1e-3).to(F16), (k * 1e-2).to(F16), big, decay, state))


def test_no_tokens(dev):
    g = _gen(dev, 2)
    q, k, v, decay, state = _case(g, 3, 4, 2, 16, 24, F16)
    o, s = ops.decay_attention(q[:, :0], k[:, :0], v[:, :0], decay, state=state)
    assert o.shape == (3, 0, 2, 24) and torch.equal(s, state)
    o, s = ops.decay_attention(q[:, :0], k[:, :0], v[:, :0], decay)
    assert (s == 0).all()
    o, s = ops.decay_attention(q[:0], k[:0], v[:0], decay)
    assert o.shape == (0, 4, 2, 24) and s.shape == (0, 2, 16, 24)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_segments_and_one_workgroup_a_head(dev, dtype):
    """The C entry with scratch memory that holds other values, with too little, without, and without a state to store."""
    g = _gen(dev, 8)
    B, L, H, dk, dv = 2, 3000, 2, 64, 48
    q, k, v, decay, state = _case(g, B, L, H, dk, dv, dtype)
    lengths = torch.tensor([2999, 1200], dtype=torch.int32, device=dev)
    want = ref.decay_attention(q, k, v, decay, state, lengths)
    d = _lib.DecayDesc(B=B, L=L, H=H, dk=dk, dv=dv, type=1 if dtype == F16 else 3, scale=1 / math.sqrt(dk))
    s3, s2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
    d.q_stride = d.k_stride = s3(L * H * dk, H * dk, dk)
    d.v_stride = d.out_stride = s3(L * H * dv, H * dv, dv)
    d.state_stride = d.state_out_stride = s2(H * dk * dv, dk * dv)
    lib, n = _lib.load(), ctypes.c_size_t()
    assert lib.sengine_amd_decay_attention_workspace(ctypes.byref(d), ctypes.byref(n)) == 0 and n.value > 0
    scratch = torch.full((n.value,), 255, dtype=torch.uint8, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    base = [t.data_ptr() for t in (q, k, v, decay, state, lengths)]
    for size in (n.value, n.value - 4, 0):
        out, last = torch.full((B, L, H, dv), -7.0, dtype=dtype, device=dev), torch.empty_like(state)
        rc = lib.sengine_amd_decay_attention_ws(ctypes.byref(d), *base, out.data_ptr(), last.data_ptr(),
                                                scratch.data_ptr() if size else None, size, stream)
        assert rc == 0
        _check((out, last), want)
    out = torch.full((B, L, H, dv), -7.0, dtype=dtype, device=dev)
    assert lib.sengine_amd_decay_attention(ctypes.byref(d), *base, out.data_ptr(), None, stream) == 0
    _check((out, last), want)


def test_side_stream_graph_and_repeats(dev):
    """The same bits on another stream and in a graph replayed with eager work in between."""
    g = _gen(dev, 1)
    cases = [_case(g, 2, 1, 3, 48, 48, F16), _case(g, 2, 90, 3, 64, 64, BF16), _case(g, 1, 2000, 2, 64, 64, F16)]

    def run():
        return [t for q, k, v, decay, state in cases for t in ops.decay_attention(q, k, v, decay, state=state)]

    want = run()
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(3):
        for q, k, v, decay, state in cases:
            v.copy_(v.flip(1) * 0.5)
            state.copy_(state.flip(2))
        want = run()
        for t in held:
            t.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i
