"""The C entry on rows that lie backwards in memory (negative strides), for few rows and many."""
import ctypes

import pytest
import torch

from oracle import token_ops as ref
from sparsesnn_amd import _lib
from tests.test_gpu_token_ops import _gen, _linear_case, _randn, _within

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("M,N,K", [(5, 40, 64), (70, 200, 256), (40, 64, 8192), (2100, 2050, 128)])
@pytest.mark.parametrize("back_x,back_w,back_out", [(True, False, False), (False, True, False), (True, True, False),
                                                    (False, False, True)])
def test_rows_backwards(dev, M, N, K, back_x, back_w, back_out):
    g = _gen(dev, M + N)
    x, w, _, _ = _linear_case(g, M, N, K, BF16)
    r = _randn(g, M, N, dtype=BF16)
    want, bound = ref.linear(x, w, None, "silu", r, None, None, BF16)

    def rows(t, back):  # (pointer to row 0, stride, what keeps it alive)
        if not back:
            return t.data_ptr(), t.stride(0), t
        t = t.flip(0).contiguous()
        return t[-1].data_ptr(), -t.stride(0), t

    (xp, xs, x_), (wp, ws, w_), (rp, rs, r_) = rows(x, back_x), rows(w, back_w), rows(r, back_out)
    out = torch.zeros(M, N, dtype=BF16, device=dev)
    lib = _lib.load()
    desc = _lib.LinearDesc(M=M, x_stride=xs, weight_stride=ws, residual_stride=rs, out_stride=N, N=N, K=K, in_type=3,
                           out_type=3, bias_type=0, activation=4)
    size = ctypes.c_size_t()
    assert lib.sengine_amd_linear_workspace(ctypes.byref(desc), ctypes.byref(size)) == 0
    scratch = torch.empty(size.value, dtype=torch.uint8, device=dev)
    assert lib.sengine_amd_linear_ws(ctypes.byref(desc), xp, wp, None, None, None, rp, out.data_ptr(),
                                     scratch.data_ptr() if size.value else None, size.value,
                                     torch.cuda.current_stream().cuda_stream) == 0
    _within(out, want, bound)
