"""Outputs whose rows overlap across two dimensions, refused on the host; strides of any order that keep them apart are not."""
import ctypes

import pytest

from sparsesnn_amd import _lib
from tests.test_cross_output_host import _call
from tests.test_decay_attention_host import _desc
from tests.test_linear_e2m1_host import _rc, _rotary

P, ODD = 0x1000, 0x1008
D3 = 300 * 4 * 48


@pytest.mark.parametrize("kw", [
    dict(out_stride=(48, 48, 48)), dict(out_stride=(D3, 48, 48)), dict(out_stride=(D3, 192, 192)),
    dict(out_stride=(192, 192, 48)), dict(out_stride=(D3 - 8, 192, 48)), dict(out_stride=(D3, -48, 48)),
    dict(out_stride=(D3, 48, 300 * 48 - 8)), dict(out_stride=(-2**62, 2**62, 48)), dict(out_stride=(2**63 - 8, 2**61, 48)),
    dict(state_out_stride=(64 * 48, 64 * 48)), dict(state_out_stride=(4 * 64 * 48 - 4, 64 * 48)),
    dict(state_out_stride=(64 * 48, 2 * 64 * 48 - 4)), dict(state_out_stride=(64 * 48, -64 * 48))])
def test_decay_attention_refuses(kw):
    rc, text = _rc("sengine_amd_decay_attention", _desc(**kw), P, P, P, P, P, P, P, P, None)
    assert rc == -2 and "overlap" in text


@pytest.mark.parametrize("kw", [
    dict(out_stride=(D3, 48, 300 * 48)), dict(out_stride=(192, 2 * 192, 48)), dict(out_stride=(D3, 192, -48)),
    dict(out_stride=(0, 192, 48), B=1), dict(out_stride=(48, 2 * 192, 2 * 48)), dict(state_out_stride=(64 * 48, 2 * 64 * 48)),
    dict(state_out_stride=(-4 * 64 * 48, 64 * 48)), dict(out_stride=(2**62, 192, 48))])
def test_decay_attention_takes(kw):
    """The next check, of q's address, is what these meet."""
    rc, text = _rc("sengine_amd_decay_attention", _desc(**kw), ODD, P, P, P, P, P, P, P, None)
    assert rc == -2 and "overlap" not in text and "16 bytes" in text


@pytest.mark.parametrize("kw", [
    dict(out_q_stride=(48, 48, 48)), dict(out_q_stride=(576, 192, 192)), dict(out_q_stride=(192, 192, 48)),
    dict(out_q_stride=(575, 192, 48)), dict(out_k_stride=(288, 96, 96)), dict(out_k_stride=(288, 48, -48)),
    dict(out_k_stride=(144, 48, 143))])
def test_rotary_refuses(kw):
    rc, text = _rc("sengine_amd_rotary", _rotary(**kw), P, P, P, P, P, P, None)
    assert rc == -2 and "overlap" in text


@pytest.mark.parametrize("stride", [(64, 64, 64), (768, 256, 256), (256, 256, 64), (760, 256, 64), (768, -64, 64)])
def test_cross_attention_refuses(stride):
    rc, text = _call({}, stride)
    assert rc == -2 and "overlap" in text


def test_the_workspace_entry_refuses_too():
    d = _desc(out_stride=(48, 48, 48))
    rc = _lib.load().sengine_amd_decay_attention_ws(ctypes.byref(d), P, P, P, P, P, P, P, P, None, 0, None)
    assert rc == -2 and "overlap" in _lib.load().sengine_amd_last_error().decode()
