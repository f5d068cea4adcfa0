"""Calls of the token operators that compare equal to a remembered one and are not the same, on the host (nothing is
launched)."""
import pytest
import torch

from sparsesnn_amd import ops
from tests.test_linear_e2m1_host import _t


@pytest.mark.parametrize("sections", [(1, 8.0, 15), (1.0, 8, 15), [1, 8, 15.0], (True, 8, 15), ([1], 8, 15)])
def test_sections_are_whole_numbers(monkeypatch, sections):
    monkeypatch.setattr(ops, "_launch", lambda *args: None)
    q, pos, f = _t(2, 5, 4, 48), _t(2, 5, 3, dtype=torch.int32), _t(24, dtype=torch.float32)
    for given in ((1, 8, 15), [1, 8, 15]):
        ops.rotary(q, None, pos, f, given)
        with pytest.raises(ops.SEngineError, match="sections"):
            ops.rotary(q, None, pos, f, sections)
