"""The numbers that the token operators take as eps and scale, checked on the host."""
import numpy as np
import pytest
import torch

from sparsesnn_amd import ops


def test_numbers():
    for x in (0.5, np.float32(0.5), np.array(0.5), torch.tensor(0.5), torch.tensor([0.5], dtype=torch.float64)):
        got = ops._token_number(x, "eps")
        assert type(got) is float and got == 0.5
    assert ops._token_number(3, "eps") == 3.0 and ops._token_number(True, "eps") == 1.0
    assert ops._token_number(0.1, "eps") == float(np.float32(0.1))


def test_what_is_no_number_is_refused():
    for x in ("1.0", None, [1.0], 1j):
        with pytest.raises(TypeError):
            ops._token_number(x, "eps")
    value = torch.nn.Parameter(torch.tensor(0.5))
    with pytest.raises(ops.SEngineError, match="eps requires a gradient"):
        ops._token_number(value, "eps")
    with torch.no_grad():
        assert ops._token_number(value, "eps") == 0.5
