"""TokenReader's weights, made on the host: nothing of them holds on to the parameters' gradients."""
import pytest
import torch

from sparsesnn_amd import token_reader as tr


@pytest.mark.parametrize("eight_bit", [False, True])
def test_weights_ask_for_no_gradient(eight_bit):
    p = {k: torch.nn.Parameter(v) for k, v in tr.random_reader_params(0, embed=64, depth=2, num_classes=10).items()}
    reader = tr.TokenReader(p, heads=4, eight_bit=eight_bit, device="cpu")
    held = [*reader.p.values(), *(t for pair in reader.fc1 or () for t in pair)]
    assert len(held) == len(p) + (4 if eight_bit else 0)
    assert not any(t.requires_grad or t.grad_fn is not None for t in held)
