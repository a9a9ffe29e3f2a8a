"""What the layer norm's Python surface does before anything is launched (no GPU needed: tensors on the host or without
memory stand for the device's)."""
import numpy as np
import pytest
import torch

from noeira_amd import NQError
from noeira_amd.norm import LayerNorm


def norm_on(device, DIM):
    norm = LayerNorm.__new__(LayerNorm)
    norm.DIM, norm.eps = DIM, 1e-5
    norm.gamma, norm.beta = torch.ones(DIM, device=device), torch.zeros(DIM, device=device)
    return norm


def test_parameters_are_copied_without_their_graph():
    """gamma and beta of a module that trains are leaves of a graph; the norm's copies are no part of it."""
    module = torch.nn.LayerNorm(5)
    with torch.no_grad():
        module.weight.copy_(torch.arange(5.0)), module.bias.fill_(0.5)
    norm = norm_on("cpu", 5)
    for _ in range(2):
        norm.set_params(module.weight, module.bias)
        assert torch.equal(norm.gamma, module.weight) and torch.equal(norm.beta, module.bias)
        for t in (norm.gamma, norm.beta):
            assert not t.requires_grad and t.grad_fn is None
    norm.set_params(np.zeros(5), module.weight * 2)
    assert norm.beta.grad_fn is None and norm.beta[4] == 8 and not norm.gamma.any()
    with pytest.raises(NQError, match="gamma is \\[4\\], expected \\[5\\]"):
        norm.set_params(np.zeros(4), module.bias)
