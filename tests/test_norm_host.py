"""What the Python surface of the layer norm and the block-scaled layer does before anything is launched (no GPU needed:
tensors on the host or without memory stand for the device's)."""
import numpy as np
import pytest
import torch

from noeira_amd import _lib as L
from noeira_amd import norm as norm_module
from noeira_amd import qlinear
from noeira_amd.norm import LayerNorm
from noeira_amd.qlinear import FP8BlockLinear


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
    with pytest.raises(L.NQError, match="gamma is \\[4\\], expected \\[5\\]"):
        norm.set_params(np.zeros(4), module.bias)


@pytest.mark.parametrize("M", [2 ** 31, 2 ** 32, 2 ** 32 + 5])
def test_counts_beyond_32_bits_are_refused(M, monkeypatch):
    """The C ABI counts in int32: 2^32 + 5 rows would arrive there as 5, 2^32 as none, with the outputs left as they were."""
    def meta(rows, cols, dtype=torch.float32):
        return torch.empty((rows, cols), dtype=dtype, device="meta")

    for module in (norm_module, qlinear):
        monkeypatch.setattr(module, "_check_dev", lambda t, *a: t)
    monkeypatch.setattr(qlinear, "_stream_now", lambda: 0)
    monkeypatch.setattr(norm_module, "_stream_now", lambda: 0)
    norm, x = norm_on("meta", 2), meta(M, 2, torch.bfloat16)
    stats = torch.empty(M, device="meta")
    lin = FP8BlockLinear(16, 16, grad=True)
    codes, scales = meta(M, 16, torch.uint8), meta(M, 1)
    for call in (lambda: norm.forward(x), lambda: norm.forward_train(x), lambda: norm.forward_fp8(x),
                 lambda: norm.vjp(x, stats, stats, x), lambda: qlinear.quantize_rows_fp8_block(x),
                 lambda: lin.forward_a8(codes, scales), lambda: lin.vjp_a8(codes, scales)):
        with pytest.raises(L.NQError, match=f"{M} rows, at most 2\\^31 - 1"):
            call()
    with pytest.raises(L.NQError, match=f"{M} columns, at most"):
        qlinear.quantize_rows_fp8_block(meta(1, M))
    with pytest.raises(L.NQError, match="values in a row"):
        LayerNorm(M)
    with pytest.raises(L.NQError, match="DIM must be positive"):
        LayerNorm(0)
