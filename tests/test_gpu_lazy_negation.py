"""Tensors that PyTorch has negated in name only (the imaginary part of a conjugate): memory holds the other sign."""
import pytest
import torch

from alphazero_amd.network import adamw as A
from alphazero_amd.network.layer_norm import layer_norm

pytestmark = pytest.mark.gpu


def _negated(n):
    """-2, -4, ... held as 2, 4, ...: dense where n is 1, else with steps of two."""
    z = torch.complex(torch.zeros(n), 2.0 * torch.arange(1, n + 1)).cuda().conj()
    assert z.imag.is_neg() and float(z.imag[0]) == -2.0
    return z.imag


def test_layer_norm():
    x = torch.randn(5, 1, device="cuda")
    assert torch.equal(layer_norm(x, None, _negated(1)), torch.full((5, 1), -2.0, device="cuda"))      # y is the bias
    w, b = torch.ones(1, device="cuda", requires_grad=True), torch.zeros(1, device="cuda", requires_grad=True)
    db, = torch.autograd.grad(layer_norm(x, w, b), b, _negated(5).view(5, 1))
    assert float(db) == -30.0
    row = torch._neg_view(torch.arange(8.0, device="cuda"))
    assert torch.equal(layer_norm(row.view(1, 8)), layer_norm(-torch.arange(8.0, device="cuda").view(1, 8)))
    leaf = torch.randn(2, 8, device="cuda", requires_grad=True)
    dy = torch.randn(2, 8, device="cuda")
    want, = torch.autograd.grad(layer_norm(leaf), leaf, -dy)
    got, = torch.autograd.grad(layer_norm(leaf), leaf, torch._neg_view(dy))
    assert torch.equal(got, want)


def test_adamw():
    p, m, v = (torch.zeros(1, device="cuda") for _ in range(3))
    A.adamw_step([p], [_negated(1)], [m], [v], 1)
    assert float(m) == pytest.approx(-0.2) and float(p) > 0
    for k in range(3):
        args = [torch.zeros(1, device="cuda") for _ in range(3)]
        args[k] = _negated(1)
        with pytest.raises(TypeError, match="negat"):
            A.adamw_step([args[0]], [torch.ones(1, device="cuda")], [args[1]], [args[2]], 1)
    with pytest.raises(TypeError, match="negat"):
        A.dequantize_state(torch.ones(1, dtype=torch.int8, device="cuda"), _negated(1))
