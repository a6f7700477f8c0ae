"""Layer norm of rows without spread, on CPU tensors."""
import pytest
import torch

from alphazero_amd.network.layer_norm import layer_norm


@pytest.mark.parametrize("cols", [1, 3, 300, 361, 722, 9001])
@pytest.mark.parametrize("value", [0.1, -1000.1, 123456.7, 1.2e36, -3.1e38])
def test_rows_of_one_value(cols, value):
    x = torch.full((3, cols), value, requires_grad=True)
    w, b = torch.full((cols,), 2.0, requires_grad=True), torch.randn(cols)
    y = layer_norm(x, w, b)
    assert torch.equal(y, b.expand(3, cols))
    dy = torch.randn(3, cols)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = 2.0 * (dy.double() - dy.double().mean(1, keepdim=True)) / 1e-5 ** 0.5
    # a mean of float32 values and a handful of operations, each off by half a step
    assert not dw.any() and bool(((dx.double() - want).abs() <= 64 * 2.0 ** -24 * 2.0 * (dy.double().abs() + dy.double().abs().mean(1, keepdim=True)) / 1e-5 ** 0.5).all())


def test_rows_of_both_signs_of_the_largest_numbers():
    x = torch.tensor([[3e38, -3e38] * 50, [-3e38, 3e38] * 50])
    assert torch.equal(layer_norm(x), torch.zeros(2, 100))


def test_derivative_does_not_see_what_the_row_is_taken_relative_to():
    x = torch.randn(4, 30, dtype=torch.float32, requires_grad=True)
    dy = torch.randn(4, 30)
    dx, = torch.autograd.grad(layer_norm(x), x, dy)
    y = x.detach().double().requires_grad_()
    h = (y - y.mean(1, keepdim=True)) / (y.var(1, unbiased=False, keepdim=True) + 1e-5) ** 0.5
    want, = torch.autograd.grad(h, y, dy.double())
    assert float((dx.double() - want).abs().max()) < 1e-5
