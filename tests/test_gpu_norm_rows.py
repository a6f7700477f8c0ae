"""Layer norm on the GPU in rows whose mean is very large against their spread: rows of one value, rows of neighbouring float32
values, rows next to the largest numbers."""
import pytest
import torch

from alphazero_amd.network.layer_norm import layer_norm
from tests import train_ops_ref as R
from tests.test_gpu_train_ops import _gen, _inside

pytestmark = pytest.mark.gpu

DEV, F32 = "cuda", torch.float32


@pytest.mark.parametrize("cols", [1, 3, 16, 30, 256, 257, 512, 700, 1024, 2048, 4096, 8192, 8194, 16384, 20000])
@pytest.mark.parametrize("value,eps", [(2.0 ** 112, 1e-12), (-(2.0 ** 110), 1e-12), (2.0 ** 100, 1e-30)])
def test_rows_of_one_large_value(cols, value, eps):
    """No spread, |x| / sqrt(eps) past the largest float32: y is the bias, dx what eps leaves of dy less its mean.  (A power of two,
    whose sums are exact.)"""
    x = torch.full((3, cols), value, device=DEV)
    w = 1.0 + 0.1 * torch.randn(cols, generator=_gen(1), device=DEV)
    b = torch.randn(cols, generator=_gen(2), device=DEV)
    dy = 1e-3 * torch.randn(3, cols, generator=_gen(3), device=DEV)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y, b.expand(3, cols)) and not dw.any()
    g = dy.double() * w.detach().double()
    want = (g - g.mean(1, keepdim=True)) / eps ** 0.5
    # g, its sum (chains as in R.norm_bounds) and its mean, a difference and r: each off by half a step or, r, by two
    tol = ((40 + cols / 1024) * R.U32 * (g.abs() + g.abs().mean(1, keepdim=True))) / eps ** 0.5 + R.tiny(F32)
    _inside(dx, want, tol, "dx")
    _inside(db, dy.double().sum(0), 8 * R.U32 * dy.double().abs().sum(0), "dbias")


WIDTHS = [1, 3, 16, 30, 65, 300, 361, 400, 700, 722, 1023, 1500, 2047, 3001, 5000, 9001, 16383, 20001]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("value", [0.1, -1000.1, 123456.7, 16777213.0, 1.2e36, -3.1e38, 1e-42])
def test_rows_of_one_value(cols, value):
    """Every value is exactly the mean: y is the bias to the bit, dweight is 0, dx what eps leaves of dy less its mean."""
    for rows in (2, 300):
        x = torch.full((rows, cols), value, device=DEV)
        w = 1.0 + 0.1 * torch.randn(cols, generator=_gen(4), device=DEV)
        b = torch.randn(cols, generator=_gen(5), device=DEV)
        dy = torch.randn(rows, cols, generator=_gen(6), device=DEV)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = layer_norm(*leaves)
        dx, dw, _ = torch.autograd.grad(y, leaves, dy)
        assert torch.equal(y, b.expand(rows, cols)) and not dw.any()
        g, r = dy.double() * w.detach().double(), 1e-5 ** -0.5
        want = (g - g.mean(1, keepdim=True)) * r
        # g, its sum (chains as in R.norm_bounds) and its mean, a difference and r: each off by half a step or, r, by two
        _inside(dx, want, (40 + cols / 1024) * R.U32 * (g.abs() + g.abs().mean(1, keepdim=True)) * r + R.tiny(F32), "dx")


def _far_bounds(x, w, b, dy, eps):
    """As R.norm_bounds, with rows taken relative to their first value: differences from it are off by half a step of their own
    size, not of the mean's, so the mean is off by k max|x - x[0]| (the same chains), h by that times r and by r's own error.
    The backward pass has the mean rounded to float32: half a step of the mean more."""
    y, mean, r, h = R.norm_forward(x, w, b, eps)
    rows, cols = x.shape
    k = (32 + cols / 1024) * R.U32
    off = r * k * (x.double() - x[:, :1].double()).abs().amax(1, keepdim=True)     # of h, from the mean
    eh = off + h.abs() * (k + off * off)                                            # and from r: the variance takes the square of it
    ty = w.double().abs() * eh + 4 * R.U32 * (y.abs() + b.double().abs()) + R.half_step(F32) * y.abs() + R.tiny(F32)
    eb = eh + r * R.U32 * mean.abs()
    g = (dy.double() * w.double()).abs()
    m0, m1 = g.mean(1, keepdim=True), (g * h.abs()).mean(1, keepdim=True)
    raw = r * (g + m0 + h.abs() * m1) * (8 * R.U32 + 2 * k + off * off) + r * (eb * m1 + (h.abs() + eb) * (g * eb).mean(1, keepdim=True))
    tx = raw + R.half_step(F32) * raw + R.tiny(F32)
    k2 = (96 + rows / 1024) * R.U32
    tw = R.over_rows(dy.double().abs() * eb) + k2 * R.over_rows(dy.double().abs() * (h.abs() + eb))
    return y, r, h, ty, tx, tw


@pytest.mark.parametrize("cols", WIDTHS[1:])
@pytest.mark.parametrize("mean,spread", [(1e4, 1.0), (-3e5, 1.0), (1e6, 0.3), (1000.1, 0.0), (5e6, 0.0)])
def test_rows_far_from_zero(cols, mean, spread):
    """A mean up to a million times the spread; a spread of 0 stands for two neighbouring float32 values."""
    for rows in (3, 270):
        g = _gen(cols)
        x = torch.full((rows, cols), mean, device=DEV)
        if spread:
            x += spread * torch.randn(rows, cols, generator=g, device=DEV)
        else:
            up = torch.nextafter(x, torch.full_like(x, float("inf")))
            x = torch.where(torch.rand(rows, cols, generator=g, device=DEV) < 0.3, up, x)
        w = 1.0 + 0.1 * torch.randn(cols, generator=g, device=DEV)
        b, dy = torch.randn(cols, generator=g, device=DEV), torch.randn(rows, cols, generator=g, device=DEV)
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = layer_norm(*leaves)
        dx, dw, _ = torch.autograd.grad(y, leaves, dy)
        want, r, h, ty, tx, tw = _far_bounds(x, w, b, dy, 1e-5)
        rdx, rdw, _ = R.norm_backward(dy, w, r, h)
        _inside(y, want, ty, "y")
        _inside(dx, rdx, tx, "dx")
        _inside(dw, rdw, tw, "dweight")


def test_rows_whose_first_value_is_far_from_the_others():
    """What the row is taken relative to is then far from its mean; the spread is of that size too."""
    for first in (1e6, -1e30, 2.0 ** 103, 3e38):
        x = torch.randn(4, 361, generator=_gen(7), device=DEV)
        x[:, 0] = first
        w, b = torch.full((361,), 2.0, device=DEV), torch.randn(361, generator=_gen(8), device=DEV)
        y = layer_norm(x, w, b)
        if abs(first) > 1e18:       # the variance is past float32: its root is taken as infinite, h as 0
            assert torch.equal(y, b.expand(4, 361))
        else:
            want, _, _, ty, _, _ = _far_bounds(x, w, b, torch.zeros_like(x), 1e-5)
            _inside(y, want, ty, "y")


def test_differences_past_the_largest_number():
    """Rows of both signs of the largest numbers: no difference of two values overflows on the way to h = 0."""
    for cols in (2, 256, 361, 5000, 20000):
        x = torch.full((2, cols), 3e38, device=DEV)
        x[:, 1::2] = -3e38
        assert torch.equal(layer_norm(x), torch.zeros(2, cols, device=DEV))


def test_sixteen_bit_rows_of_one_value():
    for dtype in (torch.bfloat16, torch.float16):
        for cols in WIDTHS:
            x = torch.full((5, cols), 1003.0, device=DEV).to(dtype)
            b = torch.randn(cols, generator=_gen(9), device=DEV)
            assert torch.equal(layer_norm(x, None, b), b.to(dtype).expand(5, cols))
