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
