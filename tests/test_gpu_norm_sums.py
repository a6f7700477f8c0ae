"""The sums over rows of layer norm's gradient, with so many rows that the order of the additions counts."""
import pytest
import torch

from alphazero_amd import _lib
from alphazero_amd.network.layer_norm import layer_norm
from tests import train_ops_ref as R

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,dtype", [(40000, 8192, torch.bfloat16), (10000, 8200, torch.bfloat16), (60000, 8200, torch.float16),
                                             (60000, 8200, torch.float32), (60000, 20000, torch.bfloat16), (100003, 5000, torch.bfloat16),
                                             (150000, 3000, torch.float16), (300000, 1000, torch.float32)])
def test_sums_over_many_rows(rows, cols, dtype):
    """One row of x and dy read over and over: equal addends, whose roundings do not cancel.  The bound is that of
    R.norm_bounds, chains of at most rows / 1024 + 96 additions, each off by half a step of a partial sum."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, dy = torch.randn(1, cols, generator=g, device=DEV).to(dtype), torch.randn(1, cols, generator=g, device=DEV).to(dtype)
    w, b = torch.ones(cols, device=DEV, requires_grad=True), torch.zeros(cols, device=DEV, requires_grad=True)
    many = x.expand(rows, cols).detach().requires_grad_()
    dx, dw, db = torch.autograd.grad(layer_norm(many, w, b), (many, w, b), dy.expand(rows, cols))
    _, _, r, h = R.norm_forward(x, w.detach(), b.detach(), 1e-5)
    k2, k = (96 + rows / 1024) * R.U32, (32 + cols / 1024) * R.U32
    eh = (k + r * k * x.double().abs().max()) * (1.0 + 2.0 * h.abs())
    d = dy.double()
    off = (dw.double() - rows * (d * h)[0]).abs() / (rows * (d.abs() * eh)[0] + k2 * rows * (d * h).abs()[0])
    assert float(off.max()) <= 1.0
    off = (db.double() - rows * d[0]).abs() / (k2 * rows * d.abs()[0])
    assert float(off.max()) <= 1.0
    # (with each other: a single row of 20000 is worked on in chunks, in another order)
    assert torch.equal(dx[[1, rows // 2, rows - 1]], dx[:1].expand(3, cols))


def test_no_chain_is_longer_than_stated():
    """The number of partial rows, from the size of the workspace: rows summed by one thread, the groups of a workgroup, every 64th
    partial row and the last 18 additions together stay below the bound of the numerics tests (the first addition of each of the
    four stages is to 0 and exact)."""
    L = _lib.lib()
    for kind, per in ((0, 4), (1, 8), (2, 8)):
        for cols in (1, 7, 30, 64, 100, 256, 361, 722, 1024, 2000, 2048, 2056, 4096, 4104, 8192, 8200, 16384, 16400, 20000, 300000):
            packs = cols // per
            wide, apart = packs > 16384 // per, packs > 8192 // per
            groups = 1 if apart or packs > 256 else 64 if packs <= 4 and kind == 0 else 32 if packs <= 8 else 16 if packs <= 16 else 8 if packs <= 32 else 4
            for rows in (1, 5, 63, 64, 65, 300, 4096, 4097, 6600, 10000, 40000, 65536, 65537, 200000, 10 ** 6):
                chunks = 2 * rows * -(-cols // 8192) if wide and rows < 256 else 0
                parts, rest = divmod(L.az_layer_norm_bwd_workspace(kind, rows, cols) - chunks, 2 * cols)
                assert rest == 0 and 1 <= parts <= 1536
                longest = -(-rows // (parts * groups))
                if groups == 1 and not apart:          # 512 or 256 workgroups, each of which may write several partial rows
                    longest = min(max(64, -(-rows // 1024)), -(-rows // min(parts, 512 if packs <= 512 else 256)))
                chain = longest + groups + -(-parts // 64) + 18 - 4
                assert chain <= rows / 1024 + 96, (kind, rows, cols, parts)
