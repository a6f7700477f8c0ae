"""Layer norm and the AdamW step in 64 bits, written from their formulas, with bounds on what float32 arithmetic may be off by."""
from fractions import Fraction

import torch

U32 = 2.0 ** -24          # half a step of float32, relative


def half_step(dtype):
    """Largest relative error of rounding a value to a type once."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest step of a type: what rounding can cost near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def norm_forward(x, w, b, eps):
    x = x.double()
    n = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / n
    var = ((x - mean) ** 2).sum(-1, keepdim=True) / n
    r = 1.0 / (var + eps) ** 0.5
    h = (x - mean) * r
    y = h if w is None else h * w.double()
    return y if b is None else y + b.double(), mean, r, h


def over_rows(t):
    return t.reshape(-1, t.shape[-1]).sum(0)


def norm_backward(dy, w, r, h):
    g = dy.double() if w is None else dy.double() * w.double()
    n = g.shape[-1]
    dx = r * (g - g.sum(-1, keepdim=True) / n - h * ((g * h).sum(-1, keepdim=True) / n))
    return dx, over_rows(dy.double() * h), over_rows(dy.double())


def norm_bounds(x, w, b, dy, eps, dtype, affine_dtype):
    """(tol_y, tol_dx, tol_dw, tol_db): the sums over a row are trees with a chain of at most cols / 1024 + 24 additions, each
    of which may be off by half a step of its partial sum, at most n max|x| in total; what follows are a handful of
    operations, each off by half a step.  The sums over rows are chains of at most rows / 1024 + 96 additions."""
    y, mean, r, h = norm_forward(x, w, b, eps)
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    k = (32 + cols / 1024) * U32
    rel = k + r * k * x.double().abs().amax(-1, keepdim=True)      # of r, and of h against max(1, |h|)
    eh = rel * (1.0 + 2.0 * h.abs())                               # of h
    aw = torch.ones_like(x[..., :1]).double() if w is None else w.double().abs()
    tol_y = aw * eh + 4 * U32 * (y.abs() + (0 if b is None else b.double().abs())) + half_step(dtype) * (y.abs() + aw * eh) + tiny(dtype)
    if dy is None:
        return tol_y
    dx, dw, db = norm_backward(dy, w, r, h)
    g = dy.double().abs() * aw
    m0, m1 = g.mean(-1, keepdim=True), (g * h.abs()).mean(-1, keepdim=True)
    raw = r * (g + m0 + h.abs() * m1) * (8 * U32 + 2 * k + 2 * rel) + r * (eh * m1 + h.abs() * (g * eh).mean(-1, keepdim=True))
    tol_dx = raw + half_step(dtype) * (dx.abs() + raw) + tiny(dtype)
    k2 = (96 + rows / 1024) * U32
    t = over_rows(dy.double().abs() * eh) + k2 * over_rows(dy.double().abs() * h.abs())
    tol_dw = t + half_step(affine_dtype) * (dw.abs() + t) + tiny(affine_dtype)
    t = k2 * over_rows(dy.double().abs())
    tol_db = t + half_step(affine_dtype) * (db.abs() + t) + tiny(affine_dtype)
    return tol_y, tol_dx, tol_dw, tol_db


BLOCK = 256


def values(codes, scales):
    """What the codes of an 8-bit state stand for, in 64 bits, flat."""
    c = codes.reshape(-1).double()
    s = scales.double().repeat_interleave(BLOCK)[:c.numel()]
    return s * (c * c.abs()) * (1.0 / 127.0 ** 2) if codes.dtype == torch.int8 else s * (c * c) ** 2 * (1.0 / 255.0 ** 4)


def codes_of(x, signed):
    """The nearest codes of a flat state in 64 bits, block by block."""
    n = x.numel()
    full = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:n] = x
    full = full.view(-1, BLOCK)
    s = full.abs().amax(1).float()
    d = s.double()[:, None]
    ratio = torch.where((d > 0) & torch.isfinite(d), full.abs() / d, torch.zeros_like(full))
    x = 127.0 * torch.sqrt(ratio) if signed else 255.0 * torch.sqrt(torch.sqrt(ratio))
    c = x.round()
    # what may lie on a border is settled in whole numbers: the even code where it does
    for i, j in ((x - x.floor() - 0.5).abs() < 1e-9).nonzero().tolist():
        value, scale, low = Fraction(abs(float(full[i, j]))), Fraction(float(s[i])), int(x[i, j])
        border = scale * Fraction(2 * low + 1, 254 if signed else 510) ** (2 if signed else 4)
        c[i, j] = low + (1 if value > border or (value == border and low % 2) else 0)
    if signed:
        c = c * full.sign()
    else:
        c = torch.where((full > 0) & (d > 0) & torch.isfinite(d), c.clamp(min=1.0), c)
    return torch.nan_to_num(c).reshape(-1)[:n].to(torch.int8 if signed else torch.uint8), s


def adamw(p, g, m, v, step, lr, beta1, beta2, eps, decay):
    """New (p, m, v) and the bounds of float32 arithmetic on them; m and v as the values they stand for."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    m2 = beta1 * m + (1 - beta1) * g
    v2 = beta2 * v + (1 - beta2) * (g * g)     # (rounded in the order in which the kernels document it)
    den = (v2 / (1 - beta2 ** step)) ** 0.5 + eps
    update = lr * (m2 / (1 - beta1 ** step)) / den
    p2 = p - lr * decay * p - update
    # a rounded factor, a product and a sum for each term: four half steps, one more for the square
    small = 2.0 ** -149
    tol_m = 4 * U32 * ((beta1 * m).abs() + ((1 - beta1) * g).abs()) + 4 * small
    tol_v = 5 * U32 * (beta2 * v + (1 - beta2) * g * g) + 4 * small
    root = v2 ** 0.5 / (1 - beta2 ** step) ** 0.5
    tol_root = torch.where(v2 > 0, root * tol_v / (2 * v2.clamp(min=1e-300)), torch.zeros_like(v2))
    tol_u = lr / (1 - beta1 ** step) * tol_m / den + update.abs() * (tol_root / den + 12 * U32)
    tol_p = 4 * U32 * (p.abs() + update.abs()) + tol_u + 4 * small
    return p2, m2, v2, tol_p, tol_m, tol_v
