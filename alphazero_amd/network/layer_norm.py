"""Layer norm over the last axis, forward and backward, as hand-written HIP kernels (csrc/az_norm_kernels.h).

    y = (x - mean) / sqrt(var + eps) * weight + bias       mean, var over the last axis of x, in float32

The normalisation of the reference is a batch norm (network/util.py:18-33), whose moving averages a network carries from
training into play; a layer norm treats every position by itself, so training and play compute the same function whatever
the batch.  It stands beside `CenterBN` as `AZNet(norm="layer")`.

Tensors on the GPU go through the kernels, on PyTorch's current stream; tensors on the CPU take the same formula in PyTorch.
"""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .device_ops import TYPE_IDS, check, current_stream, library


def _rows(x, cols):
    """(tensor, elements from one row to the next): x as rows of `cols` neighbouring elements, copied only if it is not one."""
    if x.is_contiguous():
        return x, cols
    if x.dim() > 1 and (x.stride(-1) == 1 or cols == 1):
        try:
            v = x.view(-1, cols)
            return v, v.stride(0)
        except RuntimeError:
            pass   # the leading axes do not merge into one
    return x.contiguous(), cols


def _forward(x, weight, bias, eps, want_stats):
    cols = x.shape[-1]
    rows = x.numel() // cols
    device = x.device
    v, stride = _rows(x, cols)
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=device) if want_stats else None
    a, w, b = _affine(x, weight, bias)
    at = stats.data_ptr() if want_stats else None
    check(library().az_layer_norm_fwd_dev(device.index, current_stream(device.index), TYPE_IDS[x.dtype], a, rows, cols, eps, v.data_ptr(), stride,
                                          w.data_ptr() if w is not None else None, b.data_ptr() if b is not None else None,
                                          y.data_ptr(), cols, at, at + 4 * rows if want_stats else None))
    return y, stats


def _affine(x, weight, bias):
    given = weight if weight is not None else bias
    return (TYPE_IDS[given.dtype] if given is not None else 0,
            weight.contiguous() if weight is not None else None, bias.contiguous() if bias is not None else None)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.affine_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        cols = x.shape[-1]
        rows = x.numel() // cols
        device = x.device
        v, x_stride = _rows(x, cols)
        g, dy_stride = _rows(dy, cols)
        L = library()
        dx = torch.empty(x.shape, dtype=x.dtype, device=device) if want_x else None
        dw = torch.empty(cols, dtype=ctx.affine_dtype, device=device) if want_w else None
        db = torch.empty(cols, dtype=ctx.affine_dtype, device=device) if want_b else None
        n = L.az_layer_norm_bwd_workspace(TYPE_IDS[x.dtype], rows, cols) if want_w or want_b else 0
        space = torch.empty(n, dtype=torch.float32, device=device) if n else None
        w = weight.contiguous() if weight is not None else None
        at = stats.data_ptr()
        check(L.az_layer_norm_bwd_dev(device.index, current_stream(device.index), TYPE_IDS[x.dtype], TYPE_IDS[ctx.affine_dtype], rows, cols,
                                      g.data_ptr(), dy_stride, v.data_ptr(), x_stride, w.data_ptr() if w is not None else None,
                                      at, at + 4 * rows, dx.data_ptr() if want_x else None, cols,
                                      dw.data_ptr() if want_w else None, db.data_ptr() if want_b else None,
                                      space.data_ptr() if n else None, n))
        return dx, dw, db, None


def _plain(x, weight, bias, eps):
    f = x.float()
    centred = f - f.mean(-1, keepdim=True)
    y = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x (float32, bfloat16 or float16; any leading axes, any strides) over its last axis.  weight and bias have
    that axis' length and are both float32 or both of x's type; either may be None.  The result is contiguous and of x's type;
    statistics and the sums of the gradients are float32 and rounded once.  Differentiable once in x, weight and bias.
    A forward without gradients can be captured into a HIP graph; one that records gradients cannot."""
    if x.dtype not in TYPE_IDS:
        raise TypeError("layer_norm takes float32, bfloat16 or float16, not %s" % x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm needs a last axis of at least one element")
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be a non-negative number")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError("%s has shape %s, the last axis of x has %d elements" % (name, tuple(t.shape), x.shape[-1]))
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError("%s must be float32 or of x's type, not %s" % (name, t.dtype))
        if t.device != x.device:
            raise ValueError("%s is on %s, x on %s" % (name, t.device, x.device))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type")
    if x.device.type == "cpu":
        return _plain(x, weight, bias, eps)
    if x.device.type != "cuda":
        raise ValueError("layer_norm runs on the GPU or the CPU, not on %s" % x.device)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        if torch.cuda.is_current_stream_capturing():
            # the gradients of leaves are added on the stream on which the leaf was first used; where that is not the
            # captured one the capture breaks in the autograd thread and takes the process with it
            raise RuntimeError("layer_norm cannot record gradients while a HIP graph is captured: use torch.no_grad()")
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


class LayerNorm(nn.Module):
    """layer_norm over a last axis of n elements with a learned weight (1) and bias (0)."""

    def __init__(self, n, eps=1e-5):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(n))
        self.bias = nn.Parameter(torch.zeros(n))
        self.eps = eps

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
