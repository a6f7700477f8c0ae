"""Layer norm over the last axis, forward and backward, as hand-written HIP kernels (csrc/az_norm_kernels.h).

    y = (x - mean) / sqrt(var + eps) * weight + bias       mean, var over the last axis of x, in float32

The normalisation of the reference is a batch norm (network/util.py:18-33), whose moving averages a network carries from
training into play; a layer norm treats every position by itself, so training and play compute the same function whatever
the batch.  It stands beside `CenterBN` as `AZNet(norm="layer")`.

Tensors on the GPU go through the kernels, on PyTorch's current stream; tensors on the CPU take the same formula in PyTorch.
"""
import torch
import torch.nn as nn

from .device_ops import binding


def _plain(x, weight, bias, eps):
    f = x.float()
    # relative to the row's first value, as the kernels work (csrc/az_norm_kernels.h says why); the derivative is the same
    first = f[..., :1].detach()
    scale = torch.where(first.abs() < 2.0 ** 102, 1.0, 2.0 ** -30)
    d = f * scale - first * scale
    centred = d - d.mean(-1, keepdim=True)
    y = centred / (torch.sqrt((centred * centred).mean(-1, keepdim=True) / (scale * scale) + eps) * scale)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x (float32, bfloat16 or float16; any leading axes, any strides) over its last axis.  weight and bias have
    that axis' length and are both float32 or both of x's type; either may be None.  The result is contiguous and of x's type;
    statistics and the sums of the gradients are float32 and rounded once.  Differentiable once in x, weight and bias.
    A forward without gradients can be captured into a HIP graph; one that records gradients cannot.  Tracers
    (torch.jit.trace, make_fx) do not see inside it: on the GPU it refuses to be traced."""
    y = binding().layer_norm(x, weight, bias, eps)
    return y if y is not None else _plain(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """layer_norm over a last axis of n elements with a learned weight (1) and bias (0)."""

    def __init__(self, n, eps=1e-5):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(n))
        self.bias = nn.Parameter(torch.zeros(n))
        self.eps = eps

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
