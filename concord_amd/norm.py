"""Layer norm on the gfx950 kernels of csrc/layernorm.hip."""
import torch
import torch.nn as nn

from . import _lib as C


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension.

    x is float32, bfloat16 or float16 of any shape; weight and bias share a
    type of their own (either may be None).  Statistics and sums are 32 bits
    wide, the result has x's type.  Differentiable once, in x, weight and
    bias; the gradients' sums over rows have a fixed order."""
    return C.ops().layer_norm(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """layer_norm with its parameters, float32 unless dtype says otherwise."""

    def __init__(self, width, eps=1e-5, bias=True, device=None, dtype=torch.float32):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}, bias={self.bias is not None}"
