"""Embedding on the gfx950 kernels of csrc/embedding.hip."""
import torch
import torch.nn as nn

from . import _lib as C


def embedding(tokens, weight, scale=1.0, dtype=None):
    """scale * weight[tokens], in weight's type unless dtype says otherwise.

    tokens: int64 or int32 of any shape; weight [vocabulary, width]: float32,
    bfloat16 or float16, as dtype.  A token outside the vocabulary (-1, say, for
    padding) gives a row of zeros and takes part in no gradient.  The products are
    32 bits wide and rounded once.  Differentiable once, in weight: the gradient
    is that of the whole table, each row the sum over its tokens in the order of
    their positions' pieces, in 32 bits: a fixed order, the same bits every time."""
    return C.ops().embedding(tokens, weight, scale, dtype)


class Embedding(nn.Module):
    """embedding with its table, float32 unless dtype says otherwise.  out_dtype: the
    result's type, the table's unless given."""

    def __init__(self, vocabulary, width, scale=1.0, device=None, dtype=torch.float32, out_dtype=None):
        super().__init__()
        self.scale, self.out_dtype = scale, out_dtype
        self.weight = nn.Parameter(torch.randn(vocabulary, width, device=device, dtype=dtype))

    def forward(self, tokens):
        return embedding(tokens, self.weight, self.scale, self.out_dtype)

    def extra_repr(self):
        return f"{self.weight.shape[0]}, {self.weight.shape[1]}, scale={self.scale}"
