"""Norms of queries and keys with the position rotation, on the gfx950 kernels of
csrc/qk_rope.hip."""
import torch
import torch.nn as nn

from . import _lib as C


def qk_norm_rope(q, k, q_weight=None, k_weight=None, positions=None, base=10000.0, rotary_dim=None, interleaved=False,
                 eps=1e-6):
    """(q, k) with each head's row divided by its root mean square and multiplied
    by a weight, then rotated by its position.

    q [batch, token, head, dim] and k [batch, token, key head, dim], or both without
    the batch (documents packed one after another), as attention takes them; one of
    float32, bfloat16, float16, in any strides; dim a multiple of 8 up to 256.
    q_weight, k_weight [dim]: a type of their own.  None is a weight of ones: the rows
    are divided by their root mean square all the same.

    positions: int64 or int32, [batch, token] or [token] for all of the batch; each
    token's place in its sequence unless given.  Pair i of the first rotary_dim
    elements (a multiple of 8; dim unless given; 0 turns nothing) turns by position *
    base^(-2 i / rotary_dim).  Pair i is elements i and i + rotary_dim / 2, or 2 i and
    2 i + 1 where interleaved.

    Sums are 32 bits wide, angles 64; the results have q's type.  Differentiable
    once, in q, k and the weights; the weights' gradients are summed over tokens and
    heads in a fixed order.  Nothing but the inputs is kept for the backward."""
    return tuple(C.ops().qk_norm_rope(q, k, q_weight, k_weight, positions, base, rotary_dim, interleaved, eps))


class QKNormRope(nn.Module):
    """qk_norm_rope with its weights, float32 unless dtype says otherwise."""

    def __init__(self, dim, base=10000.0, rotary_dim=None, interleaved=False, eps=1e-6, device=None, dtype=torch.float32):
        super().__init__()
        self.base, self.rotary_dim, self.interleaved, self.eps = base, rotary_dim, interleaved, eps
        self.q_weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.k_weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))

    def forward(self, q, k, positions=None):
        return qk_norm_rope(q, k, self.q_weight, self.k_weight, positions, self.base, self.rotary_dim, self.interleaved,
                            self.eps)

    def extra_repr(self):
        return f"{self.q_weight.numel()}, base={self.base}, rotary_dim={self.rotary_dim}, interleaved={self.interleaved}"
