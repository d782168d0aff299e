"""Activations kept in 8 bits between forward and backward, on the gfx950 kernels of
csrc/act8.hip.

The 8-bit form: 32 adjacent values of the last dimension share a step, the smallest
power of two of which the largest value is at most 127; each value is stored as the
nearest whole number of steps (ties to even).  A value is off by at most half a step,
1/127 of the largest of its 32; no step is smaller than 2^-126, so values of a block of
nothing above 127 2^-127 (fp32 and bf16 have such) are off by up to 2^-127 instead.  A
block that holds an infinity or NaN reads back as NaN, all 32 values of it.
"""
import torch

from . import _lib as C


def gelu8(x, approximate="none"):
    """x Phi(x) (approximate="tanh": its tanh form), with x kept in 8 bits for the backward.

    x: float32, bfloat16 or float16 of any shape.  The result is that of x itself, in
    32 bits and rounded once.  The gradient is the upstream one times gelu's
    derivative at the values that the 8-bit form stands for: 33 bytes for 32 values are
    kept instead of x.  Differentiable once.  Without gradients nothing is kept."""
    return C.ops().gelu8(x, approximate)


def geglu8(x, approximate="none"):
    """a gelu(g) for the halves a, g of x's last dimension, with both kept in 8 bits for
    the backward, each half in blocks of its own (see gelu8)."""
    return C.ops().geglu8(x, approximate)


def pack8(x):
    """(codes, exponents) of x's 8-bit form: int8 of x's shape, and uint8 [..., blocks] with
    the block's power of two + 127 (255: it held an infinity or NaN).  x: float32, bfloat16
    or float16.  Not differentiable."""
    return tuple(C.ops().pack8(x))


def unpack8(codes, exponents, dtype=torch.bfloat16):
    """The values that (codes, exponents) stand for, limited to dtype's largest finite number."""
    return C.ops().unpack8(codes, exponents, dtype)
