"""Attention over whole sequences on the gfx950 kernels of csrc/attention*.hip."""
from . import _lib as C


def attention(q, k, v, starts=None, k_starts=None, causal=True, scale=None):
    """softmax(scale q k^T) v, each query over the keys of its own sequence.

    q [batch, token, head, dim] with k, v [batch, token, key head, dim]: all
    sequences of one length (queries and keys may differ in number).  Or q
    [token, head, dim] and k, v [token, key head, dim]: sequences one after
    another, sequence b from token starts[b] up to starts[b + 1] (int32, on
    the GPU), its keys from k_starts[b] where that is given; without starts,
    one sequence.  bfloat16, in any strides; dim a multiple of 8 up to 128;
    the heads share the key heads in equal groups.

    causal: query i of a sequence with Lq queries and Lk keys sees the keys up
    to i + Lk - Lq.  A query that sees no key, and one before starts[0] or
    past starts[-1], gives 0.  scale: 1 / sqrt(dim) unless given.  Other
    sequences never show, whatever they hold; an infinity or NaN in a key or
    value that the mask hides can reach queries of the same sequence whose last
    key lies less than 96 before it (the step of 64 keys is shared by 32 queries).

    The values of starts are not read on the host: they must not decrease
    (positions past the tensors are taken as their ends).  Scores, softmax
    and sums are 32 bits wide; the probabilities are rounded to bfloat16 for
    the products with v, as are the scores' gradients.  Differentiable once in
    q, k and v; all sums have a fixed order."""
    return C.ops().attention(q, k, v, starts, k_starts, causal, scale)
