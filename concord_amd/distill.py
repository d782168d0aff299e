"""Distillation from a teacher's top logits on the gfx950 kernels of csrc/distill.hip."""
from . import _lib as C


def distill_loss(logits, teacher_logits, teacher_index, temperature=1.0):
    """T^2 times the Kullback-Leibler divergence of softmax(logits / T) from
    the teacher's distribution, which its largest logits stand for: one value
    a row.

    logits [..., vocabulary] (float32, bfloat16 or float16); teacher_logits
    and teacher_index [..., K], K up to 1024, as torch.topk gives them: the
    teacher's probabilities are softmax(teacher_logits / T) over the K
    entries.  An entry whose index lies outside the vocabulary (-1, say) is
    left out; a row without an entry has loss 0.  Two entries of one index add
    up.  The mean of the result over rows is the batch's loss; a row whose
    upstream gradient is 0 (a masked token) gets gradient 0 whatever its
    logits hold.  Differentiable once, in logits alone."""
    return C.ops().distill_loss(logits, teacher_logits, teacher_index, temperature)
