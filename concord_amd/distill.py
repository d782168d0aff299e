"""Distillation from a teacher's top logits on the gfx950 kernels of csrc/distill.hip."""
import math

import torch

from . import _lib as C

MAX_TOP = 1024


def _check(logits, teacher, index, temperature):
    for name, t in (("logits", logits), ("teacher_logits", teacher), ("teacher_index", index)):
        C.require_device_tensor(t, name)
        if t.device != logits.device:
            raise ValueError(f"distill_loss: {name} is on {t.device}, logits on {logits.device}")
    if logits.dtype not in C.DTYPES or teacher.dtype not in C.DTYPES:
        raise TypeError("distill_loss: logits and teacher_logits must be float32, bfloat16 or float16")
    if index.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"distill_loss: teacher_index must be int64 or int32 (got {index.dtype})")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("distill_loss: logits need a vocabulary of at least 1")
    if teacher.shape != index.shape or teacher.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"distill_loss: logits {tuple(logits.shape)}, teacher_logits {tuple(teacher.shape)} and "
                         f"teacher_index {tuple(index.shape)} do not name the same rows")
    if teacher.shape[-1] > MAX_TOP:
        raise ValueError(f"distill_loss: at most {MAX_TOP} teacher logits a row (got {teacher.shape[-1]})")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"distill_loss: the temperature must be positive (got {temperature})")


def _forward(logits, teacher, index, temperature, keep):
    vocab, top = logits.shape[-1], teacher.shape[-1]
    rows = logits.numel() // vocab
    z, ld_z = C.rows_of(logits, rows, vocab)
    # 32-bit teacher values and 64-bit places: `top` of each a row
    t, ld_t = C.rows_of(teacher.float(), rows, top)
    i, ld_i = C.rows_of(index.long(), rows, top)
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=z.device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=z.device) if keep else None
    need = int(C.lib().concord_distill_workspace_bytes(rows, vocab))
    ws = torch.empty(need, dtype=torch.uint8, device=z.device) if need else None
    C.check(C.lib().concord_distill_fwd(C.ptr(z), ld_z, C.DTYPES[z.dtype], rows, vocab, C.ptr(t), ld_t,
                                        C.ptr(i), ld_i, top, temperature, C.ptr(loss), C.ptr(stats),
                                        C.ptr(ws), need, C.stream_of(z.device)), "distill_loss")
    return loss, (z, t, i, stats), (ld_z, ld_t, ld_i)


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, index, temperature):
        loss, kept, ctx.ld = _forward(logits, teacher, index, temperature, True)
        ctx.save_for_backward(*kept)
        ctx.temperature, ctx.z_shape = temperature, logits.shape
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        z, t, i, stats = ctx.saved_tensors
        rows, vocab, (ld_z, ld_t, ld_i) = z.shape[0], z.shape[1], ctx.ld
        # one value for all rows (a mean's or a sum's gradient) stays one value
        one = dloss.numel() > 0 and all(s == 0 or n == 1 for s, n in zip(dloss.stride(), dloss.shape))
        g, ld_g = (dloss, 0) if one else C.rows_of(dloss, rows, 1)
        dz = torch.empty(ctx.z_shape, dtype=z.dtype, device=z.device)
        C.check(C.lib().concord_distill_bwd(C.ptr(g), ld_g, C.ptr(z), ld_z, C.DTYPES[z.dtype], rows,
                                            vocab, C.ptr(t), ld_t, C.ptr(i), ld_i, t.shape[1], ctx.temperature, C.ptr(stats), C.ptr(dz), vocab,
                                            C.stream_of(z.device)), "distill_loss backward")
        return dz, None, None, None


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
    temperature = float(temperature)
    _check(logits, teacher_logits, teacher_index, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillLoss.apply(logits, teacher_logits.detach(), teacher_index, temperature)
    return _forward(logits, teacher_logits.detach(), teacher_index, temperature, False)[0]
