"""Attention over whole sequences on the gfx950 kernels of csrc/attention*.hip."""
import ctypes
import math

import torch

from . import _lib as C


def _tokens(t):
    """[tokens, heads, dim] of a tensor, and whether it is dense (4-d)."""
    if t.dim() == 3:
        return t
    b, n, h, d = t.shape
    if t.stride(0) != n * t.stride(1) and b > 1 and n > 1:
        t = t.contiguous()
    # (a view: one stride steps through the tokens of all sequences)
    return t.as_strided((b * n, h, d), (t.stride(1) if n > 1 else t.stride(0), t.stride(2), t.stride(3)))


def _operand(t):
    """(t as [tokens, heads, dim], stride of a token, of a head) as the kernels
    read it, rows on 16 bytes and dimensions adjacent: a view, or a copy
    where the tensor is laid out otherwise."""
    t = _tokens(t)
    n, h, d = t.shape
    st, sh = t.stride(0) if n > 1 else h * d, t.stride(1) if h > 1 else d
    if t.stride(2) != 1 or st % 8 or sh % 8 or st < d or st >= 1 << 24 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        st, sh = h * d, d
    return t, st, sh


def _check(q, k, v, starts, k_starts, scale):
    for name, t in (("q", q), ("k", k), ("v", v)):
        C.require_device_tensor(t, name)
        if t.dtype != torch.bfloat16:
            raise TypeError(f"attention: {name} must be bfloat16 (got {t.dtype})")
        if t.device != q.device:
            raise ValueError(f"attention: {name} is on {t.device}, q on {q.device}")
        if t.dim() != q.dim() or t.dim() not in (3, 4):
            raise ValueError("attention: q, k and v must all be [token, head, dim] or [batch, token, head, dim]")
    if k.shape != v.shape:
        raise ValueError(f"attention: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    h, hk, d = q.shape[-2], k.shape[-2], q.shape[-1]
    if k.shape[-1] != d or d % 8 or not 8 <= d <= 128:
        raise ValueError(f"attention: q and k need one head dimension, a multiple of 8 up to 128 (got {d} and "
                         f"{k.shape[-1]})")
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"attention: {h} query heads do not share {hk} key heads evenly")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"attention: the scale must be positive (got {scale})")
    if q.dim() == 4:
        if starts is not None or k_starts is not None:
            raise ValueError("attention: starts are for [token, head, dim] tensors")
        if q.shape[0] != k.shape[0]:
            raise ValueError(f"attention: {q.shape[0]} sequences of queries, {k.shape[0]} of keys")
        return
    if starts is None and k_starts is not None:
        raise ValueError("attention: k_starts without starts")
    for name, s in (("starts", starts), ("k_starts", k_starts)):
        if s is None:
            continue
        C.require_device_tensor(s, name)
        if s.dtype != torch.int32 or s.dim() != 1 or s.numel() < 1 or s.device != q.device:
            raise ValueError(f"attention: {name} must be a 1-d int32 tensor on {q.device}, one value longer than "
                             "the count of sequences")
    if k_starts is not None and k_starts.numel() != starts.numel():
        raise ValueError("attention: starts and k_starts count different sequences")
    if starts is not None and k_starts is None and q.shape[0] != k.shape[0]:
        raise ValueError("attention: k_starts is needed where q and k have different token counts")


def _args(q, k, v, out, lse, starts, k_starts, causal, scale, batch):
    """q, k, v and out as (tensor, token stride, head stride)"""
    a = C.AttnArgs()
    (tq, a.q_t, a.q_h), (tk, a.k_t, a.k_h), (tv, a.v_t, a.v_h), (to, a.o_t, a.o_h) = q, k, v, out
    a.q, a.k, a.v, a.out, a.lse = C.ptr(tq), C.ptr(tk), C.ptr(tv), C.ptr(to), C.ptr(lse)
    a.starts, a.k_starts = C.ptr(starts), C.ptr(k_starts)
    a.B = batch if starts is None else starts.numel() - 1
    a.TQ, a.TK = tq.shape[0], tk.shape[0]
    a.H, a.HK, a.D, a.causal, a.scale = tq.shape[1], tk.shape[1], tq.shape[2], int(causal), scale
    return a


def _plain(t):
    """a contiguous [tokens, heads, dim] tensor as an operand"""
    return t, t.shape[1] * t.shape[2], t.shape[2]


def _forward(q, k, v, starts, k_starts, causal, scale, keep):
    """out, and for the backward: the operands as the kernels read them and lse"""
    batch = q.shape[0] if q.dim() == 4 else 1
    q3, k3, v3 = _operand(q), _operand(k), _operand(v)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    tokens, heads, dim = q3[0].shape
    lse = torch.empty((heads, tokens), dtype=torch.float32, device=q.device) if keep else None
    a = _args(q3, k3, v3, _plain(out.view(tokens, heads, dim)), lse, starts, k_starts, causal, scale, batch)
    C.check(C.lib().concord_attention_fwd(ctypes.byref(a), C.stream_of(q.device)), "attention")
    return out, (q3, k3, v3, lse), batch


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, k_starts, causal, scale):
        out, (q3, k3, v3, lse), ctx.batch = _forward(q, k, v, starts, k_starts, causal, scale, True)
        ctx.save_for_backward(q3[0], k3[0], v3[0], out, lse, starts, k_starts)
        ctx.strides = q3[1:], k3[1:], v3[1:]
        ctx.causal, ctx.scale, ctx.shapes = causal, scale, (q.shape, k.shape)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, starts, k_starts = ctx.saved_tensors
        sq, sk, sv = ctx.strides
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        a = _args((q, *sq), (k, *sk), (v, *sv), _plain(out.view(q.shape)), lse, starts, k_starts, ctx.causal,
                  ctx.scale, ctx.batch)
        (tg, a.do_t, a.do_h), (_, a.dq_t, a.dq_h) = _operand(dout), _plain(dq)
        (_, a.dk_t, a.dk_h), (_, a.dv_t, a.dv_h) = _plain(dk), _plain(dv)
        a.dout, a.dq, a.dk, a.dv = C.ptr(tg), C.ptr(dq), C.ptr(dk), C.ptr(dv)
        ws = torch.empty(int(C.lib().concord_attention_workspace_bytes(ctypes.byref(a))), dtype=torch.uint8,
                         device=q.device)
        C.check(C.lib().concord_attention_bwd(ctypes.byref(a), C.ptr(ws), ws.numel(), C.stream_of(q.device)),
                "attention backward")
        shape_q, shape_k = ctx.shapes
        return dq.view(shape_q), dk.view(shape_k), dv.view(shape_k), None, None, None, None


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
    past starts[-1], gives 0.  scale: 1 / sqrt(dim) unless given.

    The values of starts are not read on the host: they must not decrease
    (positions past the tensors are taken as their ends).  Scores, softmax
    and sums are 32 bits wide; the probabilities are rounded to bfloat16 for
    the products with v, as are the scores' gradients.  Differentiable once in
    q, k and v; all sums have a fixed order."""
    scale = 1.0 / math.sqrt(max(q.shape[-1], 1)) if scale is None else float(scale)
    _check(q, k, v, starts, k_starts, scale)
    if starts is not None:
        starts = starts.contiguous()
        k_starts = None if k_starts is None else k_starts.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, starts, k_starts, bool(causal), scale)
    return _forward(q, k, v, starts, k_starts, bool(causal), scale, False)[0]
