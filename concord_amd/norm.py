"""Layer norm on the gfx950 kernels of csrc/layernorm.hip."""
import torch
import torch.nn as nn

from . import _lib as C


def _check(x, weight, bias):
    C.require_device_tensor(x, "x")
    if x.dtype not in C.DTYPES:
        raise TypeError(f"layer_norm: x must be float32, bfloat16 or float16 (got {x.dtype})")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm: x needs a last dimension of at least 1")
    wdtype = None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        C.require_device_tensor(p, name)
        if p.device != x.device:
            raise ValueError(f"layer_norm: {name} is on {p.device}, x on {x.device}")
        if tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f"layer_norm: {name} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.dtype not in C.DTYPES or (wdtype is not None and p.dtype != wdtype):
            raise TypeError("layer_norm: weight and bias must share one of float32, bfloat16, float16")
        wdtype = p.dtype
    return C.F32 if wdtype is None else C.DTYPES[wdtype]


def _forward(x, weight, bias, wdtype, eps, keep):
    """y, and for the backward: the rows of x as the kernel read them, mean and 1 / deviation."""
    width = x.shape[-1]
    rows = x.numel() // width
    x2, ld = C.rows_of(x, rows, width)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    mean, rstd = (stats.data_ptr(), stats.data_ptr() + 4 * rows) if keep and rows else (None, None)
    C.check(C.lib().concord_layernorm_fwd(C.ptr(x2), ld, C.DTYPES[x.dtype], C.ptr(weight), C.ptr(bias),
                                          wdtype, rows, width, eps, C.ptr(y), width, mean, rstd,
                                          C.stream_of(x.device)), "layer_norm")
    return y, x2, ld, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, wdtype, eps):
        weight = None if weight is None else weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        y, x2, ctx.ld, stats = _forward(x, weight, bias, wdtype, eps, True)
        ctx.save_for_backward(x2, weight, stats)
        ctx.wdtype, ctx.x_shape = wdtype, x.shape
        ctx.pdtype = weight.dtype if weight is not None else None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, weight, stats = ctx.saved_tensors
        rows, width = x2.shape
        dy2, ld_dy = C.rows_of(dy, rows, width)
        dx = torch.empty(ctx.x_shape, dtype=x2.dtype, device=x2.device)
        _, need_w, need_b = ctx.needs_input_grad[:3]
        dw = torch.empty(width, dtype=ctx.pdtype, device=x2.device) if need_w else None
        db = torch.empty(width, dtype=ctx.pdtype, device=x2.device) if need_b else None
        ws = None
        if need_w or need_b:
            ws = torch.empty(int(C.lib().concord_layernorm_workspace_bytes(rows, width)), dtype=torch.uint8,
                             device=x2.device)
        C.check(C.lib().concord_layernorm_bwd(
            C.ptr(dy2), ld_dy, C.ptr(x2), ctx.ld, C.DTYPES[x2.dtype], C.ptr(weight), ctx.wdtype,
            stats.data_ptr(), stats.data_ptr() + 4 * rows, rows, width, C.ptr(dx), width, C.ptr(dw), C.ptr(db),
            C.ptr(ws), 0 if ws is None else ws.numel(), C.stream_of(x2.device)), "layer_norm backward")
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension.

    x is float32, bfloat16 or float16 of any shape; weight and bias share a
    type of their own (either may be None).  Statistics and sums are 32 bits
    wide, the result has x's type.  Differentiable once, in x, weight and
    bias; the gradients' sums over rows have a fixed order."""
    wdtype = _check(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, wdtype, float(eps))
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    return _forward(x, weight, bias, wdtype, float(eps), False)[0]


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
