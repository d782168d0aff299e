"""Embedding, norms of queries and keys with the position rotation, and activations
kept in 8 bits, forward and backward, against plain implementations in 64 bits.

Tolerances count roundings: u = 2^-24 for each one of fp32 arithmetic, half a step
(finfo.eps / 2 of the value) for the result's type, and half the smallest subnormal
where fp16 underflows."""
import math

import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(sum(ord(c) * (i + 1) for i, c in enumerate(repr(key))))


def _half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0


def _tiny(dtype):
    return 2.0 ** -25 if dtype == F16 else 2.0 ** -126


def _close(got, want, bound, dtype, what=""):
    """|got - want| <= bound (fp32 roundings) and the result's own rounding"""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    limit = bound * (1 + _half(dtype)) + want.abs() * _half(dtype) + _tiny(dtype)
    over = ((got - want).abs() - limit).detach()
    assert not torch.isnan(got).any(), what
    assert not over.numel() or float(over.max()) <= 0, (what, float(over.max()), int(over.argmax()))


# ---- embedding ----------------------------------------------------------------
def _embedding_reference(tokens, w, scale, dy):
    t = tokens.reshape(-1).long()
    there = (t >= 0) & (t < w.shape[0])
    at = torch.where(there, t, 0)
    y = w.double()[at] * there[:, None] * scale
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(dw)   # sums of magnitudes
    g = dy.double().reshape(-1, w.shape[1]) * there[:, None]
    dw.index_add_(0, at, g)
    size.index_add_(0, at, g.abs())
    count = torch.zeros(w.shape[0], dtype=torch.float64, device=DEV).index_add_(0, at, there.double())
    return y.reshape(*tokens.shape, -1), dw * scale, size * abs(scale), count


def _check_embedding(tokens, w, scale, dtype, dy):
    import concord_amd as ca
    y = ca.embedding(tokens, w, scale=scale, dtype=dtype)
    dw, = torch.autograd.grad(y, (w,), dy)
    ry, rdw, size, count = _embedding_reference(tokens, w.detach(), scale, dy)
    out = dtype or w.dtype
    assert y.dtype == out and dw.dtype == w.dtype and dw.shape == w.shape
    _close(y.detach(), ry, ry.abs() * U, out, "y")
    # count - 1 additions, the scale
    _close(dw, rdw, size * (count[:, None] + 1) * U, w.dtype, "dw")
    with torch.no_grad():
        assert torch.equal(ca.embedding(tokens, w, scale=scale, dtype=dtype), y.detach())
    again, = torch.autograd.grad(ca.embedding(tokens, w, scale=scale, dtype=dtype), (w,), dy)
    assert torch.equal(again, dw)   # a fixed order
    return y.detach(), dw


@pytest.mark.parametrize("n,vocab,width", [
    (1, 1, 1), (1, 7, 8), (3, 2, 5), (63, 65, 64), (64, 511, 40), (65, 512, 384), (1000, 3, 33), (1024, 1000, 256),
    (1025, 70000, 16), (4096, 50257, 24), (4097, 300000, 8), (5000, 65, 384), (8192, 8192, 128), (20000, 1, 72),
    (33333, 50257, 100), (131073, 513, 8)])
@pytest.mark.parametrize("table,dtype", [(F32, None), (F32, BF16), (BF16, None), (F16, F32)])
def test_embedding(n, vocab, width, table, dtype):
    g = _gen("embedding", n, vocab, width, table)
    # some tokens far commoner than the rest
    tokens = (torch.rand(n, generator=g, device=DEV) ** 4 * vocab).long().clamp_max_(vocab - 1)
    w = torch.randn(vocab, width, generator=g, device=DEV).to(table).requires_grad_(True)
    dy = torch.randn(n, width, generator=g, device=DEV).to(dtype or table)
    _check_embedding(tokens, w, 1.5, dtype, dy)


@pytest.mark.parametrize("case", ["all", "none", "some", "huge"])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_embedding_tokens_outside(case, index):
    g = _gen("outside", case)
    n, vocab, width = 3000, 500, 72
    tokens = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    if case == "all":
        tokens[:] = -1
    elif case == "some":
        tokens[torch.rand(n, generator=g, device=DEV) < 0.4] = -1
        tokens[7], tokens[-1] = vocab, vocab + 1
    elif case == "huge":
        tokens[::3] = -2 ** 31
        tokens[1::3] = 2 ** 31 - 1
    w = torch.randn(vocab, width, generator=g, device=DEV).requires_grad_(True)
    y, dw = _check_embedding(tokens.to(index), w, 1.0, None, torch.randn(n, width, generator=g, device=DEV))
    if case == "all":
        assert not y.any() and not dw.any()
    if case == "huge" and index == torch.int64:
        import concord_amd as ca
        far = tokens.clone()
        far[::3] = 2 ** 32 + 5   # its low word is a token
        assert not ca.embedding(far, w)[::3].any()


@pytest.mark.parametrize("n", [0, 1, 5])
def test_embedding_of_no_token_and_no_row(n):
    import concord_amd as ca
    w = torch.randn(9, 24, device=DEV, requires_grad=True)
    y = ca.embedding(torch.full((n, 0), 1, dtype=torch.int64, device=DEV), w)
    assert y.shape == (n, 0, 24)
    dw, = torch.autograd.grad(y, (w,), torch.zeros_like(y))
    assert dw.shape == w.shape and not dw.any()
    none = torch.empty(0, 24, device=DEV, requires_grad=True)
    y = ca.embedding(torch.zeros(n, dtype=torch.int64, device=DEV), none)
    assert y.shape == (n, 24) and not y.any()
    assert torch.autograd.grad(y, (none,), torch.ones_like(y))[0].shape == (0, 24)


def test_embedding_layouts():
    """Tokens and tables in other strides, an upstream gradient that is expanded or transposed."""
    import concord_amd as ca
    g = _gen("layouts")
    tokens = torch.randint(0, 50, (40, 30), generator=g, device=DEV).t()
    big = torch.randn(50, 100, generator=g, device=DEV)
    for w in (big[:, 3:80], big[:, :64], torch.randn(64, 50, generator=g, device=DEV).t()):
        w = w.detach().requires_grad_(True)
        dy = torch.randn(w.shape[1], 30, 40, generator=g, device=DEV).permute(1, 2, 0)
        _check_embedding(tokens, w, 2.0, None, dy)
    w = big[:, :64].detach().requires_grad_(True)
    dw, = torch.autograd.grad(ca.embedding(tokens, w).sum(), (w,))
    count = torch.bincount(tokens.reshape(-1), minlength=50).float()
    assert torch.equal(dw, count[:, None].expand(50, 64))


def test_embedding_rows_of_infinities_stay_apart():
    import concord_amd as ca
    w = torch.ones(6, 40, device=DEV)
    w[2] = math.inf
    w[3] = math.nan
    w.requires_grad_(True)
    tokens = torch.tensor([0, 2, 3, -1, 5], device=DEV)
    y = ca.embedding(tokens, w)
    assert torch.equal(y[[0, 3, 4]].detach(), torch.tensor([1.0, 0.0, 1.0], device=DEV)[:, None].expand(3, 40))
    dy = torch.ones(5, 40, device=DEV)
    dy[3] = math.nan   # of a token that stands for nothing
    dw, = torch.autograd.grad(y, (w,), dy)
    assert torch.equal(dw[:, 0], torch.tensor([1.0, 0, 1, 1, 0, 1], device=DEV))


# ---- norms of queries and keys with the rotation --------------------------------
def _rotated(x, angle, rotary, adjacent):
    """x's first `rotary` elements turned, and the sums of magnitudes that each result came from"""
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if adjacent else (x[..., :rotary // 2], x[..., rotary // 2:rotary])
    c, s = angle.cos(), angle.sin()
    u, v, m = a * c - b * s, a * s + b * c, a.abs() + b.abs()
    if adjacent:
        turned, size = torch.stack((u, v), -1).flatten(-2), torch.stack((m, m), -1).flatten(-2)
    else:
        turned, size = torch.cat((u, v), -1), torch.cat((m, m), -1)
    return torch.cat((turned, x[..., rotary:]), -1), torch.cat((size, x[..., rotary:].abs()), -1)


def _qk_reference(x, w, positions, base, rotary, adjacent, eps, dy):
    """(y, its bound, dx, its bound, dw, its bound); bounds count fp32 roundings: 13 in the sum of
    squares (half of them in r) and 5 to the norm, 4 in each sine and cosine, 3 in the turn"""
    d = x.shape[-1]
    x, dy = x.double(), dy.double()
    wd = w.double() if w is not None else torch.ones(d, dtype=torch.float64, device=DEV)
    freq = base ** (-2.0 * torch.arange(rotary // 2, device=DEV, dtype=torch.float64) / max(rotary, 1))
    angle = positions.double()[..., None, None] * freq
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = x * r
    y, size = _rotated(h * wd, angle, rotary, adjacent)
    du, du_size = _rotated(dy, -angle, rotary, adjacent)
    g, g_size = du * wd, du_size * wd.abs()
    dx = r * (g - h * (g * h).mean(-1, keepdim=True))
    dx_size = r * (g_size + h.abs() * (g_size * h.abs()).mean(-1, keepdim=True))
    over = tuple(range(x.dim() - 1))
    rows = x.numel() // d
    dw, dw_size = (du * h).sum(over), (du_size * h.abs()).sum(over)
    return y, 24 * U * size, dx, 64 * U * dx_size, dw, (32 + rows) * U * dw_size


def _check_qk(q, k, wq, wk, positions, real_positions, base=10000.0, rotary=None, adjacent=False, eps=1e-6, gen=None):
    import concord_amd as ca
    leaves = [t.detach().requires_grad_(True) for t in (q, k)] + [w for w in (wq, wk) if w is not None]
    yq, yk = ca.qk_norm_rope(leaves[0], leaves[1], wq, wk, positions=positions, base=base, rotary_dim=rotary,
                             interleaved=adjacent, eps=eps)
    dq, dk = (torch.randn(t.shape, generator=gen, device=DEV).to(t.dtype) for t in (q, k))
    grads = list(torch.autograd.grad((yq, yk), leaves, (dq, dk)))
    rot = q.shape[-1] if rotary is None else rotary
    dws = grads[2:]
    for name, x, w, y, dy, dx in (("q", q, wq, yq, dq, grads[0]), ("k", k, wk, yk, dk, grads[1])):
        ry, by, rdx, bdx, rdw, bdw = _qk_reference(x, w, real_positions, base, rot, adjacent, eps, dy)
        assert y.dtype == x.dtype and dx.dtype == x.dtype
        _close(y.detach(), ry, by, x.dtype, name)
        _close(dx, rdx, bdx, x.dtype, "d" + name)
        if w is not None:
            dw = dws.pop(0)
            assert dw.dtype == w.dtype
            _close(dw, rdw, bdw, w.dtype, "dw" + name)
    with torch.no_grad():
        plain = ca.qk_norm_rope(q, k, wq, wk, positions=positions, base=base, rotary_dim=rotary, interleaved=adjacent,
                                eps=eps)
    assert torch.equal(plain[0], yq.detach()) and torch.equal(plain[1], yk.detach())


@pytest.mark.parametrize("batch,tokens,heads,kv,dim", [
    (1, 1, 1, 1, 8), (1, 1, 32, 8, 128), (3, 1, 5, 5, 64), (2, 7, 6, 3, 40), (1, 63, 4, 1, 16), (2, 129, 20, 5, 80),
    (1, 1000, 17, 1, 96), (4, 257, 3, 3, 256), (1, 2049, 8, 2, 200), (2, 3000, 1, 1, 24)])
@pytest.mark.parametrize("dtype", TYPES)
def test_qk_norm_rope(batch, tokens, heads, kv, dim, dtype):
    g = _gen("qk", batch, tokens, heads, kv, dim, dtype)
    q = (2 * torch.randn(batch, tokens, heads, dim, generator=g, device=DEV)).to(dtype)
    k = (2 * torch.randn(batch, tokens, kv, dim, generator=g, device=DEV)).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g, device=DEV)).requires_grad_(True) for _ in range(2))
    pos = torch.arange(tokens, device=DEV).expand(batch, -1)
    _check_qk(q, k, wq, wk, None, pos, gen=g)


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 32), (64, 8), (64, 0), (80, 40), (80, 72), (128, 64), (256, 248),
                                        (8, 8), (8, 0)])
def test_qk_rotary_dims(dim, rotary, adjacent):
    g = _gen("rotary", dim, rotary, adjacent)
    q, k = (torch.randn(2, 33, h, dim, generator=g, device=DEV) for h in (5, 2))
    pos = torch.randint(-100, 5000, (2, 33), generator=g, device=DEV)
    w = (1 + 0.3 * torch.randn(dim, generator=g, device=DEV)).requires_grad_(True)
    _check_qk(q, k, w, None, pos, pos, base=500.0, rotary=rotary, adjacent=adjacent, gen=g)
    _check_qk(q, k, None, w, pos.int(), pos, base=5e5, rotary=rotary, adjacent=adjacent, gen=g)
    _check_qk(q, k, None, None, pos[1], pos[1].expand(2, -1), rotary=rotary, adjacent=adjacent, gen=g)


@pytest.mark.parametrize("far", [1 << 20, 1 << 24, (1 << 31) - 1, 1 << 40])
def test_qk_far_positions(far):
    """The angle of a far position keeps its fraction: 64 bits lose 2^-52 of far / 2 pi turns, which
    is below a rounding of fp32 up to far = 2^28; past that the reference itself loses it, so both
    get an allowance of far 2^-51."""
    import concord_amd as ca
    g = _gen("far", far)
    q = torch.randn(40, 2, 64, generator=g, device=DEV)
    pos = far - torch.arange(40, device=DEV)
    got = ca.qk_norm_rope(q, q, positions=pos)[0]
    y, bound, *_ = _qk_reference(q, None, pos, 10000.0, 64, False, 1e-6, q)
    size = bound / (24 * U)
    _close(got, y, bound + size * far * 2.0 ** -51, F32)


@pytest.mark.parametrize("wtype", TYPES)
def test_qk_weights_of_other_types(wtype):
    g = _gen("wtype", wtype)
    q, k = (torch.randn(300, h, 64, generator=g, device=DEV).to(BF16) for h in (4, 2))
    wq, wk = ((1 + 0.3 * torch.randn(64, generator=g, device=DEV)).to(wtype).requires_grad_(True) for _ in range(2))
    _check_qk(q, k, wq, wk, None, torch.arange(300, device=DEV), gen=g)


def test_qk_layouts():
    """The split of one projection's output, head-major tensors, broadcast heads, rows off 16 bytes."""
    g = _gen("qk layouts")
    qkv = torch.randn(2, 50, 8, 64, generator=g, device=DEV).to(BF16)
    pos = torch.arange(50, device=DEV).expand(2, -1)
    q, k, _ = qkv.split([4, 2, 2], dim=2)
    head_major = torch.randn(2, 4, 50, 64, generator=g, device=DEV).to(BF16).transpose(1, 2)
    off = torch.randn(2, 50, 4, 65, generator=g, device=DEV).to(BF16)[..., 1:]
    one = torch.randn(2, 50, 1, 64, generator=g, device=DEV).to(BF16).expand(2, 50, 4, 64)
    dims = torch.randn(2, 50, 64, 4, generator=g, device=DEV).to(BF16).transpose(2, 3)
    w = torch.randn(128, generator=g, device=DEV)[::2].requires_grad_(True)
    for x in (q, head_major, off, one, dims, qkv[:, :, ::2]):
        _check_qk(x, k, w, None, None, pos, gen=g)
    _check_qk(q, head_major, None, w, pos.t().contiguous().t(), pos, gen=g)


def test_qk_no_tokens_and_rows_of_zeros():
    import concord_amd as ca
    q = torch.zeros(0, 4, 64, device=DEV, dtype=BF16, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = ca.qk_norm_rope(q, q, w, w)
    dq, dw = torch.autograd.grad(y, (q, w), [torch.zeros_like(t) for t in y])
    assert y[0].shape == q.shape and dq.shape == q.shape and not dw.any()
    x = torch.zeros(5, 2, 64, device=DEV, requires_grad=True)   # eps alone under the root
    y = ca.qk_norm_rope(x, x, w, w)
    dx, dw = torch.autograd.grad(y, (x, w), [torch.ones_like(t) for t in y])
    assert not y[0].any() and not dw.any() and torch.isfinite(dx).all()


def test_qk_rows_of_nan_stay_apart():
    import concord_amd as ca
    g = _gen("nan rows")
    q = torch.randn(70, 3, 80, generator=g, device=DEV)
    clean = ca.qk_norm_rope(q, q)[0]
    bad = q.clone()
    bad[5, 1], bad[64, 0, 3] = math.nan, math.inf
    got = ca.qk_norm_rope(bad, q)[0]
    rows = torch.ones(70, 3, dtype=torch.bool, device=DEV)
    rows[5, 1] = rows[64, 0] = False
    assert torch.equal(got[rows], clean[rows]) and torch.isnan(got[5, 1]).all()


def test_qk_one_result_unused():
    import concord_amd as ca
    g = _gen("unused")
    q, k = (torch.randn(20, 2, 64, generator=g, device=DEV).requires_grad_(True) for _ in range(2))
    w = torch.ones(64, device=DEV, requires_grad=True)
    yq, _ = ca.qk_norm_rope(q, k, w, w)
    dq, dk = torch.autograd.grad(yq.sum(), (q, k))
    both = torch.autograd.grad([t.sum() for t in ca.qk_norm_rope(q, k, w, w)], (q, k))
    assert torch.equal(dq, both[0]) and not dk.any()


def test_qk_gradients_against_differences():
    """Central differences in 64 bits of the formula at random directions; fp32 gradients."""
    import concord_amd as ca
    g = _gen("differences")
    q, k = (torch.randn(6, h, 32, generator=g, device=DEV).requires_grad_(True) for h in (3, 1))
    w = (1 + 0.2 * torch.randn(32, generator=g, device=DEV)).requires_grad_(True)
    pos = torch.randint(0, 1000, (6,), generator=g, device=DEV)
    ups = [torch.randn(t.shape, generator=g, device=DEV) for t in (q, k)]
    grads = torch.autograd.grad(ca.qk_norm_rope(q, k, w, w, positions=pos), (q, k, w), ups)
    dirs = [torch.randn(t.shape, generator=g, device=DEV).double() for t in (q, k, w)]

    def f(t):
        ws = w.detach().double() + t * dirs[2]
        total = 0.0
        for x, d, up in ((q, dirs[0], ups[0]), (k, dirs[1], ups[1])):
            y, *_ = _qk_reference(x.detach().double() + t * d, ws, pos, 10000.0, 32, False, 1e-6, up)
            total = total + float((y * up.double()).sum())
        return total
    step = 1e-4
    slope = (f(step) - f(-step)) / (2 * step)
    got = sum(float((a.double() * b).sum()) for a, b in zip(grads, dirs))
    size = sum(float((a.double() * b).abs().sum()) for a, b in zip(grads, dirs))
    # fp32 gradients (64 u), and the differences' own error: step^2 of a third derivative of order 10 here
    assert abs(got - slope) <= 64 * U * size + 10 * step ** 2 * size


# ---- activations in 8 bits ---------------------------------------------------------
def _kept(x):
    """(codes, exponents, values) of the 8-bit form, in exact arithmetic: blocks of 32, the smallest
    power of two that takes the largest value to 127 or less"""
    c = x.shape[-1]
    b = torch.nn.functional.pad(x.double(), (0, -c % 32)).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    powers = (torch.arange(-126, 123, device=x.device) + 1023 << 52).view(torch.float64)
    at = torch.searchsorted(127.0 * powers, torch.nan_to_num(top, nan=0.0, posinf=0.0))
    step = powers[at]
    bad = ~torch.isfinite(b).all(-1)
    codes = (b / step[..., None]).round().masked_fill(bad[..., None], 0.0)
    most = torch.finfo(x.dtype).max
    values = (codes * step[..., None]).clamp(-most, most).masked_fill(bad[..., None], math.nan)
    exps = torch.where(bad, 255, at + 1)
    return codes.flatten(-2)[..., :c].to(torch.int8), exps.to(torch.uint8), values.flatten(-2)[..., :c]


def _same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-77.0), torch.nan_to_num(b, nan=-77.0)) and \
        torch.equal(torch.isnan(a), torch.isnan(b))


def _spread(shape, dtype, g):
    """values of many magnitudes: blocks from the type's smallest to its largest"""
    x = torch.randn(shape, generator=g, device=DEV)
    mag = torch.rand(*shape[:-1], 1, generator=g, device=DEV)
    lo, hi = (-24.0, 15.0) if dtype == F16 else (-120.0, 125.0)
    x = x * torch.exp2(lo + (hi - lo) * mag)
    most = torch.finfo(dtype).max
    return x.clamp(-most, most).to(dtype)


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 31), (1, 32), (3, 33), (2, 64), (5, 7), (7, 40), (1000, 96), (33, 1283),
                                        (129, 2051), (64, 5120), (4099, 65)])
@pytest.mark.parametrize("dtype", TYPES)
def test_pack8_is_exact(rows, width, dtype):
    import concord_amd as ca
    g = _gen("pack", rows, width, dtype)
    for x in (torch.randn(rows, width, generator=g, device=DEV).to(dtype), _spread((rows, width), dtype, g)):
        codes, exps = ca.pack8(x)
        rc, re, rv = _kept(x)
        assert codes.dtype == torch.int8 and exps.dtype == torch.uint8
        assert torch.equal(exps, re) and torch.equal(codes, rc)
        back = ca.unpack8(codes, exps, dtype)
        assert back.dtype == dtype and torch.equal(back.double(), rv)
        step = torch.exp2(exps.double() - 127).repeat_interleave(32, -1)[..., :width]
        assert ((back.double() - x.double()).abs() <= step / 2).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_pack8_edges(dtype):
    """Ties, mantissas around 127 / 64, the largest and smallest numbers, zeros, infinities and NaN."""
    import concord_amd as ca
    info = torch.finfo(dtype)
    x = torch.zeros(12, 70, device=DEV, dtype=dtype)
    x[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5], device=DEV)   # step 1: ties to even
    x[1, :3] = torch.tensor([127.5, 1.0, 3.0], device=DEV)         # step 2
    x[2, 0], x[2, 33], x[2, 69] = info.max, -info.max, info.max
    x[3, :2] = torch.tensor([info.smallest_normal, -info.tiny], device=DEV)
    x[4, 0] = 2.0 ** -24 if dtype == F16 else info.tiny * 2.0 ** -7   # subnormal
    x[5, 5] = math.inf
    x[6, 40] = -math.inf
    x[7, 69] = math.nan
    x[8, 3], x[8, 4] = math.nan, math.inf
    x[9, :] = -1.0
    x[10, ::2] = 1.9921875   # 255 / 128: above 127 / 64
    x[11, ::2] = 1.984375    # 127 / 64
    codes, exps = ca.pack8(x)
    rc, re, rv = _kept(x)
    assert torch.equal(exps, re) and torch.equal(codes, rc)
    assert _same(ca.unpack8(codes, exps, dtype).double(), rv)
    assert int(exps[5, 0]) == 255 and int(exps[5, 1]) != 255
    # another type than it came from: limited to its largest number
    if dtype != F16:
        half = ca.unpack8(codes[2:3], exps[2:3], F16)
        assert float(half.max()) == 65504.0 == -float(half.min())


def test_pack8_layouts():
    import concord_amd as ca
    g = _gen("pack layouts")
    big = torch.randn(6, 50, 200, generator=g, device=DEV).to(BF16)
    for x in (big[:, :, 5:101], big[:, :, 8:104], big[:, ::2], big.transpose(1, 2), big[:, :, ::3], big[:0], big[0, 0],
              big[0, 0, 0:1].expand(70)):
        codes, exps = ca.pack8(x)
        rc, re, rv = _kept(x.contiguous())
        assert torch.equal(codes, rc) and torch.equal(exps, re) and codes.shape == x.shape
        assert torch.equal(ca.unpack8(codes, exps, BF16).double(), rv)
    codes, exps = ca.pack8(big)
    wide = codes.new_zeros(6, 50, 201)
    wide[..., 1:] = codes
    assert torch.equal(ca.unpack8(wide[..., 1:], exps.transpose(0, 1).contiguous().transpose(0, 1), BF16),
                       ca.unpack8(codes, exps, BF16))


def _gelu64(x, tanh, dtype=F32):
    """gelu, its derivative, and the share of each that roundings may take: an exponent y rounded
    at each of three steps is 3 |y| ln 2 u of its power; 16 u cover the polynomial's error (3.2e-8 of
    Phi, half a u) and its evaluation, the reciprocal and the products.  For 16-bit types the
    polynomial is off by 8.8e-6 = 148 u, and the exponent x^2 / 2 ln 2 is rounded at two steps
    (x^2 u of the tail; nothing is left of it past |x| = 16)"""
    if tanh:
        c, a = math.sqrt(2 / math.pi), 0.044715
        u = c * (x + a * x ** 3)
        sig = torch.sigmoid(2 * u)
        rel = (16 + 3 * 2 * u.abs()) * U
        du = 2 * c * (1 + 3 * a * x ** 2)
        d = sig + x * sig * torch.sigmoid(-2 * u) * du
        return x * sig, d, rel, rel * (sig + 2 * (x * sig * torch.sigmoid(-2 * u) * du).abs())
    cdf = torch.special.erfc(-x / math.sqrt(2)) / 2   # (special.ndtr loses the left tail's digits on the GPU)
    pdf = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    rel = torch.full_like(x, 16 * U) if dtype == F32 else (16 + 148 + x.clamp(-16, 16) ** 2) * U
    return x * cdf, cdf + x * pdf, rel, rel * (cdf + (x * pdf).abs())


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 8), (3, 31), (5, 64), (129, 333), (64, 1536), (2, 4099)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tanh", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_gelu8(rows, width, dtype, tanh, gated):
    import concord_amd as ca
    g = _gen("gelu", rows, width, dtype, tanh, gated)
    # the whole range in which the normal distribution is neither 0 nor 1
    x = (torch.randn(rows, width * (2 if gated else 1), generator=g, device=DEV) * 4).to(dtype).requires_grad_(True)
    dy = torch.randn(rows, width, generator=g, device=DEV).to(dtype)
    f = ca.geglu8 if gated else ca.gelu8
    y = f(x, approximate="tanh" if tanh else "none")
    dx, = torch.autograd.grad(y, (x,), dy)
    assert y.dtype == dtype == dx.dtype and dx.shape == x.shape and y.shape == dy.shape
    d = dy.double()
    if gated:
        a, b = x.detach().double().chunk(2, -1)
        v, _, rel, _ = _gelu64(b, tanh, dtype)
        _close(y.detach(), a * v, (a * v).abs() * (rel + U) + a.abs() * 2.0 ** -120, dtype, "y")
        ka, kb = (_kept(t)[2] for t in x.detach().chunk(2, -1))
        v, dv, rel, bound = _gelu64(kb, tanh, dtype)
        _close(dx[:, :width], d * v, (d * v).abs() * (rel + U) + d.abs() * 2.0 ** -120, dtype, "da")
        _close(dx[:, width:], d * ka * dv, (d * ka).abs() * (bound + 2 * U * dv.abs() + 2.0 ** -120), dtype, "dg")
    else:
        v, _, rel, _ = _gelu64(x.detach().double(), tanh, dtype)
        _close(y.detach(), v, v.abs() * rel + 2.0 ** -120, dtype, "y")
        _, dv, _, bound = _gelu64(_kept(x.detach())[2], tanh, dtype)
        _close(dx, d * dv, d.abs() * (bound + U * dv.abs() + 2.0 ** -120), dtype, "dx")
    with torch.no_grad():
        assert torch.equal(f(x, approximate="tanh" if tanh else "none"), y.detach())


@pytest.mark.parametrize("tanh", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_gelu8_far_out(dtype, tanh):
    """Past |x| = 16 the result is x or 0 and the derivative 1 or 0, up to the type's largest number."""
    import concord_amd as ca
    most = torch.finfo(dtype).max
    x = torch.tensor([most, -most, 1e4, -1e4, 17.0, -17.0, 0.0, -0.0], device=DEV).to(dtype)
    x = x[:, None].repeat(1, 32).requires_grad_(True)   # a block of each
    y = ca.gelu8(x, approximate="tanh" if tanh else "none")
    dx, = torch.autograd.grad(y, (x,), torch.ones_like(y))
    want = x.detach().clamp_min(0)
    assert torch.equal(y.detach(), want)
    slope = torch.tensor([1.0, 0, 1, 0, 1, 0, 0.5, 0.5], device=DEV)[:, None].expand(8, 32)
    _close(dx, slope.double(), slope.double() * 164 * U + 2.0 ** -100, dtype)


def test_gelu8_infinities_and_nan_stay_in_their_block():
    import concord_amd as ca
    g = _gen("gelu nan")
    x = torch.randn(4, 128, generator=g, device=DEV)
    bad = x.clone()
    bad[1, 40] = math.nan
    bad[2, 3] = math.inf
    x.requires_grad_(True), bad.requires_grad_(True)
    y, z = ca.gelu8(x), ca.gelu8(bad)
    up = torch.ones_like(x)
    (dx,), (dz,) = torch.autograd.grad(y, (x,), up), torch.autograd.grad(z, (bad,), up)
    rest = torch.ones(4, 128, dtype=torch.bool, device=DEV)
    rest[1, 40] = rest[2, 3] = False
    assert torch.equal(y[rest], z[rest]) and torch.isnan(z[1, 40]) and float(z[2, 3].detach()) == math.inf
    rest[1, 32:64] = rest[2, :32] = False
    assert torch.equal(dx[rest], dz[rest]) and torch.isnan(dz[~rest]).all()


def test_gelu8_layouts():
    import concord_amd as ca
    g = _gen("gelu layouts")
    big = torch.randn(6, 50, 208, generator=g, device=DEV).to(BF16)
    for x in (big[:, :, 5:101], big[:, :, 8:104], big[:, ::2], big.transpose(1, 2), big[:0], big[0, 0]):
        for f in (ca.gelu8, ca.geglu8):
            a = x.detach().requires_grad_(True)
            b = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
            ya, yb = f(a), f(b)
            up = torch.randn(ya.shape, generator=g, device=DEV).to(BF16)
            wide = torch.zeros(*up.shape[:-1], up.shape[-1] + 3, device=DEV, dtype=BF16)
            wide[..., 1:-2] = up
            da, = torch.autograd.grad(ya, (a,), wide[..., 1:-2])
            db, = torch.autograd.grad(yb, (b,), up)
            assert torch.equal(ya, yb) and torch.equal(da, db)


def test_gelu8_gradient_against_differences():
    """x on a grid that the 8-bit form holds exactly, so the gradient is gelu's own."""
    import concord_amd as ca
    g = _gen("gelu differences")
    x = (torch.randint(-64, 64, (8, 64), generator=g, device=DEV) / 32.0).requires_grad_(True)
    for f, tanh in ((ca.gelu8, False), (ca.gelu8, True), (ca.geglu8, False)):
        y = f(x, approximate="tanh" if tanh else "none")
        up = torch.randn(y.shape, generator=g, device=DEV)
        dx, = torch.autograd.grad(y, (x,), up)
        direction = torch.randn(x.shape, generator=g, device=DEV).double()

        def value(t):
            z = x.detach().double() + t * direction
            if f is ca.geglu8:
                a, b = z.chunk(2, -1)
                return float((a * _gelu64(b, tanh)[0] * up.double()).sum())
            return float((_gelu64(z, tanh)[0] * up.double()).sum())
        slope = (value(1e-4) - value(-1e-4)) / 2e-4
        size = float((dx.double() * direction).abs().sum())
        assert abs(float((dx.double() * direction).sum()) - slope) <= (64 * U + 10 * 1e-8) * size


# ---- used together -----------------------------------------------------------------
def _chain(n, gen, width=128, heads=4, kv=2, vocab=50):
    """(leaves, step): tokens to a feed-forward's result and all gradients"""
    import concord_amd as ca
    dim = width // heads
    table = torch.randn(vocab, width, generator=gen, device=DEV)
    wqkv = torch.randn(width, (heads + 2 * kv) * dim, generator=gen, device=DEV) / width ** 0.5
    wfc = torch.randn(width, 4 * width, generator=gen, device=DEV) / width ** 0.5
    wq, wk = torch.ones(dim, device=DEV), torch.ones(dim, device=DEV)
    leaves = [t.requires_grad_(True) for t in (table, wqkv, wq, wk, wfc)]
    tokens = torch.randint(-1, vocab, (n,), generator=gen, device=DEV)
    positions = torch.arange(n, device=DEV)
    up = torch.randn(n, 2 * width, generator=gen, device=DEV).to(BF16)

    def step():
        x = ca.embedding(tokens, table, scale=2.0)
        qkv = torch.matmul(ca.layer_norm(x), wqkv).to(BF16).view(n, heads + 2 * kv, dim)
        q, k, v = qkv.split([heads, kv, kv], dim=1)
        q, k = ca.qk_norm_rope(q, k, wq, wk, positions=positions)
        x = x + ca.attention(q, k, v).reshape(n, width)
        y = ca.geglu8(ca.gelu8(torch.matmul(ca.layer_norm(x), wfc).to(BF16)))
        return [y] + list(torch.autograd.grad(y, leaves, up))
    return leaves, tokens, up, step


def test_chain_against_plain_operators():
    """Embedding, norms and rotation, attention and both activations in one graph, against the same
    with torch's operators in fp32 and every bf16 rounding of activations at its place.  Roundings
    that fall otherwise (2^-8 of a value, at 5 places forward and as many backward) and the 8-bit
    steps (2^-7 of a block's largest at 2 places, both sides' the same but where a value differs
    already) leave 2^-3.5 of a gradient's norm at most, 2^-5 of the result's."""
    import concord_amd as ca
    leaves, tokens, up, step = _chain(150, _gen("chain"))
    got = [t.detach().double() for t in step()]
    table, wqkv, wq, wk, wfc = leaves

    class Kept(torch.autograd.Function):   # f(x), its gradient at the 8-bit form of x
        @staticmethod
        def forward(ctx, x, f):
            ctx.f, ctx.z = f, x
            return f(x)

        @staticmethod
        def backward(ctx, dy):
            halves = ctx.z.chunk(2, -1) if ctx.f is gated else (ctx.z,)
            z = torch.cat([_kept(h)[2] for h in halves], -1).to(ctx.z.dtype).requires_grad_(True)
            with torch.enable_grad():
                y = ctx.f(z)
            return torch.autograd.grad(y, z, dy)[0], None

    def gelu(x):
        return torch.nn.functional.gelu(x.float()).to(x.dtype)

    def gated(x):
        a, b = x.chunk(2, -1)
        return (a.float() * torch.nn.functional.gelu(b.float())).to(x.dtype)

    def norm_rope(x, w):
        h = x.float() * (x.float().square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        half = x.shape[-1] // 2
        angle = torch.arange(x.shape[0], device=DEV)[:, None, None] * 10000.0 ** (
            -torch.arange(half, device=DEV, dtype=torch.float64) / half)
        c, s = angle.cos().float(), angle.sin().float()
        return torch.cat((h[..., :half] * c - h[..., half:] * s, h[..., :half] * s + h[..., half:] * c), -1).to(BF16)
    n, width, heads, kv, dim = 150, 128, 4, 2, 32
    x = table[tokens.clamp_min(0)] * (tokens >= 0)[:, None] * 2.0
    qkv = torch.matmul(torch.nn.functional.layer_norm(x, (width,)), wqkv).to(BF16).view(n, heads + 2 * kv, dim)
    q, k, v = qkv.split([heads, kv, kv], dim=1)
    q, k = norm_rope(q, wq), norm_rope(k, wk)
    qf, kf, vf = (t.float().transpose(0, 1) for t in (q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)))
    z = torch.matmul(qf, kf.transpose(1, 2).contiguous()) / dim ** 0.5
    z = z.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), -math.inf)
    x = x + torch.matmul(z.softmax(-1), vf).to(BF16).transpose(0, 1).reshape(n, width)
    y = Kept.apply(Kept.apply(torch.matmul(torch.nn.functional.layer_norm(x, (width,)), wfc).to(BF16), gelu), gated)
    want = [y.detach().double()] + [t.double() for t in torch.autograd.grad(y, leaves, up)]
    for i, (a, b) in enumerate(zip(got, want)):
        assert float((a - b).norm()) <= 2.0 ** (-5 if i == 0 else -3.5) * float(b.norm()), i


def test_chain_in_a_captured_step():
    """One HIP graph of the step, replayed with new inputs and with eager work between the replays:
    the eager results, bit for bit."""
    gen = _gen("graph")
    leaves, tokens, up, step = _chain(700, gen)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [t.detach() for t in step()]
    for _ in range(4):
        with torch.no_grad():
            tokens.copy_(torch.randint(-1, 50, tokens.shape, generator=gen, device=DEV))
            leaves[0].copy_(torch.randn(leaves[0].shape, generator=gen, device=DEV))
        graph.replay()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n,vocab", [(300, 70000), (6000, 65), (70000, 300)])
def test_embedding_gradient_in_a_graph(n, vocab):
    """Each of the sort's forms, captured and replayed with other tokens."""
    import concord_amd as ca
    gen = _gen("embedding graph", n)
    tokens = torch.randint(0, vocab, (n,), generator=gen, device=DEV)
    w = torch.randn(vocab, 40, generator=gen, device=DEV, requires_grad=True)
    dy = torch.randn(n, 40, generator=gen, device=DEV)

    def step():
        return torch.autograd.grad(ca.embedding(tokens, w), (w,), dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        tokens.copy_(torch.randint(-3, vocab + 3, (n,), generator=gen, device=DEV))
        graph.replay()
        got = held.clone()
        assert torch.equal(got, step())


def test_streams_do_not_share_anything():
    """The same calls on two streams at once give what each gives alone."""
    import concord_amd as ca
    gen = _gen("streams")
    jobs = []
    for n, vocab in ((9000, 300), (9000, 300)):
        tokens = torch.randint(0, vocab, (n,), generator=gen, device=DEV)
        w = torch.randn(vocab, 256, generator=gen, device=DEV, requires_grad=True)
        q = torch.randn(n, 4, 64, generator=gen, device=DEV).to(BF16).requires_grad_(True)
        x = torch.randn(n, 256, generator=gen, device=DEV).to(BF16).requires_grad_(True)
        qw = torch.ones(64, device=DEV, requires_grad=True)
        jobs.append((tokens, w, q, qw, x))

    def run(tokens, w, q, qw, x):
        y = ca.embedding(tokens, w)
        a, b = ca.qk_norm_rope(q, q, qw, qw)
        z = ca.gelu8(x)
        return torch.autograd.grad([y, a, b, z], [w, q, qw, x], [torch.ones_like(t) for t in (y, a, b, z)])
    alone = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], []
    for _ in range(3):
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(run(*j))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, alone[i % 2]))


def test_block_operators_are_differentiable_once():
    import concord_amd as ca
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    q = torch.randn(4, 1, 64, device=DEV, requires_grad=True)
    idx = torch.zeros(4, dtype=torch.int64, device=DEV)
    for y, leaf in ((ca.embedding(idx, x), x), (ca.qk_norm_rope(q, q)[0], q), (ca.gelu8(x), x), (ca.geglu8(x), x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


def test_block_operators_see_a_change_of_a_saved_tensor():
    import concord_amd as ca
    q = torch.randn(4, 2, 64, device=DEV, requires_grad=True)
    tokens = torch.zeros(4, dtype=torch.int64, device=DEV)
    w = torch.randn(5, 64, device=DEV, requires_grad=True)
    y, (z, _) = ca.embedding(tokens, w), ca.qk_norm_rope(q * 1.0, q * 1.0, positions=tokens)
    tokens.add_(1)
    for t in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            t.sum().backward()


def test_modules():
    import concord_amd as ca
    e = ca.Embedding(11, 48, scale=3.0, device=DEV, out_dtype=BF16)
    t = torch.tensor([[1, 10], [-1, 0]], device=DEV, dtype=torch.int32)
    assert e(t).dtype == BF16 and torch.equal(e(t), ca.embedding(t, e.weight, 3.0, BF16)) and e(t).requires_grad
    m = ca.QKNormRope(64, base=500.0, rotary_dim=32, interleaved=True, eps=1e-5, device=DEV)
    q = torch.randn(2, 7, 3, 64, device=DEV)
    got, want = m(q, q[:, :, :1]), ca.qk_norm_rope(q, q[:, :, :1], m.q_weight, m.k_weight, None, 500.0, 32, True, 1e-5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert [p.shape for p in m.parameters()] == [(64,), (64,)]


# ---- the packed linear's input in 8 bits ------------------------------------------------
@pytest.mark.parametrize("N,K,M", [(64, 96, 70), (136, 333, 50), (256, 512, 300)])
def test_linear_input_in_8_bits(N, K, M):
    """Forward and the input's gradient are bit for bit those of the bf16 input; the weight gradient,
    v-hat and update are bit for bit those of a layer whose input is the 8-bit form's values."""
    import concord_amd as ca
    from concord_amd import packed_b as pb
    g = _gen("linear 8", N, K)
    W = torch.randn(N, K, generator=g, device=DEV) * 0.05
    x = torch.randn(M, K, generator=g, device=DEV).to(BF16)
    kept = ca.unpack8(*ca.pack8(x))
    dy = (torch.randn(M, N, generator=g, device=DEV) * 1e-2).to(BF16)

    def run(inp, bits):
        pb._get_step_counter(torch.device(DEV)).zero_()
        layer = ca.ConcordLinearPackedB(K, N, bias=True, device=DEV, lr=5e-3)
        layer.load_weights(W)
        layer.set_input_bits(bits)
        leaf = inp.clone().requires_grad_(True)
        y = layer(leaf)
        y.backward(dy)
        return y.detach(), leaf.grad, layer
    y16, dx16, _ = run(x, 16)
    y8, dx8, layer8 = run(x, 8)
    _, _, want = run(kept, 16)
    assert torch.equal(y8, y16) and torch.equal(dx8, dx16)
    for n, t in want.state_dict().items():
        if isinstance(t, torch.Tensor):
            assert torch.equal(layer8.state_dict()[n], t), n
    assert torch.equal(layer8.bias.grad, want.bias.grad)
    with torch.no_grad():
        assert torch.equal(layer8(x), layer8(x))


def test_linear_keeps_33_bytes_for_32_values():
    import concord_amd as ca
    layer = ca.ConcordLinearPackedB(1024, 64, bias=False, device=DEV)
    layer.set_input_bits(8)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        layer(torch.randn(8, 1024, device=DEV, requires_grad=True))
    assert sorted(t.numel() * t.element_size() for t in saved) == [8 * 32, 8 * 1024]


@pytest.mark.parametrize("rotary,keep8", [(True, False), (False, True), (True, True)])
def test_example_runs(rotary, keep8):
    from examples import distill_gpt as ex
    m = ex.GPT(layers=2, device=DEV, rotary=rotary, keep8=keep8)
    batch = ex.documents(700, 65, 256, torch.Generator().manual_seed(1), DEV)
    m(*batch).float().square().mean().backward()
    layers = {id(p) for c in m.concord_layers() for p in c.parameters()}
    own = [p for p in m.parameters() if id(p) not in layers]
    assert len(own) > 5 and all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any() for p in own)
    assert all(math.isfinite(v) for v in ex.train(2, tokens=600, device=DEV, rotary=rotary, keep8=keep8))


# ---- offsets past 32 bits ------------------------------------------------------------------
def test_embedding_offsets_past_32_bits():
    """2^31 elements and more of the result, of its gradient and of the table."""
    import concord_amd as ca
    n, width, vocab = 33000, 65600, 33001
    w = torch.zeros(vocab, width, device=DEV, dtype=BF16)
    w[-1], w[5] = 3.0, 2.0
    w.requires_grad_(True)
    tokens = torch.full((n,), 7, device=DEV)
    tokens[-1], tokens[-2] = vocab - 1, 5
    y = ca.embedding(tokens, w)
    assert (y[-1] == 3).all() and (y[-2] == 2).all() and not y[-3].any()
    dy = torch.zeros(n, width, device=DEV, dtype=BF16)
    dy[-1], dy[-2], dy[0] = 0.5, 0.25, 1.0
    dw, = torch.autograd.grad(y, (w,), dy)
    assert (dw[-1] == 0.5).all() and (dw[5] == 0.25).all() and (dw[7] == 1).all() and not dw[-2].any() and not dw[0].any()


def test_qk_offsets_past_32_bits():
    import concord_amd as ca
    n, heads, dim = 131100, 128, 128
    q = torch.ones(n, heads, dim, device=DEV, dtype=BF16)
    g = _gen("large qk")
    last = torch.randn(3, heads, dim, generator=g, device=DEV).to(BF16)
    q[-3:] = last
    q.requires_grad_(True)
    k = torch.ones(n, 1, dim, device=DEV, dtype=BF16)
    pos = torch.arange(n, device=DEV)
    y, _ = ca.qk_norm_rope(q, k, positions=pos)
    dq, = torch.autograd.grad(y, (q,), y.detach().flip(2).contiguous())
    part = q.detach()[-3:].clone().requires_grad_(True)
    z, _ = ca.qk_norm_rope(part, k[-3:], positions=pos[-3:])
    dz, = torch.autograd.grad(z, (part,), z.detach().flip(2).contiguous())
    # (few tokens and many take lanes of other widths: sums in another order, so a rounding apart)
    _close(y.detach()[-3:], z.detach().double(), z.detach().double().abs() * 2.0 ** -8 + 24 * U, BF16)
    _close(dq[-3:], dz.double(), dz.double().abs() * 2.0 ** -8 + 64 * U * 16, BF16)


@pytest.mark.parametrize("width", [4096, 4099])
def test_act8_offsets_past_32_bits(width):
    import concord_amd as ca
    rows = 2 ** 31 // 4096 + 10
    x = torch.zeros(rows, width, device=DEV, dtype=BF16)
    g = _gen("large act", width)
    x[-2:] = torch.randn(2, width, generator=g, device=DEV).to(BF16)
    x.requires_grad_(True)
    y = ca.gelu8(x)
    dx, = torch.autograd.grad(y, (x,), torch.ones_like(y))
    small = x.detach()[-2:].clone().requires_grad_(True)
    z = ca.gelu8(small)
    dz, = torch.autograd.grad(z, (small,), torch.ones_like(z))
    assert torch.equal(y[-2:], z) and torch.equal(dx[-2:], dz) and not y[-3].any() and (dx[-3] == 0.5).all()
    codes, exps = ca.pack8(x.detach())
    assert torch.equal(ca.unpack8(codes, exps, BF16)[-2:].double(), _kept(small.detach())[2])
