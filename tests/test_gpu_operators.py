"""Layer norm, attention and distillation against plain 64-bit implementations
on the CPU, forward and backward.

Tolerances are elementwise bounds derived from the arithmetic: u is half a
unit in the last place of the stored type (2^-24, 2^-8 bf16, 2^-11 fp16), and
a value rounded to it is off by at most u of itself.  Sums in 32 bits of n
terms, chained at most 64 deep before a tree, are off by at most 2^-24 (64 +
log2 n) of the sum of magnitudes; EPS32 = 2^-17 covers that with the handful of
roundings around it."""
import math
import zlib

import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EPS32 = 2.0 ** -17
# smallest magnitudes: below them a type rounds by a fixed step
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 6e-8}


def _close(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()),
                           float(((got - want).abs() / bound.clamp_min(1e-300)).max()), bad.nonzero()[:4].tolist())


def _gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


# ---- layer norm ---------------------------------------------------------------
def _norm_ref(x, w, b, dy, eps):
    """y, dx, dw, db in 64 bits and, for each, the bound of a 32-bit evaluation"""
    n = x.shape[1]
    mu = x.mean(1, keepdim=True)
    c = x - mu
    r = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    h = c * r
    y = h * w + b
    # the mean is off by EPS32 of the row's mean magnitude, which moves h
    eh = EPS32 * ((x.abs() + x.abs().mean(1, keepdim=True)) * r + h.abs() + 1e-30)
    out = {"y": (y, eh * w.abs() + EPS32 * (h * w).abs() + 2.0 ** -23 * b.abs())}
    g = dy * w
    ga, m = g.abs(), lambda t: t.mean(1, keepdim=True)  # noqa: E731
    dx = r * (g - m(g) - h * m(g * h))
    e = EPS32 * (ga + m(ga) + h.abs() * m(ga * h.abs())) + eh * m(ga * h.abs()) + h.abs() * m(ga * eh)
    out["dx"] = (dx, r * e + EPS32 * dx.abs())
    out["dw"] = ((dy * h).sum(0), (EPS32 * (dy * h).abs() + dy.abs() * eh).sum(0) + 1e-30)
    out["db"] = (dy.sum(0), EPS32 * dy.abs().sum(0) + 1e-30)
    assert n == w.numel()
    return out


def _norm_case(rows, width, dtype, wdtype=torch.float32, offset=0.3):
    g = _gen("norm", rows, width, str(dtype))
    x = (torch.randn(rows, width, generator=g) * (1 + 10 * (torch.rand(width, generator=g) < 0.02)) + offset).to(dtype)
    dy = torch.randn(rows, width, generator=g).to(dtype)
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(wdtype)
    b = (0.2 * torch.randn(width, generator=g)).to(wdtype)
    return x, w, b, dy


def _norm_check(x, w, b, dy, eps=1e-5, to=lambda t: t.to(DEV)):
    import concord_amd as ca
    dt, wt = x.dtype, w.dtype
    ref = _norm_ref(x.double(), w.double(), b.double(), dy.double(), eps)
    xd, wd, bd = (to(t).requires_grad_(True) for t in (x, w, b))
    y = ca.layer_norm(xd, wd, bd, eps)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), to(dy))
    with torch.no_grad():
        assert torch.equal(ca.layer_norm(xd, wd, bd, eps), y)
    assert y.dtype == dx.dtype == dt and dw.dtype == db.dtype == wt
    for name, got, t in (("y", y, dt), ("dx", dx, dt), ("dw", dw, wt), ("db", db, wt)):
        want, e = ref[name]
        _close(got, want, e + U[t] * (want.abs() + e) + TINY[t], name)


# one column, one vector and its neighbours, each count of waves a row takes
# and its ends, rows longer than a block holds
@pytest.mark.parametrize("rows,width", [
    (70, 24), (130, 120), (65, 128), (66, 129), (600, 33),
    (1, 1), (3, 2), (5, 7), (4, 8), (1, 384), (130, 384), (7, 511), (7, 512), (9, 513), (6, 1000), (5, 1024),
    (5, 1025), (1, 1280), (3, 2048), (3, 2051), (2, 4096), (3, 4097), (2, 8192), (2, 8200), (2, 12288), (2, 16384),
    (2, 16385), (3, 20000), (2500, 64), (1100, 1032)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_layer_norm_sizes(rows, width, dtype):
    _norm_check(*_norm_case(rows, width, dtype))


@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float16])
def test_layer_norm_weight_types(wdtype):
    _norm_check(*_norm_case(33, 640, torch.bfloat16, wdtype))


def test_layer_norm_large_offset():
    """A mean 1000 times the deviation: the squares are taken about the mean."""
    x, w, b, dy = _norm_case(16, 1536, torch.float32, offset=1000.0)
    _norm_check(x, w, b, dy)


@pytest.mark.parametrize("layout", ["cols", "rows", "transposed", "misaligned", "expanded"])
def test_layer_norm_strides(layout):
    def to(t):
        t = t.to(DEV)
        if t.dim() == 1:
            return t
        n, c = t.shape
        if layout == "cols":
            big = torch.full((n, c + 24), float("nan"), dtype=t.dtype, device=DEV)
            big[:, 8:8 + c] = t
            return big[:, 8:8 + c].detach()
        if layout == "rows":
            big = torch.full((2 * n, c), float("nan"), dtype=t.dtype, device=DEV)
            big[::2] = t
            return big[::2].detach()
        if layout == "transposed":
            return t.t().contiguous().t().detach()
        if layout == "misaligned":
            return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(n, c).detach()
        return t
    x, w, b, dy = _norm_case(21, 264, torch.bfloat16)
    if layout == "expanded":
        dy = dy[:1].expand(21, 264)
    _norm_check(x, w, b, dy, to=to)


def test_layer_norm_empty_and_partial():
    import concord_amd as ca
    x = torch.zeros(0, 48, device=DEV, requires_grad=True)
    m = ca.LayerNorm(48, device=DEV)
    y = m(x)
    y.sum().backward()
    assert y.shape == x.shape and x.grad.shape == x.shape
    assert float(m.weight.grad.abs().sum()) == 0.0 and float(m.bias.grad.abs().sum()) == 0.0
    # no weight, no bias, a gradient of one of the three alone; three dimensions
    x, w, b, dy = _norm_case(12, 96, torch.float32)
    ref = _norm_ref(x.double(), torch.ones(96, dtype=torch.float64), torch.zeros(96, dtype=torch.float64),
                    dy.double(), 1e-3)
    xd = x.to(DEV).view(3, 4, 96).requires_grad_(True)
    y = ca.layer_norm(xd, eps=1e-3)
    dx, = torch.autograd.grad(y, xd, dy.to(DEV).view(3, 4, 96))
    for got, name in ((y, "y"), (dx, "dx")):
        want, e = ref[name]
        _close(got, want.view(3, 4, 96), (e + U[torch.float32] * want.abs()).view(3, 4, 96) + 1e-30, name)
    wd = w.to(DEV).requires_grad_(True)
    dw, = torch.autograd.grad(ca.layer_norm(x.to(DEV), wd, None), wd, dy.to(DEV))
    want, e = _norm_ref(x.double(), w.double(), 0 * b.double(), dy.double(), 1e-5)["dw"]
    _close(dw, want, e + U[torch.float32] * want.abs(), "dw")


def test_layer_norm_differences():
    """Central differences of the 32-bit forward along a random direction."""
    import concord_amd as ca
    x, w, b, dy = (t.to(DEV) for t in _norm_case(9, 200, torch.float32))
    p = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ca.layer_norm(*p), p, dy)
    g = _gen("fd")
    h = 2.0 ** -7
    for i in range(3):
        u = torch.randn(p[i].shape, generator=g).to(DEV)
        vals = []
        for s in (h, -h):
            q = [t.detach() for t in p]
            q[i] = q[i] + s * u
            vals.append((ca.layer_norm(*q).double() * dy.double()).sum())
        num, ana = float(vals[0] - vals[1]) / (2 * h), float((grads[i].double() * u.double()).sum())
        size = float((grads[i].double() * u.double()).abs().sum())
        # third derivatives times h^2, and rounding of the sums over 2 h
        assert abs(num - ana) <= 20 * h * h * size + 1e-5 * float(dy.abs().sum()) / h, (i, num, ana)


def test_layer_norm_is_reproducible():
    import concord_amd as ca
    x, w, b, dy = (t.to(DEV) for t in _norm_case(3000, 768, torch.bfloat16))
    p = [t.requires_grad_(True) for t in (x, w, b)]
    first = torch.autograd.grad(ca.layer_norm(*p), p, dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(ca.layer_norm(*p), p, dy)))


# ---- attention ----------------------------------------------------------------
def _seqs(starts, k_starts, tq, tk):
    """(query rows, key rows) of each sequence"""
    return [(slice(a, b), slice(c, d)) for a, b, c, d in zip(starts, starts[1:], k_starts, k_starts[1:])]


def _attn_ref(q, k, v, g, starts, k_starts, causal, scale):
    """out, dq, dk, dv in 64 bits, each with its bound: the probabilities and
    the scores' gradients are rounded to bf16, out too before delta is formed
    from it"""
    u, e32 = U[torch.bfloat16], EPS32
    h, hk = q.shape[1], k.shape[1]
    rep = h // hk
    res = {n: (torch.zeros(t.shape, dtype=torch.float64), torch.zeros(t.shape, dtype=torch.float64))
           for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    for rq, rk in _seqs(starts, k_starts, len(q), len(k)):
        lq, lk = rq.stop - rq.start, rk.stop - rk.start
        if lq <= 0 or lk <= 0:
            continue
        for a in range(h):
            qa, ga, ka, va = q[rq, a], g[rq, a], k[rk, a // rep], v[rk, a // rep]
            s = qa @ ka.T * scale
            # scores are off by EPS32 of their terms' magnitudes; so are the probabilities, relatively
            es = e32 * (1 + (qa.abs() @ ka.abs().T) * scale)
            if causal:
                hidden = torch.arange(lk) > torch.arange(lq)[:, None] + (lk - lq)
                s = s.masked_fill(hidden, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, 1))
            ep = p * (es + (p * es).sum(1, keepdim=True))
            o = p @ va
            pv = p @ va.abs()
            eo = (u * p + ep) @ va.abs() + e32 * pv
            res["out"][0][rq, a] = o
            res["out"][1][rq, a] = eo + u * (o.abs() + eo)
            eo_b = eo + u * (o.abs() + eo)
            dp = ga @ va.T
            delta = (ga * o).sum(1, keepdim=True)
            ed = (ga.abs() * eo_b).sum(1, keepdim=True) + e32 * (ga.abs() * o.abs()).sum(1, keepdim=True)
            ds = p * (dp - delta)
            eds = ep * (dp - delta).abs() + p * (ed + e32 * (ga.abs() @ va.abs().T))
            eds = eds + u * (ds.abs() + eds)
            dq = ds @ ka * scale
            edq = (eds @ ka.abs() + e32 * ds.abs() @ ka.abs()) * scale
            res["dq"][0][rq, a] = dq
            res["dq"][1][rq, a] = edq
            res["dk"][0][rk, a // rep] += ds.T @ qa * scale
            res["dk"][1][rk, a // rep] += (eds.T @ qa.abs() + e32 * ds.abs().T @ qa.abs()) * scale
            res["dv"][0][rk, a // rep] += p.T @ ga
            res["dv"][1][rk, a // rep] += (u * p + ep).T @ ga.abs() + e32 * p.T @ ga.abs()
    for n in ("dq", "dk", "dv"):
        want, e = res[n]
        res[n] = (want, e + u * (want.abs() + e))
    return res


def _attn_inputs(tq, tk, h, hk, d, spread=1.5):
    gen = _gen("attn", tq, tk, h, hk, d)
    q = (spread * torch.randn(tq, h, d, generator=gen)).to(torch.bfloat16)
    k, v = (torch.randn(tk, hk, d, generator=gen).to(torch.bfloat16) for _ in range(2))
    return q, k, v, torch.randn(tq, h, d, generator=gen).to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _attn_check(q, k, v, g, starts=None, k_starts=None, causal=True, scale=None, tables=True, view=None):
    """tables: give the kernel `starts`; else it has the one sequence"""
    import concord_amd as ca
    s = starts or [0, len(q)]
    ks = k_starts or (starts if starts and len(q) == len(k) else [0, len(k)])
    ref = _attn_ref(*(t.double() for t in (q, k, v, g)), s, ks, causal, scale or 1 / math.sqrt(q.shape[2]))
    view = view or (lambda t: t.to(DEV))
    qd, kd, vd = (view(t).detach().requires_grad_(True) for t in (q, k, v))
    kw = dict(causal=causal, scale=scale)
    if tables:
        kw.update(starts=_i32(s), k_starts=_i32(ks) if k_starts or len(q) != len(k) else None)
    out = ca.attention(qd, kd, vd, **kw)
    with torch.no_grad():
        assert torch.equal(ca.attention(qd, kd, vd, **kw), out)
    grads = torch.autograd.grad(out, (qd, kd, vd), view(g).detach())
    for name, got in (("out", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        want, e = ref[name]
        _close(got.reshape(want.shape), want, e + 1e-30, name)
    return out, grads


@pytest.mark.parametrize("d", [8, 16, 32, 40, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_head_dimensions(d, causal):
    _attn_check(*_attn_inputs(150, 150, 2, 1, d), causal=causal)


# one token, ends of the 32-row wave, the 64-key step and the 128-row tile
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 257, 300])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_lengths(n, d):
    _attn_check(*_attn_inputs(n, n, 2, 2, d), tables=False)
    _attn_check(*_attn_inputs(n, n, 2, 2, d), causal=False, tables=False)


@pytest.mark.parametrize("h,hk", [(1, 1), (4, 4), (4, 2), (6, 1), (8, 2), (9, 3)])
def test_attention_grouped_heads(h, hk):
    _attn_check(*_attn_inputs(140, 140, h, hk, 64), starts=[0, 40, 140])


# queries and keys of different number: cross-attention, a prompt continued
# after a prefix, and more queries than keys, whose first rows see nothing
@pytest.mark.parametrize("tq,tk", [(1, 77), (1, 300), (200, 77), (70, 1), (33, 200), (129, 64), (200, 130), (64, 65)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_other_key_counts(tq, tk, causal, d):
    _attn_check(*_attn_inputs(tq, tk, 2, 1, d), causal=causal)


# empty sequences at the ends and inside, single tokens, sequences that end on
# and beside tile boundaries
PACKED = [
    [0, 1, 2, 5, 133, 133, 261, 390],
    [0, 0, 128, 256, 256, 256, 300],
    [0, 64, 128, 192, 320, 321],
    [0] + list(range(3, 214, 3)),
    [0, 129, 129],
]


@pytest.mark.parametrize("starts", PACKED)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_packed_sequences(starts, causal, d):
    _attn_check(*_attn_inputs(starts[-1], starts[-1], 4, 2, d), starts=starts, causal=causal)


@pytest.mark.parametrize("causal", [True, False])
def test_attention_packed_with_other_keys(causal):
    s, ks = [0, 5, 5, 140, 200, 201, 260], [0, 3, 70, 70, 300, 301, 301]
    _attn_check(*_attn_inputs(260, 301, 4, 2, 64), starts=s, k_starts=ks, causal=causal)


@pytest.mark.parametrize("causal", [True, False])
def test_attention_many_sequences(causal):
    """More sequences than one look-up of the table covers."""
    gen = _gen("many")
    lens = torch.randint(0, 5, (5000,), generator=gen).tolist()
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    q, k, v, g = _attn_inputs(starts[-1], starts[-1], 1, 1, 32)
    _attn_check(q, k, v, g, starts=starts, causal=causal)


def test_attention_tokens_outside_the_sequences():
    """Rows before the first and after the last sequence: 0, whatever stands there."""
    q, k, v, g = _attn_inputs(400, 400, 2, 2, 64)
    for t in (q, k, v, g):
        t[:37] = float("nan")
        t[250:] = float("inf")
    import concord_amd as ca
    qd, kd, vd = (t.to(DEV).requires_grad_(True) for t in (q, k, v))
    out = ca.attention(qd, kd, vd, starts=_i32([37, 100, 250]))
    grads = torch.autograd.grad(out, (qd, kd, vd), g.to(DEV))
    for t in (out.detach(), *grads):
        assert float(t[:37].abs().sum()) == 0.0 and float(t[250:].abs().sum()) == 0.0
    ref = _attn_ref(*(t[37:250].double() for t in (q, k, v, g)), [0, 63, 213], [0, 63, 213], True, 0.125)
    for name, got in (("out", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        _close(got[37:250], ref[name][0], ref[name][1] + 1e-30, name)


def test_attention_table_past_the_tensors():
    """Positions past the tensors are their ends; nothing outside is touched."""
    import concord_amd as ca
    q, k, v, g = (t.to(DEV) for t in _attn_inputs(200, 200, 2, 2, 64))
    want = ca.attention(q, k, v, starts=_i32([0, 90, 200]))
    got = ca.attention(q, k, v, starts=_i32([-5, 90, 100000]))
    assert torch.equal(got, want)


def test_attention_keys_of_other_sequences_do_not_leak():
    """A sequence's result does not see infinities and NaN next to it."""
    import concord_amd as ca
    q, k, v, g = _attn_inputs(300, 300, 2, 1, 128)
    for t in (q, k, v, g):
        t[:70] = float("nan")
        t[170:] = float("inf")
    qd, kd, vd = (t.to(DEV).requires_grad_(True) for t in (q, k, v))
    for causal in (True, False):
        out = ca.attention(qd, kd, vd, starts=_i32([0, 70, 170, 300]), causal=causal)
        grads = torch.autograd.grad(out, (qd, kd, vd), g.to(DEV))
        ref = _attn_ref(*(t[70:170].double() for t in (q, k, v, g)), [0, 100], [0, 100], causal, 1 / math.sqrt(128))
        for name, got in (("out", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
            _close(got[70:170], ref[name][0], ref[name][1] + 1e-30, name)


@pytest.mark.parametrize("spread", [40.0, 1e-3])
def test_attention_score_ranges(spread):
    """Scores of hundreds (a softmax of nearly one key, a maximum that grows over
    the keys) and of nearly nothing."""
    q, k, v, g = _attn_inputs(260, 260, 2, 2, 64, spread=spread)
    k = (k.float() * torch.linspace(0.2, 2.0, 260)[:, None, None]).to(torch.bfloat16)
    _attn_check(q, k, v, g)
    _attn_check(q, k.flip(0), v, g, causal=False)


@pytest.mark.parametrize("tq,tk,h,hk,d,causal", [
    (2048, 2048, 4, 1, 64, True), (1500, 1500, 8, 2, 128, True), (1200, 333, 2, 1, 64, False),
    (900, 900, 6, 2, 96, True), (1000, 1500, 2, 1, 128, False)])
def test_attention_few_tiles(tq, tk, h, hk, d, causal):
    """Too few tiles to fill the chip: the work along the long axis is split and
    joined (backward: dk and dv over the queries)."""
    q, k, v, g = _attn_inputs(tq, tk, h, hk, d)
    _attn_check(q, k, v, g, causal=causal, tables=False)
    if tq == tk:
        _attn_check(q, k, v, g, starts=[0, 3, 3, 700, tq], causal=causal)


@pytest.mark.parametrize("tq,tk,h,hk,d,causal", [
    (1, 5000, 4, 1, 64, True), (1, 4097, 8, 2, 128, False), (40, 3000, 2, 2, 96, True), (130, 2500, 2, 1, 128, True),
    (200, 1700, 1, 1, 32, False)])
def test_attention_few_queries(tq, tk, h, hk, d, causal):
    """Few queries of many keys: the keys are split and joined."""
    q, k, v, g = _attn_inputs(tq, tk, h, hk, d)
    _attn_check(q, k, v, g, causal=causal)
    _attn_check(q, k, v, g, starts=[0, 0, tq // 2, tq, tq], k_starts=[0, 1, 1200, tk - 1, tk], causal=causal)


def test_attention_scale():
    _attn_check(*_attn_inputs(90, 90, 2, 2, 64), scale=0.7)
    _attn_check(*_attn_inputs(90, 90, 2, 2, 64), scale=1e-4)


@pytest.mark.parametrize("layout", ["projection", "head_major", "odd_rows", "misaligned", "expanded_heads",
                                    "expanded_tokens"])
def test_attention_strides(layout):
    q, k, v, g = _attn_inputs(150, 150, 4, 4, 64)
    if layout == "expanded_heads":
        k, v = (t[:, :1].expand(-1, 4, -1) for t in (k, v))
    if layout == "expanded_tokens":
        g = g[:1].expand(150, -1, -1)

    def view(t):
        if layout.startswith("expanded"):
            return t.to(DEV) if 0 not in t.stride() else t[:1].to(DEV).expand(t.shape) if t.stride(0) == 0 else \
                t[:, :1].to(DEV).expand(t.shape)
        t = t.to(DEV)
        n, h, d = t.shape
        if layout == "projection":
            big = torch.full((n, 3 * h + 1, d), float("nan"), dtype=t.dtype, device=DEV)
            big[:, h:2 * h] = t
            return big[:, h:2 * h]
        if layout == "head_major":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "odd_rows":
            big = torch.full((n, h, d + 3), float("nan"), dtype=t.dtype, device=DEV)
            big[..., :d] = t
            return big[..., :d]
        return torch.cat([t.new_zeros(3), t.reshape(-1)])[3:].view(n, h, d)
    _attn_check(q, k, v, g, view=view)


@pytest.mark.parametrize("tq,tk", [(150, 150), (1, 40), (40, 1)])
@pytest.mark.parametrize("layout", ["token", "head", "projection"])
def test_attention_dense_batches(tq, tk, layout):
    """[batch, token, head, dim], as views of what projections give, equal to
    the packed form bit for bit."""
    import concord_amd as ca
    b, h, hk, d = 3, 4, 2, 64
    q, k, v, g = _attn_inputs(b * tq, b * tk, h, hk, d)

    def four(t, n):
        t = t.to(DEV).view(b, n, t.shape[1], d)
        if layout == "head":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "projection":
            return torch.cat([t, t], 2)[:, :, t.shape[2]:]
        return t
    packed = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    po = ca.attention(*packed, starts=_i32(list(range(0, b * tq + 1, tq))), k_starts=_i32(list(range(0, b * tk + 1, tk))))
    pg = torch.autograd.grad(po, packed, g.to(DEV))
    dense = [four(t, n).detach().requires_grad_(True) for t, n in ((q, tq), (k, tk), (v, tk))]
    do = ca.attention(*dense)
    dg = torch.autograd.grad(do, dense, four(g, tq))
    for a, c in zip((po, *pg), (do, *dg)):
        assert torch.equal(a, c.reshape(a.shape))
    ref = _attn_ref(*(t.double() for t in (q, k, v, g)), list(range(0, b * tq + 1, tq)),
                    list(range(0, b * tk + 1, tk)), True, 0.125)
    _close(po, ref["out"][0], ref["out"][1] + 1e-30, "out")


def test_attention_empty():
    import concord_amd as ca
    z = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    assert ca.attention(z, z, z).shape == z.shape
    assert ca.attention(z, z, z, starts=_i32([0])).shape == z.shape
    q = torch.randn(5, 2, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    out = ca.attention(q, z, z, starts=_i32([0, 5]), k_starts=_i32([0, 0]))
    out.sum().backward()
    assert float(out.detach().abs().sum()) == 0.0 and float(q.grad.abs().sum()) == 0.0
    k = torch.randn(5, 2, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    out = ca.attention(z, k, k, starts=_i32([0, 0]), k_starts=_i32([0, 5]))
    out.sum().backward()
    assert out.shape == z.shape and float(k.grad.abs().sum()) == 0.0
    z4 = torch.zeros(0, 7, 2, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    ca.attention(z4, z4, z4).sum().backward()


def test_attention_differences():
    """The gradients along random directions against central differences of the
    64-bit forward."""
    import concord_amd as ca
    q, k, v, g = _attn_inputs(70, 70, 2, 1, 64)
    starts = [0, 30, 70]
    p = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(ca.attention(*p, starts=_i32(starts)), p, g.to(DEV))
    base = [t.double() for t in (q, k, v)]

    def loss(args):
        return float((_attn_ref(*args, g.double(), starts, starts, True, 0.125)["out"][0] * g.double()).sum())
    gen = _gen("fd-attn")
    h = 1e-4
    for i in range(3):
        u = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * u, base[i] - h * u
        num = (loss(up) - loss(dn)) / (2 * h)
        terms = grads[i].double().cpu() * u
        # each gradient is off by a few bf16 roundings; they add at random: 2^-7 of the terms' norm, times 4
        assert abs(num - float(terms.sum())) <= 4 * 2.0 ** -7 * float(terms.norm()) + 1e-6, (i, num, float(terms.sum()))


def test_attention_is_reproducible_and_stream_safe():
    import concord_amd as ca
    q, k, v, g = (t.to(DEV) for t in _attn_inputs(2000, 2000, 8, 2, 64))
    starts = _i32([0, 3, 700, 2000])
    p = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        out = ca.attention(*p, starts=starts)
        return (out.detach(), *torch.autograd.grad(out, p, g))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [step() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for o in other + [step()]:
        assert all(torch.equal(a, b) for a, b in zip(first, o))


# ---- distillation ----------------------------------------------------------------
def _distill_ref(z, t, idx, temp, g):
    """loss and gradient in 64 bits with the bounds of a 32-bit evaluation"""
    rows, vocab = z.shape
    loss, el = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    dz, ez = torch.zeros_like(z), torch.zeros_like(z)
    logq = torch.log_softmax(z / temp, 1)
    q = logq.exp()
    # an exponent's argument is off by 2^-23 of its size: so is the exponential, relatively
    span = ((z - z.amax(1, keepdim=True)) / temp).abs().nan_to_num(posinf=0.0)
    eq = q * (EPS32 + 2.0 ** -21 * (1 + span))
    for r in range(rows):
        ok = (idx[r] >= 0) & (idx[r] < vocab) & (t[r] > -math.inf)
        if not ok.any() or g[r] == 0 and not math.isfinite(float(z[r].abs().max())):
            continue
        i, logp = idx[r][ok], torch.log_softmax(t[r][ok] / temp, 0)
        p = logp.exp()
        terms = torch.where(p > 0, p * (logp - logq[r, i]), torch.zeros_like(p))
        loss[r] = temp ** 2 * terms.sum()
        tspan = ((t[r][ok] - t[r][ok].max()) / temp).abs()
        ep = p * (EPS32 + 2.0 ** -21 * (1 + tspan))
        el[r] = temp ** 2 * (EPS32 * (p * (logp.abs() + logq[r, i].abs() + tspan + span[r, i] + 1)).nan_to_num(0.0).sum()
                             + (ep * (logp - logq[r, i]).abs()).nan_to_num(0.0).sum())
        if g[r] == 0:
            continue
        d = q[r].clone()
        e = eq[r].clone()
        d.index_add_(0, i, -p)
        e.index_add_(0, i, ep)
        dz[r] = g[r] * temp * d
        ez[r] = abs(float(g[r])) * temp * e
    return (loss, el + 1e-30), (dz, ez + 1e-37)


def _distill_case(rows, vocab, top, dtype, spread=2.5):
    gen = _gen("distill", rows, vocab, top, str(dtype))
    z = (spread * torch.randn(rows, vocab, generator=gen)).to(dtype)
    idx = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(rows)]) if rows else \
        torch.zeros(0, top, dtype=torch.int64)
    t = (2 * torch.randn(rows, top, generator=gen)).sort(1, descending=True).values
    g = torch.randn(rows, generator=gen)
    return z, t, idx, g


def _distill_check(z, t, idx, g, temp=1.0, to=lambda t: t.to(DEV), index_dtype=torch.int64):
    import concord_amd as ca
    (loss, el), (dz, ez) = _distill_ref(z.double(), t.double(), idx, temp, g.double())
    zd = to(z).requires_grad_(True)
    got = ca.distill_loss(zd, t.to(DEV), idx.to(index_dtype).to(DEV), temperature=temp)
    with torch.no_grad():
        assert torch.equal(ca.distill_loss(zd, t.to(DEV), idx.to(DEV), temperature=temp), got)
    gz, = torch.autograd.grad(got, zd, g.to(DEV))
    assert got.dtype == torch.float32 and gz.dtype == z.dtype
    _close(got, loss, el + 2.0 ** -22 * loss.abs(), "loss")
    u = U[z.dtype]
    _close(gz, dz, ez + u * (dz.abs() + ez) + TINY[z.dtype], "dlogits")
    return gz


@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (130, 65, 16), (9, 1000, 64), (6, 1024, 20), (6, 1025, 20), (4, 4096, 1),
    (5, 5003, 100), (3, 9999, 64), (2, 50257, 50), (1, 160001, 256), (1030, 1500, 8), (2, 3000, 1024), (4, 100, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_distill_sizes(rows, vocab, top, dtype):
    _distill_check(*_distill_case(rows, vocab, top, dtype))


@pytest.mark.parametrize("temp", [0.5, 2.0, 10.0])
@pytest.mark.parametrize("vocab", [65, 5003])
def test_distill_temperatures(temp, vocab):
    _distill_check(*_distill_case(12, vocab, 16, torch.float32), temp=temp, index_dtype=torch.int32)


@pytest.mark.parametrize("vocab", [65, 20001])
def test_distill_masked_entries(vocab):
    """Entries left out, rows without any, one place named twice and more, teacher
    logits of -inf and the type's lowest value."""
    z, t, idx, g = _distill_case(10, vocab, 16, torch.bfloat16)
    idx[0] = -1
    idx[1, 5:] = -1
    idx[2, ::2] = vocab + 3
    idx[3, 1:] = idx[3, 0]
    idx[4, 8:] = idx[4, :8]
    t[5, 3:] = -math.inf
    t[6] = -math.inf
    t[7, 2:] = torch.finfo(torch.float32).min
    idx[8] = torch.iinfo(torch.int64).max
    idx[9, 0] = torch.iinfo(torch.int64).min
    gz = _distill_check(z, t, idx, g)
    for r in (0, 6, 8):
        assert float(gz[r].abs().sum()) == 0.0


@pytest.mark.parametrize("vocab", [65, 20001])
def test_distill_masked_logits(vocab):
    """Student logits of -inf and the lowest value at places the teacher does not
    name, and rows of NaN whose upstream gradient is 0."""
    z, t, idx, g = _distill_case(8, vocab, 8, torch.float32)
    named = torch.zeros(8, vocab, dtype=torch.bool).scatter_(1, idx, True)
    hide = (torch.rand(8, vocab, generator=_gen("hide")) < 0.5) & ~named
    z[:3] = z[:3].masked_fill(hide[:3], -math.inf)
    z[3:6] = z[3:6].masked_fill(hide[3:6], torch.finfo(torch.float32).min)
    gz = _distill_check(z[:6], t[:6], idx[:6], g[:6])
    assert float(gz[:3][hide[:3].to(DEV)].abs().sum()) == 0.0
    import concord_amd as ca
    z[6:] = float("nan")
    zd = z.to(DEV).requires_grad_(True)
    loss = ca.distill_loss(zd, t.to(DEV), idx.to(DEV))
    assert bool(torch.isnan(loss[6:]).all()) and not bool(torch.isnan(loss[:6]).any())
    g[6:] = 0.0
    gz, = torch.autograd.grad(loss, zd, g.to(DEV))
    assert float(gz[6:].abs().sum()) == 0.0 and not bool(torch.isnan(gz).any())


def test_distill_impossible_target_is_infinite():
    import concord_amd as ca
    z, t, idx, g = _distill_case(2, 300, 4, torch.float32)
    z[0, idx[0, 1]] = -math.inf
    loss = ca.distill_loss(z.to(DEV), t.to(DEV), idx.to(DEV))
    assert math.isinf(float(loss[0])) and math.isfinite(float(loss[1]))


@pytest.mark.parametrize("layout", ["cols", "misaligned", "transposed"])
@pytest.mark.parametrize("vocab", [96, 2056])
def test_distill_strides(layout, vocab):
    def to(t):
        t = t.to(DEV)
        n, c = t.shape
        if layout == "cols":
            big = torch.full((n, c + 11), float("nan"), dtype=t.dtype, device=DEV)
            big[:, 3:3 + c] = t
            return big[:, 3:3 + c].detach()
        if layout == "misaligned":
            return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(n, c).detach()
        return t.t().contiguous().t().detach()
    for dtype in (torch.bfloat16, torch.float32):
        _distill_check(*_distill_case(7, vocab, 12, dtype), to=to)


def test_distill_upstream_gradients():
    """A mean's, a sum's and a weighted sum's gradient; rows in two dimensions."""
    import concord_amd as ca
    z, t, idx, g = _distill_case(12, 65, 8, torch.float32)
    for reduce, up in ((torch.mean, torch.full((12,), 1 / 12)), (torch.sum, torch.ones(12))):
        (_, _), (dz, ez) = _distill_ref(z.double(), t.double(), idx, 1.0, up.double())
        zd = z.to(DEV).view(3, 4, 65).requires_grad_(True)
        reduce(ca.distill_loss(zd, t.to(DEV).view(3, 4, 8), idx.to(DEV).view(3, 4, 8))).backward()
        _close(zd.grad.view(12, 65), dz, ez + 2.0 ** -22 * dz.abs() + 1e-37, "dlogits")


def test_distill_differences():
    import concord_amd as ca
    for vocab in (65, 5000):
        z, t, idx, g = _distill_case(6, vocab, 12, torch.float32)
        zd = z.to(DEV).requires_grad_(True)
        dz, = torch.autograd.grad(ca.distill_loss(zd, t.to(DEV), idx.to(DEV), 2.0), zd, g.to(DEV))
        u = torch.randn(z.shape, generator=_gen("fd-distill"))
        h = 2.0 ** -6
        up, dn = (_distill_ref((z.double() + s * u.double()), t.double(), idx, 2.0, g.double())[0][0] for s in (h, -h))
        num, ana = float(((up - dn) * g.double()).sum()) / (2 * h), float((dz.cpu().double() * u.double()).sum())
        # third derivatives times h^2
        assert abs(num - ana) <= 10 * h * h * float((dz.cpu().double() * u.double()).abs().sum()) + 1e-5, (num, ana)


def test_distill_empty():
    import concord_amd as ca
    z = torch.zeros(0, 65, device=DEV, requires_grad=True)
    loss = ca.distill_loss(z, torch.zeros(0, 4, device=DEV), torch.zeros(0, 4, dtype=torch.int64, device=DEV))
    loss.sum().backward()
    assert loss.shape == (0,) and z.grad.shape == z.shape


# ---- all three ------------------------------------------------------------------
def _all_three(tokens, gen):
    """A training step through layer norm, attention and the loss: (inputs, step)."""
    import concord_amd as ca
    x = torch.randn(tokens, 384, generator=gen).to(torch.bfloat16).to(DEV).requires_grad_(True)
    w, b = ((torch.randn(384, generator=gen) * 0.1 + c).to(DEV).requires_grad_(True) for c in (1.0, 0.0))
    starts = _i32([0, 1, tokens // 3, tokens])
    t = torch.randn(tokens, 8, generator=gen).to(DEV)
    i = torch.randint(0, 128, (tokens, 8), generator=gen).to(DEV)

    def step():
        q, k, v = ca.layer_norm(x, w, b).view(tokens, 6, 64).split([4, 1, 1], dim=1)
        z = ca.attention(q, k, v, starts=starts).reshape(tokens, 256)[:, :128]
        loss = ca.distill_loss(z, t, i, temperature=2.0).mean()
        return (loss, *torch.autograd.grad(loss, (x, w, b)))
    return x, step


def test_operators_in_a_captured_step():
    """One HIP graph of the step, replayed with new inputs and with eager work
    between the replays: the eager results, bit for bit."""
    gen = _gen("graph")
    x, step = _all_three(700, gen)
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
            x.copy_(torch.randn(x.shape, generator=gen).to(x.dtype))
        graph.replay()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_are_differentiable_once():
    import concord_amd as ca
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    q = torch.randn(4, 1, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    idx = torch.zeros(4, 1, dtype=torch.int64, device=DEV)
    for y, leaf in ((ca.layer_norm(x), x), (ca.attention(q, q, q), q),
                    (ca.distill_loss(x, torch.zeros(4, 1, device=DEV), idx), x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


def test_operators_see_a_change_of_a_saved_tensor():
    """An input overwritten between forward and backward is an error, not a wrong gradient."""
    import concord_amd as ca
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    h = x * 1.0
    y = ca.layer_norm(h)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
