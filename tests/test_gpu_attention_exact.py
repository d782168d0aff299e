"""Attention where rounding the probabilities costs nothing, so that the rest of
the kernels shows: the running maximum's rescaling, the join of key shares, and
the byte that keeps what rounding `out` left over.

Scores are whole numbers of powers of two: q and k meet in dimension 0 alone,
with small whole numbers, and scale = ln 2.  A probability under any running
maximum is then a power of two to within a few 2^-24 times the exponents, and
rounds to it in bfloat16.

Bounds are elementwise and worst-case: a sum of n terms in 32 bits, chained in any
order, truncated rather than rounded, is off by n 2^-23 of its terms' magnitudes;
16 more stand for the roundings around it."""
import ctypes
import math

import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu

U = 2.0 ** -8            # half a unit of bfloat16's last place, relatively
LOW = 2.0 ** -15         # one unit of 16 significant bits (the byte is cut, not rounded)
BF = torch.bfloat16


def eps(n):
    return (n + 16) * 2.0 ** -23


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def reference(q, k, v, g, causal, scale, exact, exact_sums=False, batch=1):
    """{name: (64-bit value, bound)} of [token, head, dim] tensors, `batch` equal
    sequences.  exact: scores without rounding, and probabilities that bfloat16
    holds in the forward.  exact_sums: so are the forward's sums over the keys."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    tq, tk = len(q) // batch, len(k) // batch
    rep, up = h // hk, 0.0 if exact else U
    ekeys = eps(0) if exact_sums else eps(tk)
    res = {n: [torch.zeros(t.shape, dtype=torch.float64) for _ in range(2)]
           for n, t in (("out", q), ("out32", q), ("dq", q), ("dk", k), ("dv", v))}
    lse = torch.full((h, len(q)), math.inf, dtype=torch.float64)
    for b in range(batch):
        rq, rk = slice(b * tq, (b + 1) * tq), slice(b * tk, (b + 1) * tk)
        for a in range(h):
            qa, ga, ka, va = q[rq, a], g[rq, a], k[rk, a // rep], v[rk, a // rep]
            s = qa @ ka.T * scale
            hidden = torch.zeros(tq, tk, dtype=torch.bool)
            if causal:
                hidden = torch.arange(tk) > torch.arange(tq)[:, None] + (tk - tq)
            s = s.masked_fill(hidden, -math.inf)
            top = s.masked_fill(hidden, 0.0).abs().amax(1, keepdim=True)
            p = torch.nan_to_num(torch.softmax(s, 1))
            # scores' sums over d terms; the scale, the maximum and lse in 24 bits: relatively in p
            es = eps(0 if exact else d) * (1 + (qa.abs() @ ka.abs().T) * scale) + 2.0 ** -21 * (1 + top)
            ep = p * (es + (p * es).sum(1, keepdim=True) + ekeys)
            lse[a, rq] = torch.logsumexp(s, 1) / math.log(2)
            lse[a, rq] = torch.where(hidden.all(1), math.inf, lse[a, rq])
            o = p @ va
            eo = (up * p + ep) @ va.abs() + ekeys * (p @ va.abs())
            res["out32"][0][rq, a], res["out32"][1][rq, a] = o, eo
            res["out"][0][rq, a], res["out"][1][rq, a] = o, eo + U * (o.abs() + eo)
            dp, delta = ga @ va.T, (ga * o).sum(1, keepdim=True)
            ed = (ga.abs() * (eo + LOW * (o.abs() + eo) + eps(d) * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            eds = ep * (dp - delta).abs() + (p + ep) * (ed + eps(d) * (ga.abs() @ va.abs().T))
            eds = eds + U * (ds.abs() + eds)
            res["dq"][0][rq, a] = ds @ ka * scale
            res["dq"][1][rq, a] = (eds + eps(tk) * ds.abs()) @ ka.abs() * scale
            res["dk"][0][rk, a // rep] += ds.T @ qa * scale
            res["dk"][1][rk, a // rep] += (eds + eps(tq * rep) * ds.abs()).T @ qa.abs() * scale
            res["dv"][0][rk, a // rep] += p.T @ ga
            res["dv"][1][rk, a // rep] += (U * p + ep + eps(tq * rep) * p).T @ ga.abs()
    for n in ("dq", "dk", "dv"):
        res[n][1] = res[n][1] + U * (res[n][0].abs() + res[n][1])
    return res, lse


def _close(got, want, bound, what):
    got = got.detach().double().cpu().reshape(want.shape)
    bad = ~((got - want).abs() <= bound + 1e-30)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()),
                           float(((got - want).abs() / (bound + 1e-30)).max()), bad.nonzero()[:4].tolist())


def check(q, k, v, g, causal, scale, exact, exact_sums=False, batch=1):
    import concord_amd as ca
    ref, _ = reference(q, k, v, g, causal, scale, exact, exact_sums, batch)

    def four(t):
        t = t.to(DEV)
        return (t.unflatten(0, (batch, -1)) if batch > 1 else t).detach()
    p = [four(t).requires_grad_(True) for t in (q, k, v)]
    out = ca.attention(*p, causal=causal, scale=scale)
    with torch.no_grad():
        assert torch.equal(ca.attention(*p, causal=causal, scale=scale), out)
    grads = torch.autograd.grad(out, p, four(g))
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        _close(got, *ref[name], name)


def stepped(tq, tk, h, hk, d, step, factors, down=False):
    """Keys of tile t (64 keys) score step (t - 1), one of them step t, all times the
    query's factor: the maximum grows by step x factor at every tile, and the tile
    before still counts 64 x 2^-step of the next one's."""
    tile = torch.arange(tk) // 64
    score = step * (tile - 1) + step * (torch.arange(tk) % 64 == (7 * tile + 5) % 64)
    if down:
        score = score.flip(0)
    k = torch.zeros(tk, hk, d)
    k[:, :, 0] = score[:, None].float()
    k[:, :, d // 2:] = _rand(tk, hk, d - d // 2, seed=1)
    q = torch.zeros(tq, h, d)
    q[:, :, 0] = torch.tensor(factors, dtype=torch.float32)[(torch.arange(tq)[:, None] + torch.arange(h)) % len(factors)]
    q[:, :, 1:d // 2] = _rand(tq, h, d // 2 - 1, seed=2)
    assert torch.equal(k.to(BF)[:, :, 0].float(), k[:, :, 0])   # (whole numbers that bfloat16 holds)
    return q.to(BF), k.to(BF), _rand(tk, hk, d, seed=3).to(BF), _rand(tq, h, d, seed=4).to(BF)


def growth(q, k, causal, scale, first):
    """powers of two by which each query's maximum grows past its first `first` keys"""
    s = torch.einsum("qhd,khd->hqk", q.double(), k.double().repeat_interleave(q.shape[1] // k.shape[1], 1)) * scale / math.log(2)
    if causal:
        s = s.masked_fill(torch.arange(len(k)) > torch.arange(len(q))[:, None] + (len(k) - len(q)), -math.inf)
    return torch.nan_to_num(s[..., first:].amax(-1) - s[..., :first].amax(-1))   # (no key at all: nan)


def shares(tq, tk, h, hk, d, causal):
    """key shares of the forward (its workspace is theirs)"""
    from concord_amd import _lib as C
    a = C.AttnArgs()
    a.B, a.TQ, a.TK, a.H, a.HK, a.D, a.causal = 1, tq, tk, h, hk, d, causal
    return C.lib().concord_attention_fwd_workspace_bytes(ctypes.byref(a)) // (tq * h * (d + 2) * 4)


# two to five tiles, whole and cut: both halves of the unrolled loop and each of
# its tails raise the maximum; steps on either side of the 2^8 that it follows
@pytest.mark.parametrize("d", [64, 72, 96, 128])
@pytest.mark.parametrize("tk", [128, 192, 257, 320])
@pytest.mark.parametrize("step", [7, 9, 24])
@pytest.mark.parametrize("causal", [True, False])
def test_maximum_that_grows(d, tk, step, causal):
    q, k, v, g = stepped(130, tk, 2, 1, d, step, [1, 0, 2, -1, 1])
    assert float(growth(q, k, causal, math.log(2), 64).max()) > 8
    check(q, k, v, g, causal, math.log(2), exact=True)
    check(*stepped(130, tk, 2, 1, d, step, [1, 0, 2, -1, 1], down=True), causal, math.log(2), exact=True)


@pytest.mark.parametrize("tq,tk,h,hk,d", [(1, 4097, 4, 1, 64), (1, 4097, 8, 2, 128), (40, 3000, 2, 2, 96), (130, 2500, 2, 1, 128)])
@pytest.mark.parametrize("down", [False, True])
def test_shares_of_different_maxima(tq, tk, h, hk, d, down):
    """Key shares whose maxima lie hundreds of powers of two apart, joined; within a
    share the maximum grows at every tile."""
    n = shares(tq, tk, h, hk, d, True)
    q, k, v, g = stepped(tq, tk, h, hk, d, 16, [1] if tq == 1 else [1, 0, 2, -1], down)
    # (a query of factor 1: its score is k's dimension 0)
    tops = torch.stack([part.max() for part in k[:, 0, 0].float().chunk(n)])
    assert n > 1 and float(tops.max() - tops.min()) > 100
    for causal in (True, False):
        check(q, k, v, g, causal, math.log(2), exact=True)


@pytest.mark.parametrize("tq,tk,h,hk,d", [(1, 3000, 4, 2, 64), (33, 1700, 2, 1, 128), (5, 2049, 2, 2, 96)])
@pytest.mark.parametrize("causal", [True, False])
def test_shares_of_dense_batches(tq, tk, h, hk, d, causal):
    """[batch, token, head, dim] with few queries of many keys."""
    b = 3
    q, k, v, g = (_rand(b * n, m, d, seed=s).to(BF) for n, m, s in ((tq, h, 1), (tk, hk, 2), (tk, hk, 3), (tq, h, 4)))
    check(q, k, v, g, causal, 1 / math.sqrt(d), exact=False, batch=b)


# ---- the byte that the rounding of out leaves over ---------------------------------
def forward_parts(q, k, v, causal, scale):
    """out, out_low and lse of the C entry, and its share count"""
    from concord_amd import _lib as C
    q, k, v = (t.to(DEV).contiguous() for t in (q, k, v))
    (tq, h, d), (tk, hk, _) = q.shape, k.shape
    out, low = torch.empty_like(q), torch.full(q.shape, 99, dtype=torch.int8, device=DEV)
    lse = torch.full((h, tq), float("nan"), device=DEV)
    a = C.AttnArgs()
    for n, t in (("q", q), ("k", k), ("v", v), ("out", out), ("lse", lse), ("out_low", low)):
        setattr(a, n, t.data_ptr())
    for n, heads in (("q", h), ("k", hk), ("v", hk), ("o", h)):
        setattr(a, n + "_t", heads * d)
        setattr(a, n + "_h", d)
    a.B, a.TQ, a.TK, a.H, a.HK, a.D, a.causal, a.scale = 1, tq, tk, h, hk, d, causal, scale
    need = C.lib().concord_attention_fwd_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV) if need else None
    rc = C.lib().concord_attention_fwd(ctypes.byref(a), ws.data_ptr() if need else None, need,
                                       torch.cuda.current_stream().cuda_stream)
    assert rc == C.OK
    torch.cuda.synchronize()
    return out.cpu(), low.cpu(), lse.cpu(), need


def joined(out, low):
    """out and its byte as one number: the byte counts 2^-8 of out's last place"""
    bits = (out.view(torch.int16).int() << 16) + low.int() * 256
    return bits.view(torch.float32)


def small_whole(tq, tk, h, hk, d, seed):
    """Probabilities of 1 to 2^-3 before the division, values of 8 bits: every sum over
    up to 2^13 keys is exact in 24 bits."""
    gen = torch.Generator().manual_seed(seed)
    q, k, _, g = stepped(tq, tk, h, hk, d, 0, [1, 0, 1])
    k[:, :, 0] = -torch.randint(0, 4, (tk, hk), generator=gen).to(BF)
    return q, k, (128 + torch.randint(0, 128, (tk, hk, d), generator=gen)) / 128, g, gen


@pytest.mark.parametrize("tq,tk,h,hk,d,causal", [
    (33, 40, 2, 1, 64, True), (130, 130, 4, 2, 128, True), (150, 90, 2, 2, 40, True), (70, 300, 2, 1, 96, False),
    (1, 4097, 8, 2, 128, False), (40, 3000, 2, 2, 96, True), (130, 2500, 2, 1, 64, True)])
def test_out_has_16_significant_bits(tq, tk, h, hk, d, causal):
    q, k, v, g, gen = small_whole(tq, tk, h, hk, d, tq + tk)
    # both signs, and every dimension of a size of its own
    v = v * (1 - 2 * torch.randint(0, 2, v.shape, generator=gen)) * 2.0 ** torch.randint(-12, 12, (1, hk, d), generator=gen)
    v = v.to(BF)
    out, low, lse, need = forward_parts(q, k, v, causal, math.log(2))
    assert (need > 0) == (tk > 2000)
    ref, want_lse = reference(q, k, v, g, causal, math.log(2), exact=True, exact_sums=True)
    want, e = ref["out32"]
    _close(joined(out, low), want, e + LOW * (want.abs() + e), "out with its byte")
    # (the byte is needed: out alone is off by more at most places with a sum behind them)
    some = want.abs() > 0
    missed = (out.double() - want).abs() > e + LOW * (want.abs() + e)
    assert float(missed[some].double().mean()) > 0.5, float(missed[some].double().mean())
    # rows without a key: 0 in both, and lse = inf
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), none)
    rows = none.T[:, :, None].expand(out.shape)
    assert not out[rows].any() and not low[rows].any()
    have = ~none
    _close(lse[have], want_lse[have], 2.0 ** -20 * (1 + want_lse[have].abs()), "lse")


@pytest.mark.parametrize("tq,tk,h,hk,d,causal", [(60, 60, 2, 1, 64, True), (90, 40, 2, 2, 128, False), (20, 2200, 2, 1, 64, True)])
def test_gradients_where_delta_dominates(tq, tk, h, hk, d, causal):
    """Values of 1 and 1 + 2^-7: dP - delta is a small difference of large numbers, and
    half a unit in out's last place is as large as it.  The bound counts out in 16
    bits; with out in 8 (planted in the oracle here) most rows of dq miss it."""
    q, k, v, g, gen = small_whole(tq, tk, h, hk, d, tk)
    k[:, :, d // 2:] = (1 + k[:, :, d // 2:].float().abs()).to(BF)
    v = (1 + 2.0 ** -7 * torch.randint(0, 2, v.shape, generator=gen)).to(BF)
    scale = math.log(2)
    # the planted mistake: delta from the rounded out
    ref, _ = reference(q, k, v, g, causal, scale, exact=True, exact_sums=True)
    want, e = ref["dq"]
    out8 = ref["out"][0].to(BF).double()
    shift = (g.double() * (ref["out"][0] - out8)).sum(2)                       # error of delta
    rep = h // hk
    mean_k = torch.zeros_like(want)
    for a in range(h):
        s = q.double()[:, a] @ k.double()[:, a // rep].T * scale
        if causal:
            s = s.masked_fill(torch.arange(tk) > torch.arange(tq)[:, None] + (tk - tq), -math.inf)
        mean_k[:, a] = torch.nan_to_num(torch.softmax(s, 1)) @ k.double()[:, a // rep]
    missed = ((shift[:, :, None] * mean_k * scale).abs() > e)[:, :, d // 2:]
    assert float(missed.any(2).double().mean()) > 0.5, float(missed.any(2).double().mean())
    check(q, k, v, g, causal, scale, exact=True, exact_sums=True)
