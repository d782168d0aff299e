"""Operators of a language model's training step around the packed layers, as
measured cases: layer norm, attention over packed sequences and distillation
from a teacher's top logits.

A case is one pass on one GPU: the operator alone (evaluation, a teacher's
pass), or the operator and its gradients through autograd, as a training step
takes them.  Where `own` is false the same values come from elementary torch
operations in 32 bits, rounded once at the end.

Sizes are those of the char-level GPT and the SDXL UNet that this repository
trains, and generic ones up to a language model's: tens of thousands of
tokens, grouped heads of 128, a vocabulary of tens of thousands.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------
def _norm(name, rows, width, dtype="bf16", train=True):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "train": train}


def _dense(name, batch, tq, heads, dim, tk=None, kv_heads=None, causal=True, train=True):
    """[batch, token, head, dim] tensors, all sequences of one length."""
    return {"name": name, "op": "attn", "dense": True, "batch": batch, "tq": tq, "tk": tk or tq, "heads": heads,
            "kv_heads": kv_heads or heads, "dim": dim, "causal": causal, "train": train}


def _ragged(name, lens, heads, kv_heads, dim, causal=True, train=True):
    """[token, head, dim] tensors that hold sequences of the lengths `lens` one after another."""
    return {"name": name, "op": "attn", "dense": False, "lens": " ".join(str(n) for n in lens), "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "causal": causal, "train": train}


def _distill(name, rows, vocab, top, dtype="bf16", temperature=1.0, train=True):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype,
            "temperature": temperature, "train": train}


def listed():
    return [
        # the smallest call: the norm of one generated token, latency only
        _norm("norm_one_token", 1, 1280, train=False),
        # char GPT: 64 sequences of 256 tokens, width 384
        _norm("norm_char", 16384, 384),
        # a width that no vector load divides, in half precision
        _norm("norm_odd_width", 4099, 2051, dtype="f16"),
        # a language model's micro-batch, bound by memory
        _norm("norm_wide", 32768, 4096),
        # char GPT's attention: many short sequences
        _dense("attn_char", 64, 256, 6, 64),
        # SDXL self-attention at the 64 x 64 level, no mask
        _dense("attn_image", 2, 4096, 10, 64, causal=False),
        # SDXL cross-attention on 77 text tokens, forward alone
        _dense("attn_cross", 4, 1024, 20, 64, tk=77, causal=False, train=False),
        # documents of very different lengths packed into one row of 16384 tokens
        _ragged("attn_packed", [1, 4099, 17, 640, 2, 2048, 333, 5000, 129, 64, 1111, 63, 1500, 7, 1370], 32, 8, 128),
        # one long prompt, forward alone
        _ragged("attn_long", [32768], 32, 8, 128, train=False),
        # char GPT distilled: a vocabulary of 65, fp32 logits
        _distill("distill_char", 16384, 65, 16, dtype="fp32", temperature=2.0),
        # few rows of a long vocabulary, forward alone (evaluation of one short text)
        _distill("distill_few_rows", 32, 32000, 64, train=False),
        # a vocabulary whose rows begin at every alignment
        _distill("distill_wide", 8192, 50257, 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "attn", "attn", "distill"])
    train = rng.random() < 0.7
    if op == "norm":
        while True:
            rows, width = _log_int(rng, 1, 65536), _log_int(rng, 32, 12288)
            if rng.random() < 0.7:
                width = max(32, width // 32 * 32)
            if rows * width <= 32768 * 4096:
                break
        c = _norm("", rows, width, dtype=rng.choice(["bf16", "bf16", "f16", "fp32"]), train=train)
        if c["dtype"] == "fp32" and rows * width > 16384 * 4096:
            c["dtype"] = "bf16"
    elif op == "distill":
        while True:
            rows, vocab = _log_int(rng, 1, 32768), _log_int(rng, 65, 160000)
            if rows * vocab <= 8192 * 50257:
                break
        c = _distill("", rows, vocab, min(vocab, rng.choice([1, 8, 20, 50, 64, 100, 256])),
                     dtype=rng.choice(["bf16", "bf16", "fp32"]), temperature=rng.choice([1.0, 2.0, 4.0]),
                     train=train)
        if c["dtype"] == "fp32" and rows * vocab > 4096 * 50257:
            c["dtype"] = "bf16"
    else:
        dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 5, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        if rng.random() < 0.5:
            while True:
                batch, tq = _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
                tk = tq if rng.random() < 0.7 else _log_int(rng, 1, 8192)
                if batch * max(tq, tk) <= 32768:
                    break
            c = _dense("", batch, tq, heads, dim, tk=tk, kv_heads=kv_heads, causal=tk >= tq and rng.random() < 0.7,
                       train=train)
        else:
            lens, left = [], _log_int(rng, 16, 32768)
            while left > 0 and len(lens) < 64:
                n = min(left, _log_int(rng, 1, 16384))
                lens.append(n)
                left -= n
            c = _ragged("", lens, heads, kv_heads, dim, causal=rng.random() < 0.8, train=train)
        while work(c)["flops"] > 8e12:   # the listed long prompt has 8.8e12
            c["heads"], c["kv_heads"] = c["heads"] // c["kv_heads"], 1
            if work(c)["flops"] > 8e12:
                c["train"] = False
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------
def _lens(case):
    if case["dense"]:
        return [case["tq"]] * case["batch"], [case["tk"]] * case["batch"]
    lens = [int(n) for n in case["lens"].split()]
    return lens, lens


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    s = dict(case)
    train = case["train"]
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        dt = DTYPES[case["dtype"]]
        # a residual stream: an offset, and a few channels far larger than the rest
        gain = torch.where(torch.rand(width, generator=gen, device=DEV) < 0.01, 20.0, 1.0)
        s["x"] = (randn(rows, width) * gain + 0.3).to(dt).requires_grad_(train)
        s["weight"] = (1.0 + 0.2 * randn(width)).requires_grad_(train)
        s["bias"] = (0.1 * randn(width)).requires_grad_(train)
        if train:
            s["dy"] = (1e-2 * randn(rows, width)).to(dt)
    elif case["op"] == "attn":
        lq, lk = _lens(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        tq, tk = sum(lq), sum(lk)
        if tq == tk:
            # one projection's output, split: rows of q, k and v side by side
            qkv = randn(tq, h + 2 * hk, d).to(torch.bfloat16)
            q, k, v = qkv.split([h, hk, hk], dim=1)
        else:
            q = randn(tq, h, d).to(torch.bfloat16)
            k, v = randn(tk, 2 * hk, d).to(torch.bfloat16).split([hk, hk], dim=1)
        if case["dense"]:
            q, k, v = (t.unflatten(0, (case["batch"], -1)) for t in (q, k, v))
        else:
            s["starts"] = torch.tensor(_starts(lq), dtype=torch.int32, device=DEV)
        s["q"], s["k"], s["v"] = (t.detach().requires_grad_(train) for t in (q, k, v))
        if train:
            s["dout"] = (1e-2 * randn(tq, h, d)).to(torch.bfloat16).view(q.shape)
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        s["logits"] = (2.5 * randn(rows, vocab)).to(DTYPES[case["dtype"]]).requires_grad_(train)
        # the teacher's largest logits, in order, each at a place of its own
        first = torch.randint(0, vocab, (rows, 1), generator=gen, device=DEV)
        stride = torch.randint(1, vocab // top + 1, (rows, 1), generator=gen, device=DEV)
        s["index"] = (first + stride * torch.arange(top, device=DEV)) % vocab
        s["teacher"] = (8.0 + 2.0 * randn(rows, top)).sort(dim=1, descending=True).values
        if train:
            s["dloss"] = torch.full((rows,), 1.0 / rows, device=DEV)
    return s


# ---- the passes -------------------------------------------------------------
def run(s):
    one = {"norm": _run_norm, "attn": _run_attn, "distill": _run_distill}[s["op"]]
    if not s["train"]:
        with torch.no_grad():
            return one(s)
    return one(s)


def _run_norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    if own:
        import concord_amd as ca
        y = ca.layer_norm(x, w, b, EPS)
        if not s["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    with torch.no_grad():
        xf = x.float()
        c = xf - xf.mean(1, keepdim=True)
        rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
        xhat = c * rstd
        y = (xhat * w + b).to(x.dtype)
        if not s["train"]:
            return {"y": y}
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return {"y": y, "dx": dx.to(x.dtype), "dw": (dy * xhat).sum(0), "db": dy.sum(0)}


def _run_attn(s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        import concord_amd as ca
        out = ca.attention(q, k, v, starts=s.get("starts"), causal=s["causal"])
        if not s["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        return _plain_attn(s)


def _blocks(s):
    """(q rows, k rows, batch of equal sequences, first query of each, count of queries) in
    pieces whose scores take at most 1 GB."""
    lq, lk = _lens(s)
    sq, sk = _starts(lq), _starts(lk)
    if s["dense"]:
        tq, tk = s["tq"], s["tk"]
        per = max(1, int(2.5e8 // (s["heads"] * tq * tk)))
        if per > 1 or s["batch"] == 1 and s["heads"] * tq * tk <= 2.5e8:
            for b in range(0, s["batch"], per):
                n = min(per, s["batch"] - b)
                yield slice(b * tq, (b + n) * tq), slice(b * tk, (b + n) * tk), n, 0, tq, tq, tk
            return
    for b in range(len(lq)):
        if lq[b] == 0:
            continue
        step = max(1, int(2.5e8 // (s["heads"] * max(lk[b], 1))))
        for i in range(0, lq[b], step):
            n = min(step, lq[b] - i)
            # under the causal mask the piece's last query ends the keys
            end = min(lk[b], max(0, i + n + lk[b] - lq[b])) if s["causal"] else lk[b]
            yield slice(sq[b] + i, sq[b] + i + n), slice(sk[b], sk[b] + end), 1, i, n, lq[b], lk[b]


def _plain_attn(s):
    shape_q, shape_k = s["q"].shape, s["k"].shape
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    scale = 1.0 / math.sqrt(d)
    # [head, token, dim], shared heads repeated
    q, k, v = (t.detach().reshape(-1, n, d).float().transpose(0, 1)
               for t, n in ((s["q"], h), (s["k"], hk), (s["v"], hk)))
    rep = h // hk
    out = torch.zeros(h, q.shape[1], d, device=DEV)
    if s["train"]:
        dout = s["dout"].reshape(-1, h, d).float().transpose(0, 1)
        dq = torch.zeros_like(out)
        dk, dv = torch.zeros(hk, k.shape[1], d, device=DEV), torch.zeros(hk, k.shape[1], d, device=DEV)
    for qs, ks, n, first, rows, len_q, len_k in _blocks(s):
        if ks.stop == ks.start:
            continue

        def piece(t, sl, heads):
            return t[:, sl].reshape(heads, n, -1, d).contiguous()
        qb = piece(q, qs, h)
        kb, vb = (piece(t, ks, hk).repeat_interleave(rep, 0) for t in (k, v))
        p = torch.matmul(qb, kb.transpose(2, 3).contiguous()) * scale
        if s["causal"]:
            i = torch.arange(first, first + rows, device=DEV)[:, None] + (len_k - len_q)
            p.masked_fill_(torch.arange(kb.shape[2], device=DEV)[None, :] > i, float("-inf"))
        p -= p.amax(-1, keepdim=True).clamp_min(-1e30)
        p.exp_()
        p /= p.sum(-1, keepdim=True).clamp_min(1e-30)
        out[:, qs] = torch.matmul(p, vb).reshape(h, -1, d)
        if s["train"]:
            gb = piece(dout, qs, h)

            def shared(t, x):   # t^T x, summed over the query heads that share a key head
                return torch.matmul(t.transpose(2, 3).contiguous(), x).view(hk, rep, -1, d).sum(1)
            dv[:, ks] += shared(p, gb)
            ds = torch.matmul(gb, vb.transpose(2, 3).contiguous())
            ds -= (p * ds).sum(-1, keepdim=True)
            ds *= p
            ds *= scale
            del p
            dq[:, qs] = torch.matmul(ds, kb).reshape(h, -1, d)
            dk[:, ks] += shared(ds, qb)

    def back(t, shape):
        return t.transpose(0, 1).to(torch.bfloat16).reshape(shape)
    if not s["train"]:
        return {"out": back(out, shape_q)}
    return {"out": back(out, shape_q), "dq": back(dq, shape_q), "dk": back(dk, shape_k), "dv": back(dv, shape_k)}


def _run_distill(s):
    z, t, idx, temp = s["logits"], s["teacher"], s["index"], s["temperature"]
    if own:
        import concord_amd as ca
        loss = ca.distill_loss(z, t, idx, temperature=temp)
        if not s["train"]:
            return {"loss": loss}
        dz, = torch.autograd.grad(loss, (z,), s["dloss"])
        return {"loss": loss.detach(), "dlogits": dz}
    with torch.no_grad():
        zf = z.float() / temp
        zf -= zf.amax(1, keepdim=True)
        tf = t.float() / temp
        tf = tf - tf.amax(1, keepdim=True)
        p = tf.exp()
        psum = p.sum(1, keepdim=True)
        p = p / psum
        picked = torch.gather(zf, 1, idx)
        q = zf.exp()
        qsum = q.sum(1, keepdim=True)
        loss = (p * (tf - psum.log() - picked + qsum.log())).sum(1) * (temp * temp)
        if not s["train"]:
            return {"loss": loss}
        q /= qsum
        q.scatter_add_(1, idx, -p)
        return {"loss": loss, "dlogits": (q * (s["dloss"][:, None] * temp)).to(z.dtype)}


# ---- work -------------------------------------------------------------------
def _pairs(case):
    """Query-key pairs that the mask leaves, for one head."""
    total = 0
    for a, b in zip(*_lens(case)):
        if not case["causal"]:
            total += a * b
            continue
        # query i sees keys 0 .. i + b - a
        lo = max(0, a - b)
        n = a - lo
        total += n * (lo + 1 + b - a) + n * (n - 1) // 2
    return total


def work(case):
    train = case["train"]
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        es = 4 if case["dtype"] == "fp32" else 2
        # x and y; for training dy and dx too; the weight, the bias and their gradients
        return {"bytes": n * es * (4 if train else 2) + case["width"] * 4.0 * (4 if train else 2),
                "flops": n * (16.0 if train else 7.0)}
    if case["op"] == "attn":
        lq, lk = _lens(case)
        q, kv = sum(lq) * case["heads"] * case["dim"] * 2.0, sum(lk) * case["kv_heads"] * case["dim"] * 2.0
        # two products forward; five backward, the scores formed again (to keep
        # them would take memory that grows with the square of the length)
        return {"bytes": (4 * q + 4 * kv) if train else (2 * q + 2 * kv),
                "flops": (14.0 if train else 4.0) * _pairs(case) * case["heads"] * case["dim"]}
    n = case["rows"] * case["vocab"]
    es = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": n * es * (2.0 if train else 1.0) + case["rows"] * (case["top"] * 12.0 + (8 if train else 4)),
            "flops": n * (8.0 if train else 4.0)}


# ---- the definitions in 64 bits ---------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "attn": _exact_attn, "distill": _exact_distill}[case["op"]](s)


def _exact_norm(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    var, mean = torch.var_mean(x, 1, unbiased=False)
    sd = torch.sqrt(var + EPS)[:, None]
    xhat = (x - mean[:, None]) / sd
    out = {"y": w * xhat + b}
    if s["train"]:
        dy = s["dy"].double()
        dxhat = dy * w
        n = x.shape[1]
        # the projection off the constant vector and off xhat, over the deviation
        along = (dxhat * xhat).sum(1, keepdim=True) / n
        out.update(dx=(dxhat - dxhat.sum(1, keepdim=True) / n - along * xhat) / sd, dw=(dy * xhat).sum(0),
                   db=dy.sum(0))
    return out


def _exact_attn(s):
    lq, lk = _lens(s)
    sq, sk = _starts(lq), _starts(lk)
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    if _pairs(s) * h * d > 3e12:
        return None
    q, g = s["q"].reshape(-1, h, d), s["dout"].reshape(-1, h, d) if s["train"] else None
    k, v = s["k"].reshape(-1, hk, d), s["v"].reshape(-1, hk, d)
    names = ("out", "dq", "dk", "dv") if s["train"] else ("out",)
    res = {n: torch.zeros(t.shape, dtype=torch.float64, device=DEV)
           for n, t in zip(names, (q, q, k, v))}
    for b in range(len(lq)):
        rows_k = slice(sk[b], sk[b + 1])
        if lq[b] == 0 or lk[b] == 0:
            continue
        for head in range(h):
            kh, vh = k[rows_k, head // (h // hk)].double(), v[rows_k, head // (h // hk)].double()
            step = max(1, int(3e7 // lk[b]))
            for i in range(sq[b], sq[b + 1], step):
                rows = slice(i, min(i + step, sq[b + 1]))
                qh = q[rows, head].double()
                z = qh @ kh.T / math.sqrt(d)
                if s["causal"]:
                    at = torch.arange(rows.start - sq[b], rows.stop - sq[b], device=DEV)
                    hidden = torch.arange(lk[b], device=DEV) - (lk[b] - lq[b]) > at[:, None]
                    z = z.masked_fill(hidden, -math.inf)
                p = torch.nan_to_num(torch.softmax(z, 1))
                o = p @ vh
                res["out"][rows, head] = o
                if s["train"]:
                    gh = g[rows, head].double()
                    dz = p * (gh @ vh.T - (gh * o).sum(1, keepdim=True)) / math.sqrt(d)
                    res["dq"][rows, head] = dz @ kh
                    res["dk"][rows_k, head // (h // hk)] += dz.T @ qh
                    res["dv"][rows_k, head // (h // hk)] += p.T @ gh
    shapes = (s["q"].shape, s["q"].shape, s["k"].shape, s["v"].shape)
    return {n: res[n].reshape(shape) for n, shape in zip(names, shapes)}


def _exact_distill(s):
    temp = s["temperature"]
    z, t = s["logits"].double() / temp, s["teacher"].double() / temp
    logq = z - torch.logsumexp(z, 1, keepdim=True)
    logp = t - torch.logsumexp(t, 1, keepdim=True)
    p = logp.exp()
    out = {"loss": temp ** 2 * (p * (logp - logq.gather(1, s["index"]))).sum(1)}
    if s["train"]:
        d = logq.exp().scatter_add(1, s["index"], -p)
        out["dlogits"] = d * (temp * s["dloss"].double()[:, None])
    return out
