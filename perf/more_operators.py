"""Operators of a training step from tokens to the feed-forward, as measured
cases: embedding with its gradient by sorted tokens, norms of queries and keys
with the position rotation, activations that keep their input in 8 bits for the
backward, and the 8-bit form itself.

A case is one pass on one GPU: the operator alone (evaluation, decoding), or the
operator and its gradients through autograd, as a training step takes them.
Where `own` is false the same values come from elementary torch operations in 32
bits (64 for angles and for sums over tokens), rounded once at the end.

Sizes are those of the char-level GPT and the SDXL UNet that this repository
trains, and generic ones up to a language model's: tens of thousands of tokens,
grouped heads of 128, a vocabulary of tens of thousands.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
BLOCK = 32   # values that share an exponent in the 8-bit form
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------
def _embed(name, tokens, vocab, width, table="fp32", dtype="fp32", scale=1.0, pad=0.0, train=True):
    """`pad`: the share of tokens that stand for nothing (-1)."""
    return {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "width": width, "table": table,
            "dtype": dtype, "scale": scale, "pad": pad, "train": train}


def _qk(name, batch, tokens, heads, kv_heads, dim, rotary=None, interleaved=False, base=10000.0, far=0, dtype="bf16",
        train=True):
    """`far`: the largest position (0: each sequence counts its own tokens)."""
    return {"name": name, "op": "qk", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary or dim, "interleaved": interleaved, "base": base, "far": far, "dtype": dtype,
            "train": train}


def _act(name, rows, width, gated=False, tanh=False, dtype="bf16", train=True):
    """`width` of the result; a gated input is twice as wide."""
    return {"name": name, "op": "act", "rows": rows, "width": width, "gated": gated, "tanh": tanh, "dtype": dtype,
            "train": train}


def _keep(name, rows, width, dtype="bf16"):
    return {"name": name, "op": "keep", "rows": rows, "width": width, "dtype": dtype, "train": False}


def listed():
    return [
        # one generated token's embedding: latency only
        _embed("embed_one_token", 1, 32000, 1280, table="bf16", dtype="bf16", train=False),
        # char GPT: 64 sequences of 256 tokens, each row of the gradient a sum over hundreds of tokens
        _embed("embed_char", 16384, 65, 384),
        # a language model's micro-batch: rows scaled by sqrt(width), most of the vocabulary without a token
        _embed("embed_wide", 32768, 50257, 4096, table="bf16", dtype="bf16", scale=64.0),
        # one new token of each of 64 sequences, far into long contexts
        _qk("qk_decode", 64, 1, 32, 8, 128, base=5e5, far=1 << 20, train=False),
        # char GPT with grouped heads
        _qk("qk_char", 64, 256, 6, 3, 64),
        # a head dimension between powers of two, half of it rotated in adjacent pairs, in half precision
        _qk("qk_partial", 1, 4099, 20, 5, 80, rotary=40, interleaved=True, dtype="f16"),
        # a language model's micro-batch of packed documents, bound by memory
        _qk("qk_packed", 1, 32768, 32, 8, 128, base=5e5, far=1 << 17),
        # char GPT's feed-forward
        _act("gelu_char", 16384, 1536),
        # rows that begin on no vector boundary, the tanh form
        _act("gelu_odd", 4099, 2051, tanh=True, dtype="f16"),
        # SDXL's gated feed-forward at the 64 x 64 level, two images
        _act("geglu_image", 8192, 2560, gated=True),
        # the input of SDXL's 5120 -> 1280 linear, kept in 8 bits from forward to backward
        _keep("keep8_image", 2048, 5120),
        # fp32 activations with a ragged last block
        _keep("keep8_odd", 4099, 1283, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "qk", "qk", "act", "act", "keep"])
    train = rng.random() < 0.7
    most = 1.0e9   # bytes; the listed cases' largest has 1.3e9
    while True:
        if op == "embed":
            width = _log_int(rng, 32, 8192)
            if rng.random() < 0.7:
                width = max(32, width // 32 * 32)
            c = _embed("", _log_int(rng, 1, 131072), _log_int(rng, 65, 160000), width, table=rng.choice(["fp32", "bf16"]),
                       dtype=rng.choice(["fp32", "bf16", "bf16", "f16"]), scale=rng.choice([1.0, 8.0, 0.5]),
                       pad=rng.choice([0.0, 0.0, 0.1]), train=train)
        elif op == "qk":
            dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 256])
            kv_heads = rng.choice([1, 2, 4, 5, 8])
            rotary = rng.choice([dim, dim, dim // 16 * 8])
            c = _qk("", _log_int(rng, 1, 64), _log_int(rng, 1, 16384), kv_heads * rng.choice([1, 2, 3, 4]), kv_heads, dim,
                    rotary=rotary, interleaved=rng.random() < 0.3, base=rng.choice([1e4, 5e5]),
                    far=rng.choice([0, 1 << 17, 1 << 20]), dtype=rng.choice(["bf16", "bf16", "f16", "fp32"]),
                    train=train)
        else:
            width = _log_int(rng, 16, 16384)
            if rng.random() < 0.7:
                width = max(32, width // 32 * 32)
            dtype = rng.choice(["bf16", "bf16", "f16", "fp32"])
            rows = _log_int(rng, 1, 65536)
            if op == "act":
                c = _act("", rows, width, gated=rng.random() < 0.4, tanh=rng.random() < 0.4, dtype=dtype, train=train)
            else:
                c = _keep("", rows, width, dtype=dtype)
        if work(c)["bytes"] <= most:
            del c["name"]
            return c


# ---- inputs -----------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    s = dict(case)
    train = case["train"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "embed":
        n, vocab, width = case["tokens"], case["vocab"], case["width"]
        # the r-th commonest token with probability ~ 1 / (r + 3), its number anywhere in the vocabulary
        cdf = torch.cumsum(1.0 / (torch.arange(vocab, device=DEV, dtype=torch.float64) + 3.0), 0)
        rank = torch.searchsorted(cdf / cdf[-1], rand(n).double()).clamp_max_(vocab - 1)
        tokens = torch.randperm(vocab, generator=gen, device=DEV)[rank]
        if case["pad"]:
            tokens = torch.where(rand(n) < case["pad"], -1, tokens)
        s["tokens"] = tokens
        s["weight"] = (0.02 * randn(vocab, width)).to(DTYPES[case["table"]]).requires_grad_(train)
        if train:
            s["dy"] = (1e-2 * randn(n, width)).to(dt)
    elif case["op"] == "qk":
        b, t, h, hk, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        # one projection's output, split: rows of q, k and v side by side; some channels stand out
        gain = torch.where(rand(d) < 0.05, 6.0, 1.0)
        qkv = (randn(b, t, h + 2 * hk, d) * gain).to(dt)
        q, k, _ = qkv.split([h, hk, hk], dim=2)
        s["q"], s["k"] = (x.detach().requires_grad_(train) for x in (q, k))
        s["q_weight"], s["k_weight"] = ((1.0 + 0.2 * randn(d)).requires_grad_(train) for _ in range(2))
        if case["far"]:
            # documents one after another, each from a place of its own
            first = torch.randint(0, max(1, case["far"] - t), (b, 1), generator=gen, device=DEV)
            s["positions"] = first + torch.arange(t, device=DEV)
        else:
            s["positions"] = None
        if train:
            s["dq"], s["dk"] = (1e-2 * randn(b, t, h, d)).to(dt), (1e-2 * randn(b, t, hk, d)).to(dt)
    else:
        rows = case["rows"]
        width = case["width"] * (2 if case.get("gated") else 1)
        # a feed-forward's input: a few channels far larger than the rest
        gain = torch.where(rand(width) < 0.01, 8.0, 1.0)
        s["x"] = (1.2 * randn(rows, width) * gain).to(dt).requires_grad_(train)
        if train:
            s["dy"] = (1e-2 * randn(rows, case["width"])).to(dt)
    return s


# ---- the passes -------------------------------------------------------------
def run(s):
    one = {"embed": _run_embed, "qk": _run_qk, "act": _run_act, "keep": _run_keep}[s["op"]]
    if not s["train"] or not own:
        with torch.no_grad():
            return one(s)
    return one(s)


def _run_embed(s):
    tokens, w, scale, dt = s["tokens"], s["weight"], s["scale"], DTYPES[s["dtype"]]
    if own:
        import concord_amd as ca
        y = ca.embedding(tokens, w, scale=scale, dtype=dt)
        if not s["train"]:
            return {"y": y}
        dw, = torch.autograd.grad(y, (w,), s["dy"])
        return {"y": y.detach(), "dw": dw}
    there = tokens >= 0
    at = tokens.clamp_min(0)
    y = (w[at].float() * there[:, None] * scale).to(dt)
    if not s["train"]:
        return {"y": y}
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    dw.index_add_(0, at, s["dy"].double() * there[:, None])
    return {"y": y, "dw": (dw * scale).to(w.dtype)}


def _pairs(x, rotary, interleaved):
    """(first, second, rest) of the last dimension: what is rotated, in pairs, and what is not"""
    r, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        return r[..., 0::2], r[..., 1::2], rest
    return r[..., :rotary // 2], r[..., rotary // 2:], rest


def _joined(a, b, rest, interleaved):
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _positions(s):
    if s["positions"] is not None:
        return s["positions"]
    return torch.arange(s["tokens"], device=DEV).expand(s["batch"], -1)


def _run_qk(s):
    q, k, wq, wk = s["q"], s["k"], s["q_weight"], s["k_weight"]
    if own:
        import concord_amd as ca
        yq, yk = ca.qk_norm_rope(q, k, wq, wk, positions=s["positions"], base=s["base"], rotary_dim=s["rotary"],
                                 interleaved=s["interleaved"], eps=EPS)
        if not s["train"]:
            return {"q": yq, "k": yk}
        dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), (q, k, wq, wk), (s["dq"], s["dk"]))
        return {"q": yq.detach(), "k": yk.detach(), "dq": dq, "dk": dk, "dq_weight": dwq, "dk_weight": dwk}
    half = s["rotary"] // 2
    freq = s["base"] ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    angle = _positions(s).double()[..., None, None] * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    out = {}
    for name, x, w in (("q", q, wq), ("k", k, wk)):
        xf = x.float()
        r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
        h = xf * r
        a, b, rest = _pairs(h * w, s["rotary"], s["interleaved"])
        out[name] = _joined(a * cos - b * sin, a * sin + b * cos, rest, s["interleaved"]).to(x.dtype)
        if s["train"]:
            a, b, rest = _pairs(s["d" + name].float(), s["rotary"], s["interleaved"])
            du = _joined(a * cos + b * sin, b * cos - a * sin, rest, s["interleaved"])
            g = du * w
            out["d" + name] = (r * (g - h * (g * h).mean(-1, keepdim=True))).to(x.dtype)
            out["d" + name + "_weight"] = (du * h).sum((0, 1, 2), dtype=torch.float64).float()
    return out


def _pow2(e):
    """2^e in 32 bits, e from -126 to 127: the exponent's bits (pow may be off by a rounding)"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _kept(x):
    """What the 8-bit form of x stands for, in 32 bits: blocks of 32 values share the smallest
    power of two that takes the largest to 127 or less."""
    width = x.shape[-1]
    b = torch.nn.functional.pad(x.float(), (0, -width % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)   # top = m 2^e, m in [0.5, 1)
    e = torch.where(m * 128.0 > 127.0, e - 6, e - 7).clamp_min(-126)
    e = torch.where(top == 0, -126, e)
    v = (torch.round(b * _pow2(-e)) * _pow2(e)).flatten(-2)[..., :width]
    most = torch.finfo(x.dtype).max
    return v.clamp(-most, most)


def _gelu(x, tanh):
    """gelu and its derivative"""
    if tanh:
        c, a = math.sqrt(2.0 / math.pi), 0.044715
        t = 1.0 / (1.0 + torch.exp(-2.0 * c * (x + a * x * x * x)))   # (1 + tanh) / 2
        return x * t, t + x * t * (1.0 - t) * (2.0 * c) * (1.0 + 3.0 * a * x * x)
    cdf = 0.5 * torch.special.erfc(x * -math.sqrt(0.5))
    return x * cdf, cdf + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)


def _run_act(s):
    x, tanh = s["x"], s["tanh"]
    if own:
        import concord_amd as ca
        f = ca.geglu8 if s["gated"] else ca.gelu8
        y = f(x, approximate="tanh" if tanh else "none")
        if not s["train"]:
            return {"y": y}
        dx, = torch.autograd.grad(y, (x,), s["dy"])
        return {"y": y.detach(), "dx": dx}
    if s["gated"]:
        a, g = x.chunk(2, dim=-1)
        out = {"y": (a.float() * _gelu(g.float(), tanh)[0]).to(x.dtype)}
        if s["train"]:
            a, g, dy = _kept(a), _kept(g), s["dy"].float()
            v, d = _gelu(g, tanh)
            out["dx"] = torch.cat((dy * v, dy * a * d), -1).to(x.dtype)
    else:
        out = {"y": _gelu(x.float(), tanh)[0].to(x.dtype)}
        if s["train"]:
            out["dx"] = (s["dy"].float() * _gelu(_kept(x), tanh)[1]).to(x.dtype)
    return out


def _run_keep(s):
    if own:
        import concord_amd as ca
        codes, exponents = ca.pack8(s["x"])
        return {"x": ca.unpack8(codes, exponents, s["x"].dtype)}
    return {"x": _kept(s["x"]).to(s["x"].dtype)}


# ---- work -------------------------------------------------------------------
def _size(name):
    return 4 if name == "fp32" else 2


def work(case):
    train, es = case["train"], _size(case["dtype"])
    if case["op"] == "embed":
        n, v, c, ws = case["tokens"], case["vocab"], case["width"], _size(case["table"])
        # the rows that the tokens name, each once, and the result; then its gradient and the table's
        p = 1.0 / (torch.arange(v, dtype=torch.float64) + 3.0)
        p = p / p.sum()
        rows = float((1.0 - (1.0 - p) ** n).sum())   # distinct ones to be expected
        fwd = rows * c * ws + n * c * es + n * 8
        return {"bytes": float(fwd + (n * c * es + v * c * ws if train else 0)), "flops": n * c * (2.0 if train else 1.0)}
    if case["op"] == "qk":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        # in and out; for training dy and dx too; positions, weights and their gradients
        return {"bytes": float(n * es * (4 if train else 2) + case["batch"] * case["tokens"] * (8 if case["far"] else 0) +
                               case["dim"] * 4 * (4 if train else 2)),
                "flops": n * (20.0 if train else 7.0)}
    n = case["rows"] * case["width"]
    if case["op"] == "act":
        wide = 2 if case["gated"] else 1
        # x and y; for training dy and dx too (what is kept in between is neither input nor output)
        return {"bytes": float(n * es * (wide + 1) * (2 if train else 1)), "flops": n * (30.0 if train else 12.0)}
    return {"bytes": float(n * es * 2), "flops": n * 4.0}


# ---- the definitions in 64 bits ---------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embed": _exact_embed, "qk": _exact_qk, "act": _exact_act, "keep": _exact_keep}[case["op"]](s)


def _exact_embed(s):
    # a row of zeros behind the table takes the tokens that stand for nothing
    w = s["weight"].double()
    v, c = w.shape
    at = torch.where(s["tokens"] < 0, v, s["tokens"])
    table = torch.cat((w, w.new_zeros(1, c)))
    out = {"y": s["scale"] * torch.index_select(table, 0, at)}
    if s["train"]:
        order = torch.argsort(at, stable=True)
        count = torch.bincount(at, minlength=v + 1)
        dw = torch.segment_reduce(s["dy"].double()[order], "sum", lengths=count, initial=0.0)
        out["dw"] = s["scale"] * dw[:v]
    return out


def _exact_qk(s):
    d, rot = s["dim"], s["rotary"]
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    theta = _positions(s).double()[:, :, None, None] / s["base"] ** (2.0 * i / rot)
    turn = torch.polar(torch.ones_like(theta), theta)
    # places of the pairs' real and imaginary parts
    at = torch.arange(rot, device=DEV).view(-1, 2).T if s["interleaved"] else torch.arange(rot, device=DEV).view(2, -1)

    def rotated(x, by):
        y = x.clone()
        z = torch.complex(x[..., at[0]], x[..., at[1]]) * by
        y[..., at[0]], y[..., at[1]] = z.real, z.imag
        return y
    out = {}
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"].double()
        rms = torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS)
        out[name] = rotated(x / rms * w, turn)
        if s["train"]:
            du = rotated(s["d" + name].double(), turn.conj())
            along = (du * w * x).sum(-1, keepdim=True) / (d * rms ** 2)
            out["d" + name] = (du * w - along * x) / rms
            out["d" + name + "_weight"] = (du * x / rms).flatten(0, 2).sum(0)
    return out


def _exact_kept(x):
    """block by block: the step by search among the powers of two"""
    w = x.shape[-1]
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    full = w // BLOCK * BLOCK
    for piece in (slice(0, full), slice(full, w)):
        v = x[..., piece].double()
        if v.shape[-1] == 0:
            continue
        v = v.unflatten(-1, (-1, min(BLOCK, v.shape[-1])))
        top = v.abs().amax(-1, keepdim=True)
        # the powers of two from the exponent's bits of 64-bit numbers
        powers = (torch.arange(-126, 123, device=DEV) + 1023 << 52).view(torch.float64)
        step = powers[torch.searchsorted(127.0 * powers, top)]   # the first that takes the largest to 127 or less
        out[..., piece] = ((v / step).round() * step).flatten(-2)
    most = torch.finfo(x.dtype).max
    return out.clamp(-most, most)


def _exact_gelu(x, tanh):
    if tanh:
        u = math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)
        t = torch.tanh(u)
        du = math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * x ** 2)
        return 0.5 * x * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * du
    phi = torch.exp(-x * x / 2.0) * (2.0 * math.pi) ** -0.5
    cdf = torch.special.erfc(-x / 2.0 ** 0.5) / 2.0   # (1 + erf, or ndtr, loses the left tail)
    return x * cdf, cdf + x * phi


def _exact_act(s):
    x, c = s["x"], s["width"]
    if not s["gated"]:
        out = {"y": _exact_gelu(x.double(), s["tanh"])[0]}
        if s["train"]:
            out["dx"] = s["dy"].double() * _exact_gelu(_exact_kept(x), s["tanh"])[1]
        return out
    out = {"y": x[:, :c].double() * _exact_gelu(x[:, c:].double(), s["tanh"])[0]}
    if s["train"]:
        a, g = _exact_kept(x[:, :c]), _exact_kept(x[:, c:])
        v, d = _exact_gelu(g, s["tanh"])
        out["dx"] = s["dy"].double().repeat(1, 2) * torch.cat((v, a * d), 1)
    return out


def _exact_keep(s):
    return {"x": _exact_kept(s["x"])}
