"""CPU-side checks of embedding, norms of queries and keys with the rotation, and the
8-bit activations: every refusal comes before any GPU work, from the operators (which
look at shapes and types before the device) and from the C entries; and what the
backwards hand to their kernels where saved tensors come back in another layout."""
import ctypes
import importlib.util
import os
import re
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def L():
    from concord_amd import _lib as C
    return C.lib()


def test_cpu_tensors_are_refused():
    import concord_amd as ca
    x, q, i = torch.zeros(2, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int64)
    codes, exps = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8)
    for call in (lambda: ca.embedding(i, x), lambda: ca.qk_norm_rope(q, q), lambda: ca.gelu8(x), lambda: ca.geglu8(x),
                 lambda: ca.pack8(x), lambda: ca.unpack8(codes, exps)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_embedding_refusals():
    import concord_amd as ca
    i, w = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)
    for args, kw, kind in [((i.float(), w), {}, TypeError), ((i.short(), w), {}, TypeError), ((i, w.double()), {}, TypeError),
                           ((i, w.long()), {}, TypeError), ((i, w), {"dtype": torch.float64}, TypeError),
                           ((i, w), {"dtype": "bf16"}, TypeError), ((i, w[0]), {}, ValueError),
                           ((i, w[:, :0]), {}, ValueError), ((i, w[None]), {}, ValueError),
                           ((i, w), {"scale": float("nan")}, ValueError), ((i, w), {"scale": float("inf")}, ValueError),
                           ((i.to("meta"), w), {}, ValueError)]:
        with pytest.raises(kind, match="embedding"):
            ca.embedding(*args, **kw)


def test_embedding_scales_past_32_bits_are_refused(L):
    # the kernels hold the scale in fp32: infinite there, a token outside the table would get NaN for zeros
    import concord_amd as ca
    from concord_amd import _lib as C
    i, w = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)
    for scale in (1e39, -1e300):
        with pytest.raises(ValueError, match="embedding: the scale"):
            ca.embedding(i, w, scale=scale)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ca.embedding(i, w, scale=3e38)
    for scale in (float("inf"), float("nan")):
        assert L.concord_embedding_fwd(None, 1, 0, None, 8, C.F32, 5, 8, scale, None, 8, C.F32, None) == C.EINVAL
        assert L.concord_embedding_bwd(None, 1, 0, None, 8, C.F32, 0, 8, scale, None, 8, C.F32, None, 0, None) == C.EINVAL


def test_qk_refusals():
    import concord_amd as ca

    def t(*shape, dtype=F32):
        return torch.zeros(*shape, dtype=dtype)
    q, w, p = t(6, 4, 64), t(64), torch.zeros(6, dtype=torch.int64)
    bad = [
        ((q.double(), q.double()), {}, TypeError), ((q, t(6, 4, 64, dtype=BF16)), {}, TypeError),
        ((q, t(6, 4, 32)), {}, ValueError), ((t(6, 4, 12), t(6, 4, 12)), {}, ValueError),
        ((t(6, 4, 264), t(6, 4, 264)), {}, ValueError), ((t(6, 4, 0), t(6, 4, 0)), {}, ValueError),
        ((q, t(5, 4, 64)), {}, ValueError), ((q, t(1, 6, 4, 64)), {}, ValueError), ((t(6, 64), t(6, 64)), {}, ValueError),
        ((q, t(6, 0, 64)), {}, ValueError), ((q, q, t(63)), {}, ValueError), ((q, q, None, t(1, 64)), {}, ValueError),
        ((q, q, w.double()), {}, TypeError), ((q, q, w, w.bfloat16()), {}, TypeError), ((q, q, w.to("meta")), {}, ValueError),
        ((q, q), {"positions": p.float()}, TypeError), ((q, q), {"positions": p[:5]}, ValueError),
        ((q, q), {"positions": p[:, None]}, ValueError), ((q, q), {"positions": p.to("meta")}, ValueError),
        ((t(2, 3, 4, 64), t(2, 3, 4, 64)), {"positions": torch.zeros(2, dtype=torch.int64)}, ValueError),
        ((q, q), {"rotary_dim": 72}, ValueError), ((q, q), {"rotary_dim": 12}, ValueError),
        ((q, q), {"rotary_dim": -8}, ValueError), ((q, q), {"base": 0.0}, ValueError),
        ((q, q), {"base": float("nan")}, ValueError), ((q, q), {"base": float("inf")}, ValueError),
        ((q, q), {"eps": -1e-6}, ValueError), ((q, q), {"eps": float("nan")}, ValueError),
    ]
    for args, kw, kind in bad:
        with pytest.raises(kind, match="qk_norm_rope"):
            ca.qk_norm_rope(*args, **kw)


def test_activation_refusals():
    import concord_amd as ca
    x = torch.zeros(2, 64)
    for f, name in ((ca.gelu8, "gelu8"), (ca.geglu8, "geglu8"), (ca.pack8, "pack8")):
        for bad, kind in ((x.double(), TypeError), (x.long(), TypeError), (torch.zeros(()), ValueError), (x[:, :0], ValueError)):
            with pytest.raises(kind, match=name):
                f(bad)
    for f in (ca.gelu8, ca.geglu8):
        with pytest.raises(ValueError, match="approximate"):
            f(x, approximate="fast")
    with pytest.raises(ValueError, match="two halves"):
        ca.geglu8(x[:, :63])
    codes, exps = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8)
    for args, kind in (((codes.int(), exps), TypeError), ((codes, codes), TypeError), ((codes, exps, torch.float64), TypeError),
                       ((codes, exps[:, :1]), ValueError), ((codes[:1], exps), ValueError), ((codes, exps[0]), ValueError),
                       ((codes[:, :0], exps), ValueError), ((codes, exps.to("meta")), ValueError)):
        with pytest.raises(kind, match="unpack8"):
            ca.unpack8(*args)


def test_input_bits_refusals():
    from concord_amd import packed_b as pb
    for bits in (0, 4, 32, "8", None):
        with pytest.raises(ValueError, match="input bits"):
            pb.ConcordLinearPackedB.set_input_bits(object.__new__(pb.ConcordLinearPackedB), bits)
    with pytest.raises(ValueError, match="input bits"):
        pb.ConcordConv2dPackedB.set_input_bits(object.__new__(pb.ConcordConv2dPackedB), 8)


def test_embedding_entry_refusals(L):
    from concord_amd import _lib as C
    keep = ctypes.create_string_buffer(256)
    b = ctypes.addressof(keep) + 15 & ~15
    fwd = [b, 1, 2, b, 8, C.F32, 5, 8, 1.0, b, 8, C.F32, None]
    for at, v in ((0, None), (2, -1), (2, 1 << 31), (3, None), (4, 7), (5, 3), (6, -1), (6, (1 << 31) - 1), (7, 0), (7, 1 << 21),
                  (9, None), (10, 7), (11, -1)):
        args = list(fwd)
        args[at] = v
        assert L.concord_embedding_fwd(*args) == C.EINVAL, (at, v)
    assert L.concord_embedding_fwd(None, 1, 0, None, 8, C.F32, 5, 8, 1.0, None, 8, C.F32, None) == C.OK
    need = L.concord_embedding_workspace_bytes(2, 5, 8)
    assert need > 0
    for sizes in ((0, 5, 8), (2, 0, 8), (-1, 5, 8), (2, -5, 8), (2, 5, 0), (1 << 31, 5, 8), (2, 5, 1 << 21)):
        assert L.concord_embedding_workspace_bytes(*sizes) == 0, sizes
    bwd = [b, 1, 2, b, 8, C.F32, 5, 8, 1.0, b, 8, C.F32, b, need, None]
    for at, v in ((0, None), (2, -1), (3, None), (4, 7), (5, 3), (6, -1), (7, 0), (9, None), (10, 7), (11, 9), (12, b + 4)):
        args = list(bwd)
        args[at] = v
        assert L.concord_embedding_bwd(*args) == C.EINVAL, (at, v)
    assert L.concord_embedding_bwd(*bwd[:12], b, need - 1, None) == C.EWORKSPACE
    assert L.concord_embedding_bwd(*bwd[:12], None, need, None) == C.EWORKSPACE
    assert L.concord_embedding_bwd(*(bwd[:6] + [0] + bwd[7:])) == C.OK   # no row
    # more work items than a launch has
    n, c = (1 << 31) - 1, (1 << 21) - 1
    big = [b, 1, n, b, c, C.F32, 5, c, 1.0, b, c, C.F32, b, L.concord_embedding_workspace_bytes(n, 5, c), None]
    assert L.concord_embedding_bwd(*big) == C.EINVAL
    assert b"too many" in L.concord_last_error()


def _qk_args(buf, **kw):
    from concord_amd import _lib as C
    a = C.QkArgs()
    p = (ctypes.addressof(buf) + 15) & ~15
    for n in ("q", "k", "q_out", "k_out", "dq_out", "dk_out", "dq", "dk", "q_weight", "k_weight", "positions"):
        setattr(a, n, p)
    for n in ("q_t", "k_t", "dq_t", "dk_t", "q_h", "k_h", "dq_h", "dk_h"):
        setattr(a, n, 64)
    a.T, a.seq, a.pos_seq, a.H, a.HK, a.D, a.R, a.base, a.eps = 4, 4, 4, 1, 1, 64, 64, 1e4, 1e-6
    for n, v in kw.items():
        setattr(a, n, p + v[0] if isinstance(v, tuple) else v)
    return a


def test_qk_entry_refusals(L):
    from concord_amd import _lib as C
    buf = ctypes.create_string_buffer(64)
    sizes = [dict(T=-1), dict(T=1 << 31), dict(H=-1), dict(H=0, HK=0), dict(H=1 << 14), dict(D=0), dict(D=12), dict(D=264),
             dict(R=-8), dict(R=72), dict(R=12)]
    both = sizes + [dict(dtype=3), dict(wtype=-1), dict(base=0.0), dict(base=float("nan")), dict(eps=-1.0), dict(seq=0),
                    dict(seq=5), dict(pos_seq=0), dict(pos_seq=5), dict(q=None), dict(k=None), dict(q=(8,)), dict(k=(4,)),
                    dict(q_t=60), dict(k_h=4)]
    for kw in both + [dict(q_out=None), dict(k_out=(8,))]:
        a = _qk_args(buf, **kw)
        assert L.concord_qk_norm_rope_fwd(ctypes.byref(a), None) == C.EINVAL, kw
    for kw in both + [dict(dq=None), dict(dk=(8,)), dict(dq_out=None), dict(dk_out=(8,)), dict(dq_t=4), dict(dk_h=9)]:
        a = _qk_args(buf, **kw)
        assert L.concord_qk_norm_rope_bwd(ctypes.byref(a), None, 0, None) == C.EINVAL, kw
    for kw in sizes:
        assert L.concord_qk_norm_rope_workspace_bytes(ctypes.byref(_qk_args(buf, **kw))) == 0, kw
    assert L.concord_qk_norm_rope_workspace_bytes(None) == 0
    assert L.concord_qk_norm_rope_fwd(None, None) == C.EINVAL
    a = _qk_args(buf, dq_weight=(0,))
    need = L.concord_qk_norm_rope_workspace_bytes(ctypes.byref(a))
    assert need > 0
    assert L.concord_qk_norm_rope_bwd(ctypes.byref(a), None, need, None) == C.EWORKSPACE
    assert L.concord_qk_norm_rope_bwd(ctypes.byref(a), buf, need - 1, None) == C.EWORKSPACE
    empty = _qk_args(buf, T=0, q=None, k=None, q_out=None, k_out=None)
    assert L.concord_qk_norm_rope_fwd(ctypes.byref(empty), None) == C.OK
    assert L.concord_qk_norm_rope_bwd(ctypes.byref(empty), None, 0, None) == C.OK


def test_qk_struct_matches_the_header():
    from concord_amd import _lib as C
    src = open(os.path.join(os.path.dirname(HERE), "include", "concord_amd.h")).read()
    body = re.search(r"typedef struct concord_qk_args \{(.*?)\} concord_qk_args;", src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for decl in body.split(";") for n in re.findall(r"\*?(\w+)\s*(?:,|$)", decl.strip())]
    assert names == [n for n, _ in C.QkArgs._fields_]


def test_act8_entry_refusals(L):
    from concord_amd import _lib as C
    buf = ctypes.create_string_buffer(64)
    b = ctypes.addressof(buf)
    pack = [b, 64, C.BF16, 2, 64, b, b, None]
    unpack = [b, b, 2, 64, b, 64, C.BF16, None]
    fwd = [b, 64, C.BF16, 2, 64, 0, 0, b, 64, b, b, None]
    bwd = [b, 64, b, b, C.BF16, 2, 64, 0, 0, b, 64, None]
    for f, base, bad in (
            (L.concord_pack8, pack, ((0, None), (1, 63), (2, 3), (3, -1), (4, 0), (5, None), (6, None), (3, 1 << 39))),
            (L.concord_unpack8, unpack, ((0, None), (1, None), (2, -1), (3, 0), (4, None), (5, 63), (6, 7), (2, 1 << 39))),
            (L.concord_gelu8_fwd, fwd, ((0, None), (1, 63), (2, 3), (3, -1), (4, 0), (5, 1), (7, None), (8, 63), (9, None),
                                        (10, None), (3, 1 << 39))),
            (L.concord_gelu8_bwd, bwd, ((0, None), (1, 63), (2, None), (3, None), (4, 3), (5, -1), (6, 0), (7, 1), (9, None),
                                        (10, 63), (5, 1 << 39)))):
        for at, v in bad:
            args = list(base)
            args[at] = v
            assert f(*args) == C.EINVAL, (f, at, v)
    assert L.concord_pack8(None, 64, C.F32, 0, 64, None, None, None) == C.OK
    assert L.concord_gelu8_fwd(None, 64, C.F32, 0, 64, 0, 0, None, 64, None, None, None) == C.OK


# ---- saved tensors that come back in another layout --------------------------------------
@pytest.fixture(scope="session")
def stub(tmp_path_factory):
    from concord_amd import build as B
    out = str(tmp_path_factory.mktemp("block_stub") / "concord_block_stub.so")
    cflags, libs = B._ops_flags()
    cflags = ["-O0" if f == "-O2" else f for f in cflags if "TORCH_EXTENSION_NAME" not in f]
    libs = [f for f in libs if f != "-lconcord_amd"] + ["-Wl,-rpath," + os.path.join(os.path.dirname(torch.__file__), "lib")]
    r = subprocess.run([B.CXX] + cflags + ["-DTORCH_EXTENSION_NAME=concord_block_stub", "-shared", "-o", out,
                                           os.path.join(HERE, "block_operators_stub.cpp")] + libs, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    spec = importlib.util.spec_from_file_location("concord_block_stub", out)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _relaid(layout, t):
    """t in a buffer of its own, other values around it"""
    t = t.detach()
    fill = float("nan") if t.is_floating_point() else 77
    if layout == "reversed":
        shape = t.shape[::-1]
        buf = torch.full(shape, fill, dtype=t.dtype)
        return buf.permute(*range(t.dim())[::-1]).copy_(t)
    gap, off = (1, 1) if layout == "shifted" else (3, 0)
    buf = torch.full((t.numel() * gap + 64,), fill, dtype=t.dtype)
    strides, n = [], gap
    for d in reversed(t.shape):
        strides.insert(0, n)
        n *= max(d, 1)
    return buf.as_strided(t.shape, strides, off).copy_(t)


def _recorded(stub, make, layout):
    if layout is None:
        y, leaves, up = make()
    else:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: _relaid(layout, t)):
            y, leaves, up = make()
    stub.recorded()
    grads = torch.autograd.grad(y, leaves, up)
    assert all(g.shape == p.shape and g.dtype == p.dtype for g, p in zip(grads, leaves))
    seen, misaligned = stub.recorded()
    assert not misaligned, misaligned
    return dict(seen)


def _randn(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("layout", ["shifted", "gaps", "reversed"])
@pytest.mark.parametrize("op", ["embedding", "embedding2", "qk", "qk4", "qk_bare", "gelu8", "geglu8"])
def test_saved_tensors_in_other_layouts(stub, op, layout):
    def make():
        if op.startswith("embedding"):
            tokens = torch.arange(12).view(3, 4).t() if op == "embedding2" else torch.arange(12, dtype=torch.int32)
            w = _randn(20, 24).requires_grad_(True)
            return stub.embedding(tokens, w, 2.0, BF16), (w,), _randn(*tokens.shape, 24, dtype=BF16, seed=1)
        if op.startswith("qk"):
            lead = (2, 5) if op == "qk4" else (7,)
            q, k = _randn(*lead, 6, 24, dtype=BF16)[..., :4, :], _randn(*lead, 2, 24, dtype=BF16, seed=1)
            q, k = (t.detach().requires_grad_(True) for t in (q, k))
            bare = op == "qk_bare"
            wq, wk = (None if bare else _randn(24, seed=s).requires_grad_(True) for s in (2, 3))
            pos = None if bare else torch.arange(lead[-1])
            y = stub.qk_norm_rope(q, k, wq, wk, pos, 1e4, 16, False, 1e-6)
            return y, (q, k) if bare else (q, k, wq, wk), [_randn(*t.shape, dtype=BF16, seed=4) for t in y]
        x = _randn(5, 3, 66, dtype=F16)[..., :64].detach().requires_grad_(True)
        y = stub.gelu8(x, "none") if op == "gelu8" else stub.geglu8(x, "tanh")
        return y, (x,), _randn(*y.shape, dtype=F16, seed=5)
    want, got = _recorded(stub, make, None), _recorded(stub, make, layout)
    assert len(want) >= 2 and want.keys() == got.keys()
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_another_saved_tensor_is_an_error(stub):
    w, q = _randn(20, 24).requires_grad_(True), _randn(7, 2, 24).requires_grad_(True)
    x = _randn(4, 64).requires_grad_(True)
    for make in (lambda: stub.embedding(torch.arange(12), w, 1.0, None), lambda: stub.qk_norm_rope(q, q, None, None, None, 1e4, None, False, 1e-6)[0],
                 lambda: stub.gelu8(x, "none")):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:2].detach()):
            y = make()
        with pytest.raises(RuntimeError, match="came back as another tensor"):
            y.sum().backward()


def test_tangents_are_errors(stub):
    import torch.autograd.forward_ad as fwd
    w, q, x = _randn(20, 24), _randn(7, 2, 24), _randn(4, 64)
    with fwd.dual_level():
        d = [fwd.make_dual(t, torch.ones_like(t)) for t in (w, q, x)]
        for call in (lambda: stub.embedding(torch.arange(12), d[0], 1.0, None),
                     lambda: stub.qk_norm_rope(q, d[1], None, None, None, 1e4, None, False, 1e-6),
                     lambda: stub.gelu8(d[2], "none"), lambda: stub.geglu8(d[2], "none"), lambda: stub.pack8(d[2])):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
