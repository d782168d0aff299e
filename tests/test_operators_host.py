"""CPU-side checks of layer norm, attention and distillation: every refusal comes
before any GPU work, from the operators (which look at shapes and types before
the device) and from the C entries."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from concord_amd import _lib as C
    return C.lib()


def test_cpu_tensors_are_refused():
    import concord_amd as ca
    t = torch.zeros(2, 3, 2, 8)
    for call in (lambda: ca.layer_norm(t), lambda: ca.attention(*[t.bfloat16()] * 3),
                 lambda: ca.distill_loss(t, t, t.long())):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_layer_norm_refusals():
    import concord_amd as ca
    x, w = torch.zeros(4, 8), torch.ones(8)
    for args, kind in [((x.double(),), TypeError), ((x, torch.ones(7)), ValueError), ((x, w.double()), TypeError),
                       ((x, w, w.bfloat16()), TypeError), ((x, torch.ones(1, 8)), ValueError),
                       ((torch.zeros(()),), ValueError), ((torch.zeros(4, 0),), ValueError)]:
        with pytest.raises(kind, match="layer_norm"):
            ca.layer_norm(*args)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ca.layer_norm(x, w)


def test_attention_refusals():
    import concord_amd as ca

    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype)
    q, s = t(6, 4, 64), torch.tensor([0, 6], dtype=torch.int32)
    bad = [
        ((t(6, 4, 64, dtype=torch.float32), q, q), {}, TypeError),
        ((q, t(6, 4, 64, dtype=torch.float16), q), {}, TypeError),
        ((q, t(6, 3, 64), t(6, 3, 64)), {}, ValueError),
        ((q, t(6, 4, 32), t(6, 4, 32)), {}, ValueError),
        ((q, q, t(5, 4, 64)), {}, ValueError),
        ((t(6, 4, 12), t(6, 4, 12), t(6, 4, 12)), {}, ValueError),
        ((t(6, 4, 136), t(6, 4, 136), t(6, 4, 136)), {}, ValueError),
        ((t(6, 4, 0), t(6, 4, 0), t(6, 4, 0)), {}, ValueError),
        ((t(6, 0, 64), t(6, 0, 64), t(6, 0, 64)), {}, ValueError),
        ((q, q, q), {"scale": 0.0}, ValueError),
        ((q, q, q), {"scale": -1.0}, ValueError),
        ((q, q, q), {"scale": float("nan")}, ValueError),
        ((q, q, q), {"starts": s.long()}, ValueError),
        ((q, q, q), {"starts": s.view(1, 2)}, ValueError),
        ((q, q, q), {"starts": s[:0]}, ValueError),
        ((q, q, q), {"k_starts": s}, ValueError),
        ((q, q, q), {"starts": s, "k_starts": s[:1]}, ValueError),
        ((q, t(7, 4, 64), t(7, 4, 64)), {"starts": s}, ValueError),
        ((q, t(1, 6, 4, 64), t(1, 6, 4, 64)), {}, ValueError),
        ((t(1, 6, 4, 64),) * 3, {"starts": s}, ValueError),
        ((t(2, 6, 4, 64), t(1, 6, 4, 64), t(1, 6, 4, 64)), {}, ValueError),
        ((t(6, 64),) * 3, {}, ValueError),
    ]
    for args, kw, kind in bad:
        with pytest.raises(kind, match="attention"):
            ca.attention(*args, **kw)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ca.attention(q, q, q)


def test_distill_refusals():
    import concord_amd as ca
    z, t, i = torch.zeros(4, 65), torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int64)
    for args, kw, kind in [((z.double(), t, i), {}, TypeError), ((z, t.long(), i), {}, TypeError),
                           ((z, t, t), {}, TypeError), ((z, t[:3], i), {}, ValueError),
                           ((z, t, i[:, :4]), {}, ValueError), ((z[:3], t, i), {}, ValueError),
                           ((z, t, i), {"temperature": 0.0}, ValueError),
                           ((z, t, i), {"temperature": float("inf")}, ValueError),
                           ((z, torch.zeros(4, 1025), torch.zeros(4, 1025, dtype=torch.int64)), {}, ValueError),
                           ((torch.zeros(4, 0), t, i), {}, ValueError)]:
        with pytest.raises(kind, match="distill_loss"):
            ca.distill_loss(*args, **kw)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ca.distill_loss(z, t, i)


def test_layernorm_entry_refusals(L):
    from concord_amd import _lib as C
    P, b = None, ctypes.create_string_buffer(256)
    fwd = lambda *a: L.concord_layernorm_fwd(*a)  # noqa: E731
    assert fwd(b, 8, C.F32, P, P, C.F32, -1, 8, 1e-5, b, 8, P, P, P) == C.EINVAL
    assert fwd(b, 8, 3, P, P, C.F32, 2, 8, 1e-5, b, 8, P, P, P) == C.EINVAL
    assert fwd(b, 7, C.F32, P, P, C.F32, 2, 8, 1e-5, b, 8, P, P, P) == C.EINVAL
    assert fwd(P, 8, C.F32, P, P, C.F32, 2, 8, 1e-5, b, 8, P, P, P) == C.EINVAL
    assert fwd(b, 8, C.F32, P, P, C.F32, 2, 8, 1e-5, b, 8, b, P, P) == C.EINVAL
    assert fwd(P, 8, C.F32, P, P, C.F32, 0, 8, 1e-5, P, 8, P, P, P) == C.OK
    need = L.concord_layernorm_workspace_bytes(100, 64)
    assert need >= 2 * 64 * 4 and L.concord_layernorm_workspace_bytes(0, 64) == 0
    bwd = (b, 64, b, 64, C.F32, P, C.F32, b, b, 100, 64, b, 64, b, P)
    assert L.concord_layernorm_bwd(*bwd, b, need - 1, P) == C.EWORKSPACE
    assert L.concord_layernorm_bwd(*bwd, P, need, P) == C.EWORKSPACE
    assert b"workspace" in L.concord_last_error()
    assert L.concord_layernorm_bwd(b, 64, b, 64, C.F32, P, C.F32, P, b, 100, 64, b, 64, P, P, P, 0, P) == C.EINVAL


def _attn_args(buf, **kw):
    from concord_amd import _lib as C
    a = C.AttnArgs()
    p = (ctypes.addressof(buf) + 15) & ~15
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv", "lse", "out_low"):
        setattr(a, n, p)
    for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        setattr(a, n + "_t", 64)
        setattr(a, n + "_h", 64)
    a.B, a.TQ, a.TK, a.H, a.HK, a.D, a.scale = 1, 4, 4, 1, 1, 64, 0.125
    for n, v in kw.items():
        setattr(a, n, p + v if n in ("q", "dk") else v)
    return a


def test_attention_entry_refusals(L):
    from concord_amd import _lib as C
    buf = ctypes.create_string_buffer(64)
    bad = [dict(TQ=-1), dict(TK=1 << 31), dict(B=-1), dict(D=4), dict(D=136), dict(D=60), dict(H=3, HK=2), dict(HK=0),
           dict(scale=0.0), dict(scale=float("inf")), dict(B=3), dict(B=0), dict(q=8), dict(v=None), dict(q_t=56),
           dict(k_t=68), dict(v_h=4), dict(q_t=1 << 24), dict(k_starts=1)]
    for kw in bad:
        a = _attn_args(buf, **kw)
        assert L.concord_attention_fwd(ctypes.byref(a), None, 0, None) == C.EINVAL, kw
        assert L.concord_attention_bwd(ctypes.byref(a), buf, 64, None) == C.EINVAL, kw
    for kw in (dict(dout=None), dict(dk=8), dict(dv_t=12), dict(lse=None), dict(out_low=None)):
        assert L.concord_attention_bwd(ctypes.byref(_attn_args(buf, **kw)), buf, 64, None) == C.EINVAL, kw
    a = _attn_args(buf)
    need = L.concord_attention_workspace_bytes(ctypes.byref(a))
    assert L.concord_attention_bwd(ctypes.byref(a), buf, need - 1, None) == C.EWORKSPACE
    assert L.concord_attention_fwd(None, None, 0, None) == C.EINVAL
    # one query of many keys: the forward needs room for its shares' sums
    long = _attn_args(buf, TQ=1, TK=32768)
    need = L.concord_attention_fwd_workspace_bytes(ctypes.byref(long))
    assert need > 0 and L.concord_attention_fwd_workspace_bytes(ctypes.byref(a)) == 0
    assert L.concord_attention_fwd(ctypes.byref(long), None, 0, None) == C.EWORKSPACE
    assert L.concord_attention_fwd(ctypes.byref(long), buf, need - 1, None) == C.EWORKSPACE
    # no token: nothing to do
    empty = _attn_args(buf, TQ=0, TK=0, B=0)
    assert L.concord_attention_fwd(ctypes.byref(empty), None, 0, None) == C.OK
    assert L.concord_attention_bwd(ctypes.byref(empty), None, 0, None) == C.OK


def test_attention_struct_matches_the_header():
    import os
    import re

    from concord_amd import _lib as C
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = open(os.path.join(root, "include", "concord_amd.h")).read()
    body = re.search(r"typedef struct concord_attn_args \{(.*?)\} concord_attn_args;", src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for decl in body.split(";") for n in re.findall(r"\*?(\w+)\s*(?:,|$)", decl.strip())]
    assert names == [n for n, _ in C.AttnArgs._fields_]


def test_distill_entry_refusals(L):
    from concord_amd import _lib as C
    P, b = None, ctypes.create_string_buffer(256)

    def fwd(z=b, ld=65, dt=0, M=2, V=65, t=b, ldt=4, i=b, ldi=4, K=4, T=1.0, loss=b, ws=P, n=0):
        return L.concord_distill_fwd(z, ld, dt, M, V, t, ldt, i, ldi, K, T, loss, P, ws, n, P)
    for kw in (dict(M=-1), dict(V=0), dict(K=1025, ldt=1025, ldi=1025), dict(K=-1), dict(dt=7), dict(ld=64), dict(ldt=3),
               dict(ldi=3), dict(T=0.0), dict(T=-1.0), dict(z=P), dict(t=P), dict(i=P), dict(loss=P)):
        assert fwd(**kw) == C.EINVAL, kw
    assert fwd(M=0, z=P, t=P, i=P, loss=P) == C.OK
    need = L.concord_distill_workspace_bytes(2, 50257)
    assert need > 0 and L.concord_distill_workspace_bytes(4096, 50257) == 0
    assert fwd(V=50257, ld=50257, ws=b, n=need - 1) == C.EWORKSPACE
    bwd = [b, 0, b, 65, 0, 2, 65, b, 4, b, 4, 4, 1.0, b, b, 65, P]
    for at, v in ((0, P), (1, -1), (13, P), (14, P), (15, 64)):
        args = list(bwd)
        args[at] = v
        assert L.concord_distill_bwd(*args) == C.EINVAL, at


BAD_ATTENTION_SIZES = [dict(B=0), dict(B=0, TQ=0), dict(B=0, TK=0), dict(B=-1), dict(B=1 << 24), dict(B=3), dict(TQ=-1), dict(TK=-4),
                       dict(TQ=1 << 31), dict(TK=1 << 31), dict(TQ=1 << 62, TK=1 << 62), dict(D=4), dict(D=0), dict(D=-8),
                       dict(D=136), dict(D=60), dict(H=0), dict(H=3, HK=2), dict(HK=0), dict(HK=-1), dict(H=1 << 16),
                       dict(k_starts=1)]


def test_attention_workspace_of_sizes_that_the_entries_refuse():
    """0, and no arithmetic on them: in a process of its own, since a division by
    B = 0 ends it."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = ("import ctypes, sys\n"
            "sys.path[:0] = [%r, %r]\n"
            "from concord_amd import _lib as C\n"
            "from test_operators_host import BAD_ATTENTION_SIZES, _attn_args\n"
            "L, buf = C.lib(), ctypes.create_string_buffer(64)\n"
            "for kw in BAD_ATTENTION_SIZES:\n"
            "    a = _attn_args(buf, **kw)\n"
            "    assert L.concord_attention_fwd(ctypes.byref(a), None, 0, None) == C.EINVAL, kw\n"
            "    assert L.concord_attention_bwd(ctypes.byref(a), None, 0, None) == C.EINVAL, kw\n"
            "    for f in (L.concord_attention_fwd_workspace_bytes, L.concord_attention_workspace_bytes):\n"
            "        print(kw, flush=True)\n"
            "        assert f(ctypes.byref(a)) == 0, kw\n"
            "assert L.concord_attention_workspace_bytes(None) == 0 == L.concord_attention_fwd_workspace_bytes(None)\n"
            % (os.path.dirname(here), here))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout[-200:], r.stderr[-2000:])


def test_a_module_that_fails_to_load_is_not_kept(monkeypatch):
    """ops() hands out the module once it has run, never before: a second thread
    would find no functions in it, and so would every call after a failed load."""
    import threading

    from concord_amd import _lib as C
    whole = C.ops()
    monkeypatch.setattr(C, "_ops", None)
    real, fail, started = C.importlib.util.spec_from_file_location, [True], []

    class Loader:
        def __init__(self, loader):
            self.loader = loader

        def create_module(self, spec):
            return self.loader.create_module(spec)

        def exec_module(self, m):
            assert C._ops is None
            started.append(threading.get_ident())
            if fail[0]:
                raise ImportError("no such symbol")
            other = threading.Thread(target=lambda: seen.append(C.ops()))
            other.start()
            other.join(0.2)   # it waits for this load, or has its own
            threads.append(other)
            self.loader.exec_module(m)

    def spec(name, path):
        s = real(name, path)
        s.loader = Loader(s.loader)
        return s
    seen, threads = [], []
    monkeypatch.setattr(C.importlib.util, "spec_from_file_location", spec)
    for _ in range(2):
        with pytest.raises(ImportError, match="no such symbol"):
            C.ops()
    fail[0] = False
    m = C.ops()
    threads[0].join(10)
    assert len(seen) == 1 and len(started) == 3
    for n in ("layer_norm", "attention", "distill_loss"):
        assert callable(getattr(m, n)) and callable(getattr(seen[0], n)) and callable(getattr(whole, n))
    assert seen[0] is m and C.ops() is m


def test_launches_past_the_grid_are_refused(L):
    """A launch has 32 bits of work items: 2^24 workgroups of 256 are too many."""
    from concord_amd import _lib as C
    buf, most = ctypes.create_string_buffer(64), (2 ** 32 - 1) // 256
    # dense: one tile a sequence and head; tables: TQ / 128 + B + 2 slots a head
    for kw in (dict(B=(most + 16) // 16, TQ=(most + 16) // 16, TK=(most + 16) // 16, H=16, HK=16),
               dict(B=1, TQ=2 ** 30, TK=64, H=64, HK=64),
               dict(B=2 ** 23, TQ=2 ** 23, TK=2 ** 23, H=2, HK=1, starts=16)):
        a = _attn_args(buf, **kw)
        assert L.concord_attention_fwd(ctypes.byref(a), None, 0, None) == C.EINVAL, kw
        assert b"too many tiles" in L.concord_last_error()
        need = L.concord_attention_workspace_bytes(ctypes.byref(a))
        assert L.concord_attention_bwd(ctypes.byref(a), buf, need, None) == C.EINVAL, kw
        assert b"too many tiles" in L.concord_last_error()
    # few queries, many keys: the backward's second launch
    a = _attn_args(buf, B=1, TQ=1, TK=2 ** 30, H=64, HK=64)
    need = L.concord_attention_workspace_bytes(ctypes.byref(a))
    assert L.concord_attention_bwd(ctypes.byref(a), buf, need, None) == C.EINVAL
    assert b"too many tiles" in L.concord_last_error()
    # gradients of logits in segments; sums over the columns, 64 a workgroup of 1024
    M, V, b = 2 ** 24 - 1, 20000, ctypes.addressof(buf) + 15 & ~15
    assert L.concord_distill_bwd(b, 0, b, V, C.F32, M, V, b, 4, b, 4, 4, 1.0, b, b, V, None) == C.EINVAL
    width = (2 ** 32 - 1) // 1024 * 32 + 32
    need = L.concord_layernorm_workspace_bytes(1, width)
    args = [b, width, b, width, C.F32, None, C.F32, b, b, 1, width, b, width, b, None, b, need, None]
    assert L.concord_layernorm_bwd(*args) == C.EINVAL
