"""What the operators' backwards hand to their kernels where a saved-tensor hook
gives the saved tensors back in another layout (offloading to the host does, for
every view that is not dense; recomputation may).

On the CPU: the nodes of csrc/torch_ops.cpp are compiled over C entries that
record their operands (operators_stub.cpp).  Each operand has to hold the values
that it holds without a hook, whatever the layout that comes back; it comes back
inside a larger buffer of NaN, so that a wrong stride reads those.

The same module shows what the nodes do with the tangents of forward mode."""
import importlib.util
import os
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="session")
def stub(tmp_path_factory):
    from concord_amd import build as B
    out = str(tmp_path_factory.mktemp("stub") / "concord_operators_stub.so")
    cflags, libs = B._ops_flags()
    cflags = ["-O0" if f == "-O2" else f for f in cflags if "TORCH_EXTENSION_NAME" not in f]
    libs = [f for f in libs if f != "-lconcord_amd"] + ["-Wl,-rpath," + os.path.join(os.path.dirname(torch.__file__), "lib")]
    r = subprocess.run([B.CXX] + cflags + ["-DTORCH_EXTENSION_NAME=concord_torch_ops", "-shared", "-o", out,
                                           os.path.join(HERE, "operators_stub.cpp")] + libs, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    spec = importlib.util.spec_from_file_location("concord_operators_stub", out)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _inside(shape, strides, offset, t):
    """t in a buffer of its own with these strides, which no stride of the original's can leave."""
    size = offset + sum((n - 1) * s for n, s in zip(shape, strides)) + 1 if t.numel() else 1
    fill = float("nan") if t.is_floating_point() else 77
    buf = torch.full((size + 64 * max(t.numel(), 64),), fill, dtype=t.dtype)
    return buf.as_strided(shape, strides, offset).copy_(t)


def _strides(order, shape, gap):
    """strides of `shape` with the dimensions of `order` from the outermost in, elements `gap` apart"""
    s, n = [0] * len(shape), gap
    for d in reversed(order):
        s[d] = n
        n *= max(shape[d], 1)
    return s


def relaid(layout, t):
    t = t.detach()
    dims = list(range(t.dim()))
    if layout == "dense":
        return _inside(t.shape, _strides(dims, t.shape, 1), 0, t)
    if layout == "shifted":   # as a slice of one flat buffer of all offloaded tensors
        return _inside(t.shape, _strides(dims, t.shape, 1), 1, t)
    if layout == "gaps":
        return _inside(t.shape, _strides(dims, t.shape, 3), 0, t)
    return _inside(t.shape, _strides(dims[::-1], t.shape, 1), 0, t)   # "reversed"


LAYOUTS = ["dense", "shifted", "gaps", "reversed"]


def _grads(stub, make, layout):
    """operands of the backward of make() -> (result, leaves, upstream)"""
    if layout is None:
        y, leaves, up = make()
    else:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: relaid(layout, t)):
            y, leaves, up = make()
    stub.recorded()
    grads = torch.autograd.grad(y, leaves, up)
    assert all(g.shape == p.shape for g, p in zip(grads, leaves))
    seen, misaligned = stub.recorded()
    assert not misaligned, misaligned
    return dict(seen)


def _same(stub, make, layout, names):
    want, got = _grads(stub, make, None), _grads(stub, make, layout)
    assert set(names) <= want.keys() and want.keys() == got.keys()
    for n in want:
        assert torch.equal(got[n], want[n]), n


def _randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("view", ["columns", "whole", "three", "copied"])
def test_layer_norm(stub, layout, view):
    def make():
        if view == "columns":
            x = _randn(6, 40)[:, 8:32]
        elif view == "three":
            x = _randn(2, 3, 40)[..., 8:32]
        elif view == "copied":
            x = _randn(24, 6).t()
        else:
            x = _randn(6, 24)
        x = x.detach().requires_grad_(True)
        w, b = (_randn(24, seed=s).requires_grad_(True) for s in (1, 2))
        return stub.layer_norm(x, w, b, 1e-5), (x, w, b), _randn(*x.shape, seed=3)
    _same(stub, make, layout, ["x", "dy", "weight", "mean", "rstd"])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("form", ["split", "head_major", "dense", "dense_split", "tables"])
def test_attention(stub, layout, form):
    def make():
        n, h, hk, d = 12, 4, 2, 8
        bf = torch.bfloat16
        starts = torch.tensor([0, 5, 12], dtype=torch.int32)
        k_starts = None
        if form in ("split", "dense_split"):
            q, k, v = _randn(n, h + 2 * hk + 2, d, dtype=bf)[:, :-2].split([h, hk, hk], dim=1)
        elif form == "head_major":
            q, k, v = (_randn(m, n, d, dtype=bf, seed=m).transpose(0, 1) for m in (h, hk, hk))
        else:
            q, k, v = (_randn(n, m, d, dtype=bf, seed=m) for m in (h, hk, hk))
        if form.startswith("dense"):
            q, k, v = (t.unflatten(0, (3, 4)) for t in (q, k, v))
            starts = None
        if form == "tables":
            k_starts = torch.tensor([0, 3, 12], dtype=torch.int32)
        p = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return (stub.attention(*p, starts, k_starts, True, None), p,
                _randn(*q.shape, dtype=bf, seed=9))
    _same(stub, make, layout, ["q", "k", "v", "out", "dout", "lse", "out_low"] +
          ([] if form.startswith("dense") else ["starts"]))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("view", ["columns", "whole", "three"])
def test_distill_loss(stub, layout, view):
    def make():
        rows = (2, 3) if view == "three" else (6,)
        z = _randn(*rows, 40)
        z = (z if view == "whole" else z[..., :33]).detach().requires_grad_(True)
        t = _randn(*rows, 12, seed=1)[..., :8]
        i = torch.arange(6 * 12).view(*rows, 12)[..., 2:10]
        return stub.distill_loss(z, t, i, 2.0), (z,), _randn(*rows, seed=4)
    _same(stub, make, layout, ["logits", "teacher", "index", "stats", "dloss"])


@pytest.mark.parametrize("other", ["type", "extent"])
def test_another_tensor_is_refused(stub, other):
    """A hook that gives back another type or fewer elements: an error, and nothing is launched."""
    def change(t):
        if other == "type":
            return t.to({torch.float32: torch.bfloat16}.get(t.dtype, torch.float32))
        return t.reshape(-1)[:max(t.numel() - 8, 0)]
    x = _randn(6, 24).requires_grad_(True)
    q = _randn(6, 2, 8, dtype=torch.bfloat16).requires_grad_(True)
    calls = [lambda: stub.layer_norm(x, None, None, 1e-5), lambda: stub.attention(q, q, q, None, None, True, None),
             lambda: stub.distill_loss(x, _randn(6, 4), torch.zeros(6, 4, dtype=torch.int64), 1.0)]
    stub.recorded()
    for call in calls:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = call()
        with pytest.raises((RuntimeError, TypeError, ValueError), match="came back|must be|attention"):
            y.sum().backward()
    assert not stub.recorded()[0]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("enabled", [True, False])
def test_forward_mode_is_refused(stub, requires_grad, enabled):
    """A tangent on any differentiable input is an error, in no_grad too (which
    leaves forward mode on); with forward mode off there is nothing to drop."""
    import torch.autograd.forward_ad as fw

    def inputs(args, dual):
        args = [a.detach().clone().requires_grad_(requires_grad) for a in args]
        args[dual] = fw.make_dual(args[dual], torch.ones_like(args[dual]))
        assert fw.unpack_dual(args[dual]).tangent is not None
        return args
    x, w = _randn(6, 24), _randn(24)
    q = _randn(6, 2, 8, dtype=torch.bfloat16)
    ops = [(stub.layer_norm, [x, w, w], (1e-5,)), (stub.attention, [q, q, q], (None, None, True, None)),
           (stub.distill_loss, [x], (_randn(6, 4), torch.zeros(6, 4, dtype=torch.int64), 1.0))]
    with fw.dual_level():
        for op, args, rest in ops:
            for dual in range(len(args)):
                given = inputs(args, dual)
                if enabled:
                    for mode in (torch.enable_grad, torch.no_grad):
                        with mode(), pytest.raises(RuntimeError, match="forward mode"):
                            op(*given, *rest)
                else:
                    with fw._set_fwd_grad_enabled(False):
                        op(*given, *rest)


# ---- on the GPU: the kernels themselves --------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["offloaded", "reversed"])
def test_gradients_under_a_hook(layout):
    """The same gradients, bit for bit, with the saved tensors offloaded to the host
    or given back in another layout, each operator on views that are not dense."""
    import concord_amd as ca

    dev = "cuda:0"
    x0 = _randn(70, 300).to(dev)
    qkv = _randn(200, 10, 64, dtype=torch.bfloat16).to(dev)
    t, i = _randn(70, 12, seed=1).to(dev)[:, :8], torch.arange(70 * 12, device=dev).view(70, 12)[:, 2:10] % 65
    starts = torch.tensor([0, 3, 130, 200], dtype=torch.int32, device=dev)

    def norm():
        x = x0[:, 8:264].detach().requires_grad_(True)
        w, b = (_randn(256, seed=s).to(dev).requires_grad_(True) for s in (2, 3))
        return ca.layer_norm(x, w, b), (x, w, b)

    def attn():
        p = [t.detach().requires_grad_(True) for t in qkv[:, :8].split([4, 2, 2], dim=1)]
        return ca.attention(*p, starts=starts), p

    def dense():
        p = [t.detach().requires_grad_(True) for t in qkv[:, :8].unflatten(0, (2, 100)).split([4, 2, 2], dim=2)]
        return ca.attention(*p, causal=False), p

    def distill(vocab):
        z = (x0 if vocab == 65 else _randn(70, 3000).to(dev))[:, 3:3 + vocab].detach().requires_grad_(True)
        return ca.distill_loss(z, t, i, 2.0), (z,)

    hooks = torch.autograd.graph.save_on_cpu() if layout == "offloaded" else \
        torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: relaid("reversed", t.cpu()).to(dev))
    for make in (norm, attn, dense, lambda: distill(65), lambda: distill(2049)):
        y, leaves = make()
        up = _randn(*y.shape, seed=5).to(y.dtype).to(dev)
        want = torch.autograd.grad(y, leaves, up)
        with hooks:
            y, leaves = make()
        assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, leaves, up)))
