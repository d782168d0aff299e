"""Gradients of norms and rotation asked for one by one: what a frozen query or key leaves."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_block_operators import BF16, F32, U, _close, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,heads,kv,dim", [(0, 2, 1, 64), (1, 3, 1, 8), (300, 6, 3, 64), (5000, 8, 2, 80)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_gradient_at_a_time(tokens, heads, kv, dim, dtype):
    import concord_amd as ca
    g = _gen("frozen", tokens, heads, kv, dim, dtype)
    t = {"q": torch.randn(tokens, heads, dim, generator=g, device=DEV).to(dtype),
         "k": torch.randn(tokens, kv, dim, generator=g, device=DEV).to(dtype),
         "wq": 1 + 0.3 * torch.randn(dim, generator=g, device=DEV), "wk": 1 + 0.3 * torch.randn(dim, generator=g, device=DEV)}
    up = [torch.randn(t[n].shape, generator=g, device=DEV).to(dtype) for n in ("q", "k")]

    def grads(names):
        leaves = {n: v.detach().requires_grad_(n in names) for n, v in t.items()}
        y = ca.qk_norm_rope(leaves["q"], leaves["k"], leaves["wq"], leaves["wk"])
        used = [i for i in range(2) if y[i].requires_grad]
        return dict(zip(names, torch.autograd.grad([y[i] for i in used], [leaves[n] for n in names], [up[i] for i in used])))
    want = grads(("q", "k", "wq", "wk"))
    for names in (("q",), ("k",), ("wq",), ("wk",), ("q", "wq"), ("k", "wk"), ("q", "wk")):
        got = grads(names)
        for n in names:
            if n in "qk":
                assert torch.equal(got[n], want[n]), (names, n)
            elif tokens:
                # another launch shape may add the rows up in another order: rows u of the sum of magnitudes
                x, dy = (t["q"], up[0]) if n == "wq" else (t["k"], up[1])
                h = x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
                # (a turned element is at most |a| + |b|)
                size = (2 ** 0.5 * h.abs() * dy.double().norm(dim=-1, keepdim=True)).sum((0, 1))
                _close(got[n], want[n].double(), 2 * (32 + x.numel() // dim) * U * size, F32, n)
            else:
                assert not got[n].any()
