"""Norms with rotation of rows whose squares leave 32 bits, above and below: the norm of such a
row is an ordinary number, and so are its results and gradients.  Against the formula in 64 bits."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_block_operators import BF16, F16, F32, U, _close, _gen, _qk_reference

pytestmark = pytest.mark.gpu


def _rows(n, heads, dim, dtype, exps, g):
    """rows of ordinary values times 2^e, e of exps one after another"""
    x = torch.randn(n, heads, dim, generator=g, device=DEV).to(dtype).double().clamp_(-7, 7)
    e = torch.tensor(exps, device=DEV, dtype=torch.float64)[torch.arange(n * heads, device=DEV) % len(exps)].view(n, heads, 1)
    return (x * torch.exp2(e)).to(dtype), e


@pytest.mark.parametrize("dim,adjacent", [(8, False), (64, False), (80, True), (128, False), (256, False)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("eps,exps", [(0.0, [-110, -64, -50, -45, -30, 0, 30, 58, 64, 90, 124]), (1e-6, [0, 58, 64, 90, 124, -110]),
                                      (1e-40, [-110, -66, -60, 0]), (1e30, [0, 45, 50, 64, 124])])
def test_rows_of_any_size(eps, exps, dtype, dim, adjacent):
    import concord_amd as ca
    g = _gen("range", eps, dtype, dim)
    (q, eq), (k, ek) = _rows(60, 5, dim, dtype, exps, g), _rows(60, 2, dim, dtype, exps[::-1], g)
    eps = float(torch.tensor(eps, dtype=F32))   # as the kernels hold it
    w = (1 + 0.3 * torch.randn(dim, generator=g, device=DEV)).requires_grad_(True)
    q.requires_grad_(True), k.requires_grad_(True)
    yq, yk = ca.qk_norm_rope(q, k, w, w, eps=eps, interleaved=adjacent)
    # gradients whose quotient by the row's norm fits: dy of the order of the square root of that norm
    ups = []
    for x, e in ((q, eq), (k, ek)):
        norm = torch.maximum(e, torch.full_like(e, eps).log2() / 2 if eps else e)
        ups.append((torch.randn(x.shape, generator=g, device=DEV).double() * torch.exp2((norm / 2).round())).to(dtype))
    dq, dk, dw = torch.autograd.grad((yq, yk), (q, k, w), ups)
    pos = torch.arange(60, device=DEV)
    sums = 0.0
    bound = 0.0
    for x, y, dx, up in ((q, yq, dq, ups[0]), (k, yk, dk, ups[1])):
        ry, by, rdx, bdx, rdw, bdw = _qk_reference(x.detach(), w.detach(), pos, 10000.0, dim, adjacent, eps, up)
        _close(y.detach(), ry, by, dtype, "y")
        _close(dx, rdx, bdx, dtype, "dx")
        sums, bound = sums + rdw, bound + bdw
    _close(dw, sums, bound + U * sums.abs(), F32, "dw")   # (torch adds the two parts)


def test_large_and_small_values_in_a_row():
    import concord_amd as ca
    x = torch.zeros(3, 1, 64, device=DEV)
    x[0, 0, :4] = torch.tensor([3e38, -3e38, 1e30, 1.0])
    x[1, 0, :] = torch.finfo(F32).max
    x[2, 0, :4] = torch.tensor([1e-44, -3e-42, 0.0, 1e-40])
    for eps in (0.0, 1e-45):
        y, _ = ca.qk_norm_rope(x, x, rotary_dim=0, eps=eps)
        d = x.double()
        want = d / (d.square().mean(-1, keepdim=True) + float(torch.tensor(eps))).sqrt()
        _close(y, want, 24 * U * want.abs(), F32)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_of_zeros_and_the_smallest_eps(dtype):
    import concord_amd as ca
    x = torch.zeros(5, 2, 64, device=DEV, dtype=dtype)
    for eps in (1e-45, 1e-40, 1e-38, 1e-30, 1e-6):
        y, _ = ca.qk_norm_rope(x, x, eps=eps)
        assert not y.any()
