"""The 8-bit form over every exponent that it has, and the gradients that read it, in
exact arithmetic: blocks of the largest numbers with small ones beside them."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_block_operators import BF16, F16, F32, U, _close, _gelu64, _kept, _same

pytestmark = pytest.mark.gpu
TYPES = [F32, BF16, F16]


def _blocks(dtype):
    """a row for each power of two that the type has: its largest values just there, just below
    the next one and around the 127 / 64 at which the step changes, small ones of both signs after it"""
    info = torch.finfo(dtype)
    lo, hi = {F32: (-149, 128), BF16: (-133, 128), F16: (-24, 16)}[dtype]
    rows = []
    for e in range(lo, hi):
        for m in (1.0, 1.25, 127 / 64, 127.5 / 64, 2.0):
            top = min(m * 2.0 ** e, info.max)
            v = torch.linspace(-1, 1, 32, dtype=torch.float64) * top * 0.9
            v[3], v[5], v[7], v[9] = (-top if len(rows) % 2 else top), 0.0, top * 2.0 ** -9, -top * 2.0 ** -30
            rows.append(v)
    return torch.stack(rows).to(dtype).to(DEV)


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_every_exponent(dtype, aligned):
    import concord_amd as ca
    x = _blocks(dtype)
    if not aligned:   # two whole blocks and 5 values of another, rows on no boundary
        x = torch.cat((x, x.flip(0), x[:, :5]), 1)
    codes, exps = ca.pack8(x)
    rc, re, rv = _kept(x)
    assert torch.equal(exps, re) and torch.equal(codes, rc)
    if dtype != F16:
        assert {1, 2, 247, 248, 249} <= set(exps.flatten().tolist())
    assert _same(ca.unpack8(codes, exps, dtype).double(), rv)


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_unpack_of_every_code(dtype, aligned):
    import concord_amd as ca
    most = torch.finfo(dtype).max
    codes = torch.arange(-128, 128, device=DEV).to(torch.int8).expand(249, 256)
    exps = torch.arange(1, 250, device=DEV).to(torch.uint8)[:, None].expand(249, 8)
    width = 256 if aligned else 249
    want = (codes.double() * torch.exp2(exps[:, :1].double() - 127))[:, :width].clamp(-most, most)
    # (rounded where a type's subnormals are coarser than the step)
    assert torch.equal(ca.unpack8(codes[:, :width], exps, dtype), want.to(dtype))


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_large_blocks(dtype, aligned):
    """The derivative is 1, 0 or (where the block's step swallowed the value) 1/2; bounds as for ordinary values."""
    import concord_amd as ca
    info = torch.finfo(dtype)
    tops = [info.max, info.max * 0.59, info.max / 2, info.max / 2 * 1.001, info.max / 4, 127 / 128 * 2.0 ** (128 if dtype != F16 else 16)]
    x = torch.zeros(len(tops), 64 if aligned else 39, device=DEV, dtype=dtype)
    for i, t in enumerate(tops):
        x[i, :6] = torch.tensor([t, -t, t / 3, -t / 50, 1.0, 0.0], dtype=torch.float64).to(dtype)
        x[i, 32:35] = torch.tensor([0.5, -2.0, 3.0])   # an ordinary block beside it
    x.requires_grad_(True)
    dy = torch.full_like(x, 2.0 ** -9)
    dx, = torch.autograd.grad(ca.gelu8(x), (x,), dy)
    d = dy.double()
    _, dv, _, bound = _gelu64(_kept(x.detach())[2], False, dtype)
    _close(dx, d * dv, d * (bound + U * dv.abs() + 2.0 ** -120), dtype, "dx")
    both = torch.cat((x.detach().flip(0), x.detach()), 1).requires_grad_(True)
    dg, = torch.autograd.grad(ca.geglu8(both), (both,), dy)
    w = x.shape[1]
    ka, kb = (_kept(t)[2] for t in both.detach().chunk(2, -1))
    v, dv, rel, bound = _gelu64(kb, False, dtype)
    _close(dg[:, :w], d * v, (d * v).abs() * (rel + U) + d * 2.0 ** -120, dtype, "da")
    _close(dg[:, w:], d * ka * dv, (d * ka).abs() * (bound + 2 * U * dv.abs() + 2.0 ** -120), dtype, "dg")


@pytest.mark.parametrize("tanh", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_gradient_of_a_large_half(dtype, tanh):
    """dy times the large half passes 32 bits, the whole product with a small derivative does not."""
    import concord_amd as ca
    a = torch.full((4, 64), 2.0 ** 127, device=DEV)
    g = torch.empty(4, 64, device=DEV)
    g[0], g[1], g[2], g[3] = -30.0, -9.0, -6.0, -20.0
    x = torch.cat((a, g), 1).to(dtype).requires_grad_(True)
    dy = torch.full((4, 64), 8.0, device=DEV, dtype=dtype)
    dx, = torch.autograd.grad(ca.geglu8(x, approximate="tanh" if tanh else "none"), (x,), dy)
    d = dy.double()
    ka, kb = (_kept(t)[2] for t in x.detach().chunk(2, -1))
    _, dv, _, bound = _gelu64(kb, tanh, dtype)
    _close(dx[:, 64:], d * ka * dv, (d * ka).abs() * (bound + 2 * U * dv.abs() + 2.0 ** -120), dtype, "dg")
