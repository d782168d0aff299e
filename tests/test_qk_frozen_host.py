"""The backward of norms and rotation reads and writes what was asked for: a frozen query or
key is left out of the launch.  Over C entries that launch nothing and record their operands."""
import pytest
import torch

from test_block_operators_host import BF16, _randn, stub  # noqa: F401


def _names(stub, leaves, up=(0, 1), frozen=()):  # noqa: F811
    """operands that the kernel was given for the gradients of `leaves`"""
    t = {"q": _randn(7, 4, 24, dtype=BF16), "k": _randn(7, 2, 24, dtype=BF16, seed=1), "wq": _randn(24, seed=2),
         "wk": _randn(24, seed=3)}
    for n in t:
        t[n].requires_grad_(n not in frozen)
    y = stub.qk_norm_rope(t["q"], t["k"], t["wq"], t["wk"], torch.arange(7), 1e4, 16, False, 1e-6)
    stub.recorded()
    grads = torch.autograd.grad([y[i] for i in up], [t[n] for n in leaves], [torch.ones_like(y[i]) for i in up])
    assert [(g.shape, g.dtype) for g in grads] == [(t[n].shape, t[n].dtype) for n in leaves]
    seen, misaligned = stub.recorded()
    assert not misaligned
    return {n for n, _ in seen} - {"positions", "settings"}


Q, K = {"q", "dq_out", "q_weight"}, {"k", "dk_out", "k_weight"}


@pytest.mark.parametrize("leaves,want", [
    (("q", "k", "wq", "wk"), Q | K), (("q",), Q), (("k",), K), (("wq",), Q), (("wk",), K), (("q", "wk"), Q | K),
    (("k", "wk"), K), (("q", "wq"), Q)])
def test_only_what_is_asked_for(stub, leaves, want):  # noqa: F811
    assert _names(stub, leaves) == want


@pytest.mark.parametrize("frozen,leaves,want", [(("k", "wk"), ("q", "wq"), Q), (("q", "wq"), ("k", "wk"), K),
                                                (("k",), ("q", "wk"), Q | K), (("wq", "wk"), ("k",), K)])
def test_frozen_ones_are_left_out(stub, frozen, leaves, want):  # noqa: F811
    assert _names(stub, leaves, frozen=frozen) == want


def test_a_result_that_nothing_used_has_a_gradient_of_zeros(stub):  # noqa: F811
    assert _names(stub, ("q", "k"), up=(0,)) == Q | K


def test_without_weights(stub):  # noqa: F811
    q, k = _randn(7, 4, 24), _randn(7, 2, 24).requires_grad_(True)
    y = stub.qk_norm_rope(q, k, None, None, None, 1e4, 16, False, 1e-6)
    stub.recorded()
    torch.autograd.grad(y[1], k, torch.ones_like(y[1]))
    assert {n for n, _ in stub.recorded()[0]} == {"k", "dk_out", "settings"}
