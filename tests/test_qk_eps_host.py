"""eps of norms with rotation, as the kernels hold it, in 32 bits: what is infinite or lost there is refused."""
import ctypes

import pytest
import torch

from test_block_operators_host import L, _qk_args  # noqa: F401


@pytest.mark.parametrize("eps", [1e39, 1e300, 1e-46, 5e-324])
def test_eps_that_32_bits_do_not_hold(eps):
    import concord_amd as ca
    q = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="qk_norm_rope: eps"):
        ca.qk_norm_rope(q, q, eps=eps)


@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-38, 3e38])
def test_eps_that_they_hold(eps):
    import concord_amd as ca
    q = torch.zeros(3, 2, 64)
    with pytest.raises(RuntimeError, match="ROCm device"):   # past the checks of values
        ca.qk_norm_rope(q, q, eps=eps)


def test_an_infinite_eps_of_the_entries(L):  # noqa: F811
    from concord_amd import _lib as C
    buf = ctypes.create_string_buffer(64)
    for eps in (float("inf"), float("nan")):
        a = _qk_args(buf, eps=eps, T=0)
        assert L.concord_qk_norm_rope_fwd(ctypes.byref(a), None) == C.EINVAL
        assert L.concord_qk_norm_rope_bwd(ctypes.byref(a), None, 0, None) == C.EINVAL
