"""When a packed linear lays its input down in 8 bits: for a backward, and only then.  On
the CPU, the product and the packing replaced by stand-ins that count."""
import pytest
import torch

from concord_amd import packed_b as pb


@pytest.fixture
def layer(monkeypatch):
    m = pb.ConcordLinearPackedB.__new__(pb.ConcordLinearPackedB)   # (its own __init__ wants a GPU)
    torch.nn.Module.__init__(m)
    for name in ("lr", "eps"):
        m.register_buffer(f"_{name}_buf", torch.ones(1))
    m.packed_w, m.row_exp, m.col_exp = torch.zeros(32, 64, dtype=torch.int32), torch.zeros(32), torch.zeros(64)
    m.bias = torch.nn.Parameter(torch.zeros(32, dtype=torch.bfloat16))
    m.alpha, m.beta1, m.optimizer_kind, m.drive, m.fast_gain = 0.1, 0.0, "adamw", "vhat", 1.0
    m.weight_decay = m.step_cap = m.v_scale = m.precond_p = m.gf_consol = m.drift_cancel_C = m.alpha_v_fast = 0.0
    m.wd_sv = m.wd_sf = m.adafactor_beta2 = m.gf_trust_delta_sq = 0.0
    m.mass_preserve_v = m.apply_chase = m.track_rebalance = m.track_adafactor_v = True
    m.v_row = m.v_col = m._sum_v_inv = m._coh_pre = None
    m.weight_cache, m.packed_calls = False, []

    def pack8(x):
        m.packed_calls.append(tuple(x.shape))
        return torch.zeros(x.shape, dtype=torch.int8), torch.zeros(x.shape[0], 2, dtype=torch.uint8)
    monkeypatch.setattr(pb, "pack8", pack8)
    monkeypatch.setattr(pb, "_gemm_fwd", lambda x2, w, *a: torch.zeros(x2.shape[0], w.shape[0], dtype=torch.bfloat16))
    m.set_input_bits(8)
    assert m.bias.requires_grad
    return m


def test_packed_once_for_a_backward(layer):
    assert layer(torch.zeros(3, 64)).requires_grad
    layer(torch.zeros(2, 5, 64, requires_grad=True))
    assert layer.packed_calls == [(3, 64), (10, 64)]


def test_not_packed_without_gradients(layer):
    for x in (torch.zeros(3, 64), torch.zeros(3, 64, requires_grad=True)):
        with torch.no_grad():
            layer(x)
        with torch.inference_mode():
            layer(x)
    layer.bias.requires_grad_(False)
    layer(torch.zeros(3, 64))
    assert layer.packed_calls == []


def test_not_packed_by_a_checkpoint_s_first_pass(layer):
    from torch.utils.checkpoint import checkpoint
    y = checkpoint(layer, torch.zeros(3, 64, requires_grad=True), use_reentrant=True)
    assert y.requires_grad and layer.packed_calls == []


def test_16_bits_pack_nothing(layer):
    layer.set_input_bits(16)
    assert layer(torch.zeros(3, 64)).requires_grad and layer.packed_calls == []
