"""The distillation example: layer norm, attention over packed documents, the
packed linears and the loss in one training step, against the same step with
torch's own operators, and over some steps."""
import math

import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu


def _plain_attention(q, k, v, starts):
    """fp32, one document at a time"""
    out = []
    rep = q.shape[1] // k.shape[1]
    s = starts.tolist()
    for a, b in zip(s, s[1:]):
        qa = q[a:b].float().transpose(0, 1)
        ka, va = (t[a:b].float().transpose(0, 1).repeat_interleave(rep, 0) for t in (k, v))
        z = torch.matmul(qa, ka.transpose(1, 2).contiguous()) / math.sqrt(q.shape[2])
        z = z.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        out.append(torch.matmul(torch.softmax(z, -1), va).transpose(0, 1))
    return torch.cat(out).to(torch.bfloat16)


def test_a_step_equals_one_of_plain_operators(monkeypatch):
    """Loss and the gradients of norms and embeddings.  Both runs round activations
    to bf16 at the same places; the operators round out to bf16 once more or
    less, 2^-8 relatively at each of 8 places: 2^-5 of a gradient's norm."""
    import concord_amd as ca
    from examples import distill_gpt as ex

    def step():
        torch.manual_seed(3)
        m = ex.GPT(layers=2, device=DEV, lr=0.0)
        gen = torch.Generator().manual_seed(4)
        batch = ex.documents(1000, 65, 256, gen, DEV)
        t = (3 * torch.randn(1000, 16, generator=gen)).to(DEV)
        i = torch.stack([torch.randperm(65, generator=gen)[:16] for _ in range(1000)]).to(DEV)
        loss = ca.distill_loss(m(*batch), t, i, temperature=2.0).mean()
        loss.backward()
        return float(loss.detach()), {n: p.grad.double().cpu() for n, p in m.named_parameters() if p.grad is not None}
    got, grads = step()

    def plain_loss(z, t, i, temperature=1.0):
        logq = torch.log_softmax(z.float() / temperature, -1)
        p = torch.softmax(t / temperature, -1)
        return temperature ** 2 * (p * (torch.log_softmax(t / temperature, -1) - logq.gather(1, i))).sum(-1)
    monkeypatch.setattr(ca, "attention", lambda q, k, v, starts: _plain_attention(q, k, v, starts))
    monkeypatch.setattr(ca, "distill_loss", plain_loss)
    monkeypatch.setattr(ca.LayerNorm, "forward", lambda self, x: torch.nn.functional.layer_norm(
        x, (x.shape[-1],), self.weight, self.bias, self.eps))
    want, ref = step()
    assert abs(got - want) <= 2.0 ** -8 * abs(want), (got, want)
    assert grads.keys() == ref.keys() and len(ref) >= 12
    for n in ref:
        assert float((grads[n] - ref[n]).norm()) <= 2.0 ** -5 * float(ref[n].norm()) + 1e-12, n


def test_the_student_learns():
    from examples import distill_gpt as ex
    losses = ex.train(60, tokens=4096, device=DEV)
    print("distillation loss:", " ".join(f"{v:.3f}" for v in losses[::10]))
    assert all(math.isfinite(v) for v in losses)
    assert sum(losses[-10:]) / 10 < 0.7 * losses[0]
