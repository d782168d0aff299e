"""A char-level GPT of packed linears distilled from a teacher's top logits.

    python examples/distill_gpt.py --steps 200

Documents of different lengths are packed into one row of tokens, one after
another; `starts` says where each begins, so nothing is padded and no token
attends to another document.  Student and teacher are one architecture
(LayerNorm, attention and ConcordLinearPackedB).  The teacher is frozen: it hands over
its largest logits and their places, as a stored teacher's output would be.
The Concord layers step themselves in backward; the norms and embeddings are
on SGD.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import concord_amd as ca  # noqa: E402


class Block(nn.Module):
    def __init__(self, width, heads, key_heads, device, lr):
        super().__init__()
        self.heads, self.key_heads, self.dim = heads, key_heads, width // heads

        def linear(i, o):
            return ca.ConcordLinearPackedB(i, o, bias=False, device=device, lr=lr)
        self.ln1, self.ln2 = ca.LayerNorm(width, device=device), ca.LayerNorm(width, device=device)
        self.qkv = linear(width, (heads + 2 * key_heads) * self.dim)
        self.proj, self.fc, self.out = linear(width, width), linear(width, 4 * width), linear(4 * width, width)

    def forward(self, x, starts):
        h, hk = self.heads, self.key_heads
        qkv = self.qkv(self.ln1(x)).to(torch.bfloat16).view(-1, h + 2 * hk, self.dim)
        a = ca.attention(*qkv.split([h, hk, hk], dim=1), starts=starts)
        x = x + self.proj(a.reshape(x.shape))
        return x + self.out(nn.functional.gelu(self.fc(self.ln2(x))))


class GPT(nn.Module):
    def __init__(self, vocab=65, width=384, heads=6, key_heads=3, layers=4, context=256, device="cuda", lr=1e-3):
        super().__init__()
        self.wte = nn.Embedding(vocab, width, device=device)
        self.wpe = nn.Embedding(context, width, device=device)
        self.blocks = nn.ModuleList(Block(width, heads, key_heads, device, lr) for _ in range(layers))
        self.ln_f = ca.LayerNorm(width, device=device)
        self.head = ca.ConcordLinearPackedB(width, vocab, bias=False, device=device, lr=lr)

    def forward(self, tokens, positions, starts):
        x = self.wte(tokens) + self.wpe(positions)
        for b in self.blocks:
            x = b(x, starts)
        return self.head(self.ln_f(x))

    def concord_layers(self):
        return [m for m in self.modules() if isinstance(m, ca.ConcordLinearPackedB)]


def documents(tokens, vocab, context, gen, device):
    """One row of `tokens` tokens cut into documents of 1 to `context` tokens:
    (tokens, position of each in its document, starts)."""
    lens, left = [], tokens
    while left > 0:
        n = min(left, int(torch.randint(1, context + 1, (1,), generator=gen)))
        lens.append(n)
        left -= n
    starts = torch.zeros(len(lens) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(lens, dtype=torch.int32).cumsum(0)
    positions = torch.cat([torch.arange(n) for n in lens])
    # not every letter is equally likely
    letters = torch.multinomial(1.0 / (1.0 + torch.arange(vocab)), tokens, replacement=True, generator=gen)
    return letters.to(device), positions.to(device), starts.to(device)


def train(steps, tokens=8192, top=16, temperature=2.0, device="cuda", seed=0, log=None):
    """Losses (mean over tokens) of `steps` distillation steps."""
    torch.manual_seed(seed)
    vocab, context = 65, 256
    teacher, student = GPT(vocab, context=context, device=device), GPT(vocab, context=context, device=device)
    with torch.no_grad():   # a teacher with opinions: logits a few units apart
        teacher.head.load_weights(torch.randn(vocab, 384, device=device) * 0.15)
    layers = student.concord_layers()
    own = {id(p) for m in layers for p in m.parameters()}
    opt = torch.optim.SGD([p for p in student.parameters() if id(p) not in own], lr=1e-2, momentum=0.9)
    gen = torch.Generator().manual_seed(seed + 1)
    losses = []
    for step in range(steps):
        batch = documents(tokens, vocab, context, gen, device)
        with torch.no_grad():
            values, index = teacher(*batch).float().topk(top, dim=-1)
        loss = ca.distill_loss(student(*batch), values, index, temperature=temperature).mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()   # the Concord layers update themselves here
        opt.step()
        for m in layers:
            m.rebalance()
        losses.append(float(loss.detach()))
        if log and step % log == 0:
            print(f"step {step:4d}  loss {losses[-1]:.4f}", flush=True)
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--top", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=2.0)
    args = ap.parse_args()
    losses = train(args.steps, args.tokens, args.top, args.temperature, log=max(1, args.steps // 20))
    print(f"loss {losses[0]:.4f} -> {sum(losses[-10:]) / len(losses[-10:]):.4f}")


if __name__ == "__main__":
    main()
