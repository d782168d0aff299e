"""The embedding's gradient of millions of tokens: a sort of hundreds of blocks and more, whose
counts a kernel of its own sums up, and the sizes at its border."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_block_operators import BF16, F32, _gen

pytestmark = pytest.mark.gpu
BORDER = 256 * 4096


@pytest.mark.parametrize("n", [BORDER, BORDER + 1, 3 * BORDER + 12345])
@pytest.mark.parametrize("vocab,width,dtype", [(3, 1, F32), (511, 8, BF16), (70000, 3, F32)])
def test_gradient_of_millions_of_tokens(n, vocab, width, dtype):
    """Whole numbers, whose sums (4 n < 2^24) are exact in fp32 in any order."""
    import concord_amd as ca
    g = _gen("many tokens", n, vocab)
    # some tokens far commoner than the rest, some outside the table
    tokens = (torch.rand(n, generator=g, device=DEV) ** 3 * (vocab + 1)).long()
    tokens[::11] = -1
    w = torch.randn(vocab, width, generator=g, device=DEV).to(dtype).requires_grad_(True)
    dy = torch.randint(-4, 5, (n, width), generator=g, device=DEV).to(dtype)
    y = ca.embedding(tokens, w)
    dw, = torch.autograd.grad(y, (w,), dy)
    key = torch.where((tokens >= 0) & (tokens < vocab), tokens, vocab)
    key, order = key.sort(stable=True)
    sums = torch.cat((torch.zeros(1, width, device=DEV, dtype=torch.float64), dy[order].double().cumsum(0)))
    ends = torch.searchsorted(key, torch.arange(vocab + 1, device=DEV))   # where each token's pairs begin
    assert torch.equal(dw, (sums[ends[1:]] - sums[ends[:-1]]).to(dtype))
    table = torch.cat((w.detach(), torch.zeros(1, width, device=DEV, dtype=dtype)))
    inside = torch.where((tokens >= 0) & (tokens < vocab), tokens, vocab)
    assert torch.equal(y.detach(), table[inside])


def test_many_tokens_in_order_and_all_alike():
    """Sums that are whole numbers, so any mistake of place shows: the token's own count."""
    import concord_amd as ca
    n, vocab = 2 * BORDER + 77, 1000
    w = torch.zeros(vocab, 4, device=DEV, requires_grad=True)
    for tokens in (torch.arange(n, device=DEV) % vocab, torch.full((n,), vocab - 1, device=DEV),
                   torch.arange(n, device=DEV) // (n // vocab + 1)):
        dw, = torch.autograd.grad(ca.embedding(tokens, w).sum(), (w,))
        assert torch.equal(dw, torch.bincount(tokens, minlength=vocab).float()[:, None].expand(vocab, 4))


def test_many_tokens_in_a_graph():
    import concord_amd as ca
    g = _gen("many tokens graph")
    n, vocab = BORDER + 4097, 5000
    tokens = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    w = torch.randn(vocab, 8, generator=g, device=DEV, requires_grad=True)
    dy = torch.randn(n, 8, generator=g, device=DEV)

    def step():
        return torch.autograd.grad(ca.embedding(tokens, w), (w,), dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        tokens.copy_(torch.randint(-3, vocab + 3, (n,), generator=g, device=DEV))
        graph.replay()
        got = held.clone()
        assert torch.equal(got, step())
