"""Training steps of the attention operators captured in a graph: every replay, on new features and
lengths, gives what the eager calls give."""
import pytest
import torch

from spira_amd.nn import functional as F
from test_gpu_attention import DTYPES, randn

pytestmark = pytest.mark.gpu


def replays(step, inputs, fresh, times=4):
    """step(leaves): outputs and gradients; fresh(i): new values of the inputs, in place."""
    leaves = [t.requires_grad_(True) for t in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
    for i in range(times):
        with torch.no_grad():
            fresh(i)
        graph.replay()
        got = [t.clone() for t in out]
        ref = step([t.detach().requires_grad_(True) for t in inputs])
        for j, (a, b) in enumerate(zip(got, ref)):
            assert torch.equal(a, b), (i, j)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,heads,kv", [(300, 4, 2), (1100, 48, 24)])
def test_attention(dev, n, heads, kv, dtype):
    dt, d = DTYPES[dtype], 32
    q, k, v, g = (randn((n, h, d), dt, i).to(dev) for i, h in enumerate((heads, kv, kv, heads)))
    offsets = torch.tensor([0, n // 3, n], dtype=torch.int32, device=dev)
    counts = torch.tensor([n // 3, n - n // 3], dtype=torch.int32, device=dev)

    def step(leaves):
        y = F.attention(*leaves, offsets, key_counts=counts, causal=True)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    def fresh(i):
        for j, t in enumerate((q, k, v, g)):
            t.copy_(randn(t.shape, dt, 10 * i + j + 20, 2.0 ** -i))
        at = n // (i + 2)
        offsets.copy_(torch.tensor([0, at, n - i]))
        counts.copy_(torch.tensor([at - 3 * i, (n - at) // (i + 1)]))
    replays(step, [q, k, v], fresh)


@pytest.mark.parametrize("dtype", DTYPES)
def test_heads(dev, dtype):
    dt, n, d = DTYPES[dtype], 500, 64
    q, k, w, u = randn((n, 4, d), dt, 1).to(dev), randn((n, 2, d), dt, 2).to(dev), randn((d,), dt, 3).to(dev), randn((d,), dt, 4).to(dev)
    g = [randn((n, h, d), dt, 5).to(dev) for h in (4, 2)]
    at = torch.arange(n, dtype=torch.int32, device=dev)

    def step(leaves):
        y = F.norm_rotate_heads(*leaves[:2], query_weight=leaves[2], key_weight=leaves[3], positions=at)
        return (*(t.detach() for t in y), *torch.autograd.grad(y, leaves, g))

    def fresh(i):
        q.copy_(randn(q.shape, dt, 30 + i)), k.copy_(randn(k.shape, dt, 40 + i)), at.add_(1000 * i)
    replays(step, [q, k, w, u], fresh)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts", [(100, 8), (20000, 64)])
def test_balance(dev, tokens, experts, dtype):
    logits = randn((tokens, experts), DTYPES[dtype], 1).to(dev)

    def step(leaves):
        r = F.balance_loss(leaves[0], F.route_experts(leaves[0].detach(), 2))
        return (r.loss.detach(), r.counts, r.probabilities, *torch.autograd.grad(r.loss, leaves))

    def fresh(i):
        logits.copy_(randn(logits.shape, DTYPES[dtype], 50 + i))
    replays(step, [logits], fresh)
