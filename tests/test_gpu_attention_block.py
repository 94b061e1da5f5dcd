"""The attention block on voxel features, alone, behind a sparse convolution and in
front of the mixture-of-experts block: outputs and gradients against the same
formulas in 64 bits, training and inference, and capture in a graph."""
import copy
import math

import pytest
import torch

from spira_amd import SparseTensor, scenes, set_kernel_map_cache
from spira_amd import nn as spnn
from spira_amd.nn import functional as F

pytestmark = pytest.mark.gpu


def scene(dev, channels, dtype, n=900, ordered=True):
    coords = torch.from_numpy(scenes.spheres_planes(n=n, grid=30, seed=1)).to(dev)
    g = torch.Generator().manual_seed(0)
    x = SparseTensor(coords, torch.randn(len(coords), channels, generator=g).to(dtype).to(dev), double=True)
    return x.order() if ordered else x


def norm(v, w, eps):
    return v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + eps) * w


def attention_reference(block, x, positions, lengths, params):
    """The block in 64 bits."""
    h, k, d = block.heads, block.kv_heads, block.head_channels
    p = (norm(x, params["entry"], block.eps) @ params["project"]).view(-1, h + 2 * k, d)
    q, keys, v = norm(p[:, :h], params["query_norm"], block.eps), norm(p[:, h:h + k], params["key_norm"], block.eps), p[:, h + k:]
    if block.rotate:
        pairs, turn = d // 2, []
        for a in range(3):
            lo, hi = a * pairs // 3, (a + 1) * pairs // 3
            turn += [positions[:, a].double() * block.base ** (-j / (hi - lo)) for j in range(hi - lo)]
        t = torch.stack(turn, 1)[:, None]
        q, keys = (torch.cat([u[..., :pairs] * t.cos() - u[..., pairs:] * t.sin(),
                              u[..., :pairs] * t.sin() + u[..., pairs:] * t.cos()], -1) for u in (q, keys))
    parts, at = [], 0
    for n in lengths:
        rows = slice(at, at + n)
        at += n
        heads = []
        for j in range(h):
            s = q[rows, j] @ keys[rows, j * k // h].t().contiguous() * d ** -0.5
            if block.causal:
                s = s.masked_fill(torch.ones_like(s).triu(1).bool(), -math.inf)
            heads.append(torch.softmax(s, 1) @ v[rows, j * k // h])
        parts.append(torch.cat(heads, 1))
    y = torch.cat(parts) @ params["out"]
    return x + block.scale * params["gate"] * norm(y, params["exit"], block.eps)


def doubles(block):
    return {k: v.detach().double().requires_grad_(True) for k, v in block.named_parameters()}


def far(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


def perturbed(block):
    """Norm weights and gates away from their start."""
    g = torch.Generator().manual_seed(3)
    for name, p in block.named_parameters():
        if p.dim() == 1:
            p.data += 0.2 * torch.randn(p.shape, generator=g).to(p)
    return block


CASES = [
    # heads, key heads, channels of a head, window, causal, rotate, ordered
    (4, 2, 12, None, False, True, True), (3, 3, 16, 128, False, True, True), (6, 2, 8, 100, True, False, True),
    (2, 1, 24, 64, True, True, False)]


@pytest.mark.parametrize("heads,kv,d,window,causal,rotate,ordered", CASES)
def test_training_step_fp32(dev, heads, kv, d, window, causal, rotate, ordered):
    """Outputs and all gradients: six products and norms in fp32, each to about 1e-6 of its result."""
    torch.manual_seed(0)
    block = perturbed(spnn.AttentionBlock(48, heads, kv, head_channels=d, window=window, causal=causal, rotate=rotate,
                                          scale=0.5).to(dev))
    x = scene(dev, 48, torch.float32, ordered=ordered)
    n = len(x.features)
    x._features.requires_grad_(True)
    y = block(x)
    assert torch.equal(y.coordinates, x.coordinates) and y.stride == x.stride
    positions = F.unflatten(x.coordinates) if ordered else x.coordinates
    lengths = [n] if window is None else [window] * (n // window) + [n % window] * (n % window > 0)
    leaf, params = x.features.detach().double().requires_grad_(True), doubles(block)
    ref = attention_reference(block, leaf, positions, lengths, params)
    assert far(y.features, ref) < 2e-5
    g = torch.randn(ref.shape, generator=torch.Generator().manual_seed(1)).to(dev)
    y.features.backward(g)
    (ref * g.double()).sum().backward()
    assert far(x.features.grad, leaf.grad) < 5e-5
    for name, p in block.named_parameters():
        assert far(p.grad, params[name].grad) < 5e-5, name


def test_scenes_do_not_see_each_other(dev):
    """Scenes behind each other with their offsets give what each gives alone."""
    torch.manual_seed(1)
    block = perturbed(spnn.AttentionBlock(32, 4, 2).to(dev)).eval()
    x = scene(dev, 32, torch.float32)
    n, cut = len(x.features), 333
    offsets = torch.tensor([0, cut, cut, n], dtype=torch.int32, device=dev)
    with torch.no_grad():
        whole = block(x, offsets).features
        for lo, hi in ((0, cut), (cut, n)):
            part = SparseTensor(x.coordinates[lo:hi], x.features[lo:hi])
            assert far(block(part).features, whole[lo:hi].double()) < 1e-5
        empty = block(SparseTensor(x.coordinates[:0], x.features[:0]))
        assert empty.features.shape == (0, 32)


@pytest.mark.parametrize("dtype,limit", [(torch.float16, 4e-3), (torch.bfloat16, 3e-2)])
def test_a_run_of_blocks(dev, dtype, limit):
    """A convolution, attention and experts as a network has them, inference in 16 bits: some ten
    roundings on the way of two updates, a fraction of the residual's size each."""
    torch.manual_seed(2)
    conv = spnn.SparseConv(16, 64, 3).to(dev).half()
    set_kernel_map_cache(conv, spnn.KernelMapCache())
    x = scene(dev, 16, torch.float16)
    with torch.no_grad():
        h = conv(x).to(dtype)
        attend = perturbed(spnn.AttentionBlock(64, 4, 2, window=256).to(dev).to(dtype)).eval()
        experts = spnn.ExpertBlock(64, 128, 8, 2).to(dev).to(dtype).eval()
        middle = attend(h)
        y, balance = experts(middle, balance=True)
        assert torch.equal(y.features, experts(middle).features)
        n = len(h.features)
        ref = attention_reference(attend, h.features.double(), F.unflatten(h.coordinates),
                                  [256] * (n // 256) + [n % 256] * (n % 256 > 0), doubles(attend))
        assert far(middle.features, ref) < limit
        assert balance.counts.sum() == 2 * n and 1 - 1e-3 <= balance.loss.item() <= 8
    assert y.features.dtype == dtype and y.stride == h.stride


def test_training_of_the_run(dev):
    """A step through both blocks: the balance loss reaches the router and, through the norm, the
    attention block; without it the gradients are the output's alone."""
    torch.manual_seed(3)
    attend = perturbed(spnn.AttentionBlock(32, 4, 2, window=200).to(dev))
    experts = spnn.ExpertBlock(32, 64, 4, 1).to(dev)
    x = scene(dev, 32, torch.float32)
    g = torch.randn(x.features.shape, generator=torch.Generator().manual_seed(1)).to(dev)

    def grads(weight):
        for p in [*attend.parameters(), *experts.parameters()]:
            p.grad = None
        y, balance = experts(attend(x), balance=True)
        ((y.features * g).sum() + weight * balance.loss).backward()
        return {k: p.grad.clone() for m in (attend, experts) for k, p in m.named_parameters(prefix=type(m).__name__)}
    plain, with_loss = grads(0.0), grads(50.0)
    assert torch.equal(plain["ExpertBlock.up"], with_loss["ExpertBlock.up"])
    # the router's own part against 64 bits: the loss's gradient alone (the rest is the same to rounding)
    middle = attend(x).features.detach().double()
    router = experts.router.detach().double().requires_grad_(True)
    logits = norm(middle, experts.entry.detach().double(), experts.eps) @ router
    chosen = F.route_experts(logits.detach().float(), 1)
    share = chosen.offsets.diff().double() / len(middle)
    (50.0 * 4 * (share * torch.softmax(logits, 1).mean(0)).sum()).backward()
    assert far(with_loss["ExpertBlock.router"] - plain["ExpertBlock.router"], router.grad) < 1e-3
    assert not torch.equal(plain["AttentionBlock.project"], with_loss["AttentionBlock.project"])


def test_captured_in_a_graph(dev):
    """Every replay on new features equals the eager call."""
    torch.manual_seed(4)
    block = spnn.AttentionBlock(48, 6, 3, window=128).to(dev).half().eval()
    x = scene(dev, 48, torch.float16)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block(x)
        for i in range(4):
            x.features.copy_(torch.randn(x.features.shape, generator=torch.Generator().manual_seed(10 + i)).half())
            graph.replay()
            got = y.features.clone()
            assert torch.equal(got, block(x).features), i
            torch.cuda.synchronize()


def test_checkpoint_and_copies(dev):
    """Recomputed in the backward pass, and copied: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(5)
    block = spnn.AttentionBlock(32, 2, window=100).to(dev)
    x = scene(dev, 32, torch.float32)

    def grads(b, call):
        b.zero_grad()
        call(b).sum().backward()
        return [p.grad.clone() for p in b.parameters()]
    plain = grads(block, lambda b: b(x).features)
    again = grads(copy.deepcopy(block), lambda b: checkpoint(lambda f: b(SparseTensor(x.coordinates, f)).features,
                                                             x.features, use_reentrant=False))
    for a, b in zip(plain, again):
        assert torch.equal(a, b)


def test_refusals(dev):
    for kw, text in ((dict(heads=3, kv_heads=2), "multiple"), (dict(heads=0), "multiple"), (dict(heads=16), "even"),
                     (dict(heads=4, head_channels=7), "even"), (dict(heads=4, head_channels=130), "128"),
                     (dict(heads=4, window=0), "window")):
        with pytest.raises(RuntimeError, match=r"\[Spira\].*" + text):
            spnn.AttentionBlock(64, **kw)
    block = spnn.AttentionBlock(32, 4).to(dev)
    with pytest.raises(RuntimeError, match="Int"):
        block(scene(dev, 32, torch.float32, 50), torch.tensor([0, 50], device=dev))
