"""The dropout masks of ``ExpertBlock``: which call has which.  On the CPU, with
plain forms in place of the kernels; and once more with the kernels."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from spira_amd import SparseTensor
from spira_amd import nn as spnn
from spira_amd.nn import functional as F


class Dropout(torch.autograd.Function):
    """A mask made of (seed, offset), and made again for the gradient."""

    @staticmethod
    def keep(x, p, seed, offset):
        g = torch.Generator().manual_seed((seed * 1000003 + offset) % 2 ** 63)
        return torch.rand(x.shape, generator=g) >= p

    @staticmethod
    def forward(ctx, x, p, seed, offset):
        ctx.mask = p, seed, offset
        return x * Dropout.keep(x, p, seed, offset) / (1 - p)

    @staticmethod
    def backward(ctx, d):
        return d * Dropout.keep(d, *ctx.mask) / (1 - ctx.mask[0]), None, None, None


def rms_norm(x, w, eps=1e-6):
    return x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + eps) * w


def route_experts(logits, k):
    value, chosen = torch.topk(logits, k, dim=1)
    order = torch.argsort(chosen.reshape(-1), stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(len(order))
    offsets = torch.bincount(chosen.reshape(-1), minlength=logits.shape[1]).cumsum(0)
    return F.ExpertRoutes(torch.softmax(value, 1), chosen, torch.cat([offsets.new_zeros(1), offsets]), order // k,
                          slots.view(chosen.shape))


def grouped_linear(x, w, groups, *, bias, relu=False):
    offsets = groups
    if isinstance(groups, F.ExpertRoutes):
        x, offsets = x[groups.rows], groups.offsets
    y = torch.cat([x[a:b] @ w[e] + bias[e] for e, (a, b) in enumerate(zip(offsets, offsets[1:]))])
    return torch.relu(y) if relu else y


@pytest.fixture
def plain(monkeypatch):
    """The block's operators in their plain form; the masks that calls make."""
    made = []

    def dropout(x, p, seed, offset=0):
        made.append((seed, offset))
        return Dropout.apply(x, p, seed, offset)

    def gated_residual_norm(x, h, *, weight, gate, scale, eps):
        return x + scale * gate * rms_norm(h, weight, eps), None

    for f in (dropout, gated_residual_norm, rms_norm, route_experts, grouped_linear):
        monkeypatch.setattr(F, f.__name__, f)
    monkeypatch.setattr(F, "combine_experts", lambda h, r: (r.weights[:, :, None] * h[r.slots]).sum(1))
    return made


def voxels(n=50, channels=12, device="cpu"):
    x = torch.randn(n, channels, generator=torch.Generator().manual_seed(3)).to(device)
    return torch.arange(n, device=device), x.requires_grad_(True)


def step(blocks, coords, x, recompute):
    """Two passes through the blocks and one backward pass: (outputs, gradients)."""
    def whole(f):
        t = SparseTensor(coords, f)
        for b in blocks:
            t = b(t)
        return t.features

    leaves = [x] + [p for b in blocks for p in b.parameters()]
    out = []
    for scale in (1.0, 2.0):
        out.append(whole(x * scale) if recompute is None else checkpoint(whole, x * scale, use_reentrant=recompute))
    loss = sum((y * torch.linspace(-1, 2, y.numel(), device=y.device).view(y.shape)).sum() for y in out)
    for t in leaves:
        t.grad = None
    loss.backward()
    return [y.detach() for y in out], [t.grad for t in leaves]


def check_recomputation(device, recompute, **kw):
    coords, x = voxels(device=device)
    torch.manual_seed(1)
    blocks = [spnn.ExpertBlock(12, 24, 4, 2, dropout=0.5, **kw).to(device) for _ in range(2)]
    results = []
    for how in (None, recompute):
        for b in blocks:
            b.calls.zero_()
        torch.manual_seed(2)
        results.append(step(blocks, coords, x, how))
        assert [int(b.calls) for b in blocks] == [2, 2]
    for a, b in zip(*(r[0] + r[1] for r in results)):
        # (the two passes' gradients may be added in another order: two roundings of fp32)
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
    return blocks


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_calls_have_their_first_masks(plain, reentrant):
    """Outputs, gradients and the count of calls of two blocks, twice each, with activation checkpointing as without."""
    check_recomputation("cpu", reentrant, seed=5)
    first, again = plain[:4], plain[4:]
    assert again[:4] == first and sorted(again[4:]) == sorted(first)


@pytest.mark.parametrize("seed", [5, None])
def test_a_recomputation_that_cannot_be_known_is_refused(plain, seed):
    coords, x = voxels()
    block = spnn.ExpertBlock(12, 24, 4, 2, dropout=0.5, seed=seed)
    y = checkpoint(lambda f: block(SparseTensor(coords, f)).features, x, use_reentrant=False, preserve_rng_state=False)
    with pytest.raises(RuntimeError, match="repeats none"):
        y.sum().backward()


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_calls_without_a_seed(plain, reentrant):
    check_recomputation("cpu", reentrant)
    first, again = plain[:4], plain[4:]
    assert again[:4] == first and sorted(again[4:]) == sorted(first)


def test_blocks_have_masks_of_their_own(plain):
    """Without a seed: two blocks, a copy of one, and every call of each; and the same again from the same state of
    torch's generator.  With a seed: the number of the call."""
    coords, x = voxels()
    torch.manual_seed(0)
    a, b = (spnn.ExpertBlock(12, 24, 4, 2, dropout=0.5) for _ in range(2))
    blocks = [a, b, copy.deepcopy(a)]
    runs = []
    for _ in range(2):
        torch.manual_seed(9)
        del plain[:]
        for block in blocks + blocks:
            block(SparseTensor(coords, x))
        assert len(set(plain)) == 6
        runs.append(list(plain))
    assert runs[0] == runs[1] and [int(block.calls) for block in blocks] == [4, 4, 4]
    del plain[:]
    a, b = (spnn.ExpertBlock(12, 24, 4, 2, dropout=0.5, seed=s) for s in (0, 1))
    for block in (a, b, a):
        block(SparseTensor(coords, x))
    assert plain == [(0, 0), (1, 0), (0, 1)]


def test_the_count_of_calls_in_state_dicts(plain):
    """Saved and loaded with the parameters, alone and within another module; missed where it is not there."""
    coords, x = voxels()
    block = spnn.ExpertBlock(12, 24, 4, 2, dropout=0.5)
    for _ in range(3):
        block(SparseTensor(coords, x))
    saved = block.state_dict()
    assert int(saved["calls"]) == 3 and not list(block.buffers())
    for outer in (lambda b: b, lambda b: torch.nn.Sequential(torch.nn.Linear(2, 2), b)):
        state = outer(block).state_dict()
        other = spnn.ExpertBlock(12, 24, 4, 2, dropout=0.5)
        state = {k: v.clone() for k, v in state.items()}
        assert not any(outer(other).load_state_dict(state)) and int(other.calls) == 3
        assert other.double().calls.dtype == torch.int64
        (key,) = [k for k in state if k.endswith("calls")]
        del state[key]
        with pytest.raises(RuntimeError, match="calls"):
            outer(other).load_state_dict(state)
        assert outer(other).load_state_dict(state, strict=False).missing_keys == [key]


@pytest.mark.gpu
def test_data_parallel_over_rccl(dev, tmp_path):
    """A block within DistributedDataParallel, of one rank: its parameters and buffers are sent, its count is not."""
    import torch.distributed as dist

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.block = spnn.ExpertBlock(12, 24, 4, 2, dropout=0.5)

        def forward(self, coords, x):
            return self.block(SparseTensor(coords, x)).features

    dist.init_process_group("nccl", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        net = torch.nn.parallel.DistributedDataParallel(Net().to(dev), device_ids=[0])
        coords, x = voxels(device=dev)
        for _ in range(2):
            net(coords, x).sum().backward()
        torch.cuda.synchronize()
        assert int(net.module.block.calls) == 2 and net.module.block.up.grad is not None
    finally:
        dist.destroy_process_group()


@pytest.mark.gpu
def test_blocks_drop_positions_of_their_own(dev):
    """Of two default blocks of one width, the kept positions agree as often as independent ones do: half of 4096 x 64
    at p = 0.5, within 6 deviations (of 256 each)."""
    x = torch.randn(4096, 64, generator=torch.Generator().manual_seed(3)).to(dev)
    kept = []
    for _ in range(2):
        block = spnn.ExpertBlock(64, 64, 4, 2, dropout=0.5).to(dev)
        y = block(SparseTensor(torch.arange(4096, device=dev), x)).features
        kept.append(y != x)
    assert abs(int((kept[0] == kept[1]).sum()) - 2 ** 17) < 6 * 256


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation_with_the_kernels(dev, reentrant):
    check_recomputation(dev, reentrant, seed=5)
