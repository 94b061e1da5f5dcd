"""The mixture-of-experts block behind a sparse convolution: its outputs and
gradients against the same formulas in 64 bits, training and inference, and its
capture in a graph."""
import pytest
import torch

from spira_amd import SparseTensor, scenes
from spira_amd import nn as spnn
from spira_amd.nn import functional as F

pytestmark = pytest.mark.gpu


def scene(dev, channels, dtype, n=3000):
    coords = torch.from_numpy(scenes.spheres_planes(n=n, grid=40, seed=1)).to(dev)
    g = torch.Generator().manual_seed(0)
    x = SparseTensor(coords, torch.randn(len(coords), channels, generator=g).to(dtype).to(dev), double=True)
    return x.order()


def reference(block, x, routes, keep):
    """The block in 64 bits with the router's choice given: (output, leaves)."""
    p = {k: v.detach().double().requires_grad_(True) for k, v in block.named_parameters()}
    x = x.detach().double().requires_grad_(True)

    def norm(v, w):
        return v / torch.sqrt(v.pow(2).mean(1, keepdim=True) + block.eps) * w

    n = norm(x, p["entry"])
    chosen = routes.experts.long()
    weights = torch.softmax((n @ p["router"]).gather(1, chosen), 1)
    out = 0
    for j in range(block.choices):
        e = chosen[:, j]
        h = torch.relu(torch.einsum("nc,nch->nh", n, p["up"][e]) + p["up_bias"][e])
        out = out + weights[:, j:j + 1] * (torch.einsum("nh,nhc->nc", h, p["down"][e]) + p["down_bias"][e])
    if keep is not None:
        out = out * keep / (1 - block.dropout)
    return x + block.scale * p["gate"] * norm(out, p["exit"]), x, p


def far(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


def test_training_step_fp32(dev):
    """Outputs and all gradients.  Seven products and norms in fp32, each to about
    1e-6 of its result; the router's choice is the block's own."""
    torch.manual_seed(0)
    block = spnn.ExpertBlock(32, 80, 6, 2, dropout=0.25, scale=0.5, seed=7).to(dev)
    for p in (block.up_bias, block.down_bias):
        torch.nn.init.normal_(p, std=0.1)
    x = scene(dev, 32, torch.float32)
    x._features.requires_grad_(True)
    y = block(x)
    assert int(block.calls) == 1 and torch.equal(y.coordinates, x.coordinates)
    with torch.no_grad():
        n = F.rms_norm(x.features, block.entry, block.eps)
        routes = F.route_experts(n @ block.router, 2)
        keep = F.dropout(torch.ones_like(x.features), 0.25, 7, 0) != 0
    ref, leaf, params = reference(block, x.features, routes, keep)
    assert far(y.features, ref) < 2e-5
    d = torch.randn(ref.shape, generator=torch.Generator().manual_seed(1)).to(dev)
    y.features.backward(d)
    (ref * d.double()).sum().backward()
    assert far(x.features.grad, leaf.grad) < 5e-5
    for name, p in block.named_parameters():
        assert far(p.grad, params[name].grad) < 5e-5, name
    # the next call has another mask; inference has none
    again = block(x).features
    assert not torch.equal(again, y.features) and int(block.calls) == 2
    block.eval()
    with torch.no_grad():
        assert far(block(x).features, reference(block, x.features, routes, None)[0]) < 2e-5
    assert int(block.calls) == 2


@pytest.mark.parametrize("dtype,limit", [(torch.float16, 4e-3), (torch.bfloat16, 3e-2)])
def test_behind_a_convolution(dev, dtype, limit):
    """Inference in 16 bits: six roundings on the way of the update, a fraction of the residual's size."""
    torch.manual_seed(1)
    conv = spnn.SparseConv(16, 64, 3).to(dev).half()
    cache = spnn.KernelMapCache()
    from spira_amd import set_kernel_map_cache
    set_kernel_map_cache(conv, cache)
    x = scene(dev, 16, torch.float16)
    with torch.no_grad():
        h = conv(x).to(dtype)
        block = spnn.ExpertBlock(64, 128, 8, 2).to(dev).to(dtype).eval()
        y = block(h)
        n = F.rms_norm(h.features, block.entry, block.eps)
        routes = F.route_experts(n @ block.router, 2)
        ref = reference(block, h.features, routes, None)[0]
    assert y.features.dtype == dtype and y.stride == h.stride
    assert far(y.features, ref) < limit


def test_captured_in_a_graph(dev):
    """Every replay on new features equals the eager call."""
    torch.manual_seed(2)
    block = spnn.ExpertBlock(48, 96, 5, 2).to(dev).half().eval()
    x = scene(dev, 48, torch.float16, 800)
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


def test_state_and_device_moves(dev):
    block = spnn.ExpertBlock(16, 32, 4, dropout=0.5).to(dev)
    assert block.calls.device.type == "cpu" and block.calls.dtype == torch.int64
    block(scene(dev, 16, torch.float32, 200))
    other = spnn.ExpertBlock(16, 32, 4, dropout=0.5).to(dev)
    other.load_state_dict(block.state_dict())
    assert int(other.calls) == 1 and other.half().calls.dtype == torch.int64


def test_gradients_are_of_first_order(dev):
    x = torch.randn(8, 16, device=dev, requires_grad=True)
    w = torch.ones(16, device=dev, requires_grad=True)
    y = F.rms_norm(x, w)
    (d,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        d.sum().backward()
