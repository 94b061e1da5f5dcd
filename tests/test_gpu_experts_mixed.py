"""The row operators where a first set of tests does not reach: shares of a token
that cancel, loops over many rows, long sums in 16 bits, groups far from even,
and the ways of autograd around a call.

Tolerances as in test_gpu_experts.py: an output's own rounding, u |ref|, and the
error of a sum of n terms in fp32, n 2^-24 times the sum of their magnitudes
(twice that, for the roundings of the terms themselves)."""
import numpy as np
import pytest
import torch

from spira_amd.nn import functional as F

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}


def close(got, ref, magnitude, terms, what=""):
    """got within its rounding of ref plus a sum of `terms` terms of total magnitude `magnitude`."""
    got, dtype = got.detach().double(), got.dtype
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = UNIT[dtype] * ref.abs() * 1.001 + 2 * (terms + 16) * 2.0 ** -24 * magnitude + TINY[dtype]
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), torch.nonzero(bad)[0].tolist(), got[bad][0].item(), ref[bad][0].item())


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,experts,ci,co", [
    (9, 2, 2, 64, 64),          # few rows to a group
    (400, 3, 4, 48, 64),        # streamed
    (500, 2, 2, 512, 256),      # tiles
    (9000, 2, 2, 1032, 64),     # large tiles
    (300, 2, 3, 1031, 65)])     # tiles through registers
def test_gradient_of_shares_that_cancel(dev, tokens, k, experts, ci, co, dtype):
    """A token's share of each of its experts is some 60000, past the largest fp16
    number for many, and their sum a few hundred: the shares may not be rounded to
    the features' type before they are added."""
    dt = DTYPES[dtype]
    routes = F.route_experts(randn((tokens, experts), torch.float32, 5).to(dev), k)
    size = 60000 / co ** 0.5
    common, own = randn((ci, co), dt, 1, size), randn((experts, ci, co), torch.float32, 2, size / 128)
    # (every second expert's weights are the others' negative, and a little of its own)
    sign = torch.tensor([1.0, -1.0] * experts)[:experts, None, None]
    w = (sign * common.float() + own).to(dt).to(dev)
    dy = randn((tokens, co), dt, 3).to(dev)
    x = torch.zeros(tokens, ci, dtype=dt, device=dev, requires_grad=True)
    slots, chosen = routes.slots.long(), routes.experts.long()
    given = torch.zeros(tokens * k, co, dtype=dt, device=dev)
    given[slots.reshape(-1)] = dy.repeat_interleave(k, 0)
    (dx,) = torch.autograd.grad(F.grouped_linear(x, w, routes), x, given)
    ref = torch.zeros(tokens, ci, dtype=torch.float64, device=dev)
    magnitude = torch.zeros_like(ref)
    for e in range(experts):
        of = (chosen == e).any(1)
        d = dy[of].double()
        ref[of] += d @ w[e].double().T
        magnitude[of] += d.abs() @ w[e].double().T.abs()
    fits = ref.abs() < 65000 if dtype == "f16" else torch.ones_like(ref, dtype=torch.bool)
    assert fits.float().mean() > 0.5
    close(dx[fits], ref[fits], magnitude[fits], k * co, "dx")


def operators(dev):
    """Each operator as a function of its floating arguments, and those."""
    routes = F.route_experts(randn((12, 4), torch.float32, 1).to(dev), 2)
    calls = {
        "grouped_linear": (lambda x, w, b: F.grouped_linear(x, w, routes, bias=b), (12, 16), (4, 16, 8), (4, 8)),
        "route_experts": (lambda l: F.route_experts(l, 2).weights, (12, 4)),
        "combine_experts": (lambda h, w: F.combine_experts(h, routes._replace(weights=w)), (24, 16), (12, 2)),
        "gated_residual_norm": (lambda x, h, w, g, n: F.gated_residual_norm(x, h, weight=w, gate=g, next_weight=n)[1],
                                (12, 16), (12, 16), (16,), (12, 16), (16,)),
        "rms_norm": (F.rms_norm, (12, 16), (16,)),
        "dropout": (lambda x, r: F.dropout(x, 0.5, 1, residual=r), (12, 16), (12, 16)),
    }
    for name, (f, *shapes) in calls.items():
        yield name, f, [randn(s, torch.float32, 10 + i).to(dev) for i, s in enumerate(shapes)]


@pytest.mark.parametrize("wants", [False, True])
def test_tangents_of_forward_mode_are_refused(dev, wants):
    """Of each argument, with and without a gradient asked for; where forward mode is off they do not matter."""
    from torch.autograd import forward_ad
    for name, f, args in operators(dev):
        for i in range(len(args)):
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(t.clone().requires_grad_(wants), torch.ones_like(t)) if j == i else t
                        for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match=r"\[Spira\].*forward mode"):
                    f(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match=r"\[Spira\].*forward mode"):
                    f(*dual)
                with forward_ad._set_fwd_grad_enabled(False):
                    assert torch.equal(f(*dual).detach(), f(*args)), (name, i)


def test_sigmoid_gate_in_fp32(dev):
    """The gate alone (residual 0, update 1): the exponential is good to one ulp (2^-23 of it), the sum and the
    division to half of one each, so that the gate is within 2^-22 of its value."""
    n, c = 64, 1024
    gate = torch.linspace(-80, 80, n * c, dtype=torch.float32, device=dev).view(n, c)
    r, _ = F.gated_residual_norm(torch.zeros_like(gate), torch.ones_like(gate), gate=gate, gate_sigmoid=True)
    ref = 1 / (1 + torch.exp(-gate.double()))
    off = ((r.double() - ref).abs() / ref).max().item()
    assert off <= 2.0 ** -22, off


class Cut(torch.autograd.Function):
    """Passes values on, and no gradient back."""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, d):
        return None


def test_no_gradient_comes_back(dev):
    """A function behind an operator that returns no gradient leaves those of the rest as they are."""
    for name, f, args in operators(dev):
        leaves = [t.requires_grad_(True) for t in args]
        grads = torch.autograd.grad(Cut.apply(f(*leaves)).sum() + sum(t.sum() for t in leaves), leaves)
        for i, g in enumerate(grads):
            assert torch.equal(g, torch.ones_like(g)), (name, i)


def test_seeds_of_other_integer_types(dev):
    """NumPy's integers and tensors of one value, as a program's counters are; other numbers are refused."""
    x = randn((40, 16), torch.float32, 1).to(dev)
    for seed in (5, -5, 2 ** 62 + 1):
        ref = F.dropout(x, 0.5, seed, 7)
        assert torch.equal(F.dropout(x, 0.5, np.int64(seed), np.int32(7)), ref)
        assert torch.equal(F.dropout(x, 0.5, torch.tensor(seed), torch.tensor(7)), ref)
    with pytest.raises(TypeError):
        F.dropout(x, 0.5, 5.0)
    with pytest.raises(TypeError):
        F.dropout(x, 0.5, 5, 0.5)


def test_combine_gradient_of_more_rows_than_a_launch_has_threads_for(dev):
    """2^27 tokens and as many rows, 16 threads to each: past 2^32 threads, which is what one launch can have."""
    n = (1 << 27) + 21
    slots = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=dev)
    rows = slots.clone()  # (row r is that of token n - 1 - r)
    slots[::1000], rows[(n - 1 - torch.arange(0, n, 1000, device=dev))] = -1, -1
    offsets = torch.zeros(2, dtype=torch.int32, device=dev)
    h = (torch.arange(n, device=dev) % 61).half().view(n, 1).requires_grad_(True)
    weights = (torch.arange(n, device=dev) % 7 + 1).float().view(n, 1).requires_grad_(True)
    y = F.combine_experts(h, F.ExpertRoutes(weights, slots.view(n, 1), offsets, rows, slots.view(n, 1)))
    dy = (torch.arange(n, device=dev) % 5).half().view(n, 1)
    dh, dw = torch.autograd.grad(y, (h, weights), dy)
    # (small whole numbers throughout: exact)
    there = (slots >= 0).view(n, 1)
    taken = h.detach().flip(0)
    assert torch.equal(y, (taken * weights.half()).masked_fill(~there, 0))
    assert torch.equal(dw, (taken * dy).float().masked_fill(~there, 0))
    assert torch.equal(dh.flip(0), (weights.half() * dy).masked_fill(~there, 0))


def test_combine_refuses_features_of_other_routes(dev):
    routes = F.route_experts(randn((10, 4), torch.float32, 1).to(dev), 2)
    for rows in (10, 19, 21):
        for grad in (False, True):
            with pytest.raises(RuntimeError, match=r"\[Spira\].*do not fit"):
                F.combine_experts(torch.zeros(rows, 8, device=dev, requires_grad=grad), routes)
    with pytest.raises(RuntimeError, match=r"\[Spira\].*do not fit"):
        F.combine_experts(torch.zeros(20, device=dev), routes)
    with torch.inference_mode():
        assert F.combine_experts(torch.zeros(20, 8, device=dev), routes).shape == (10, 8)
