"""The row operators of the mixture-of-experts block against plain
implementations in 64 bits.

Tolerances follow from the arithmetic: a value is off by at most its own
rounding to the output type, u |ref| with u = 2^-11 (fp16), 2^-8 (bf16) or 2^-24
(fp32), plus the error of a sum of n terms in fp32, n 2^-24 times the sum of the
terms' magnitudes (twice that, for the roundings of the terms themselves)."""
import math

import pytest
import torch

from spira_amd.nn import functional as F

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}


def close(got, ref, magnitude, terms, what="", dtype=None):
    """got within its rounding of ref plus a sum of `terms` terms of total magnitude `magnitude`."""
    dtype = dtype or got.dtype
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = UNIT[dtype] * ref.abs() * 1.001 + 2 * (terms + 16) * 2.0 ** -24 * magnitude.double().cpu() + TINY[dtype]
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), torch.nonzero(bad)[0].tolist(), got[bad][0].item(), ref[bad][0].item())


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


# ---------------------------------------------------------------------------
# grouped_linear
# ---------------------------------------------------------------------------
def linear_reference(x, w, b, offsets, rows, relu):
    """(y, magnitude of its terms) in 64 bits."""
    x, w = x.double(), w.double()
    n = len(rows) if rows is not None else len(x)
    y = torch.zeros(n, w.shape[2], dtype=torch.float64)
    m = torch.zeros_like(y)
    for e in range(len(w)):
        at = slice(offsets[e], offsets[e + 1])
        xe = x[rows[at].long()] if rows is not None else x[at]
        y[at], m[at] = xe @ w[e], xe.abs() @ w[e].abs()
        if b is not None:
            y[at] += b[e].double()
            m[at] += b[e].double().abs()
    return (y.clamp(min=0) if relu else y), m


def group_sizes(kind, groups, rows, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "even":
        return [rows // groups] * groups
    if kind == "one":  # everything in one group, none in the others
        return [rows if e == groups // 2 else 0 for e in range(groups)]
    if kind == "ends":  # rows outside all groups follow
        return [0] * (groups - 1) + [max(rows - 5, 0)]
    cuts = sorted(torch.randint(0, rows + 1, (groups - 1,), generator=g).tolist())
    return [b - a for a, b in zip([0] + cuts, cuts + [rows])]


LINEAR = [
    # groups, rows, c_in, c_out, sizes
    (1, 1, 1, 1, "even"), (3, 0, 16, 16, "even"), (4, 7, 16, 32, "random"), (2, 130, 64, 128, "random"),
    (5, 300, 63, 130, "random"), (8, 513, 96, 384, "random"), (8, 1000, 33, 17, "ends"), (3, 400, 200, 72, "one"),
    (70, 333, 40, 24, "random"), (130, 129, 8, 8, "random"), (2, 257, 129, 257, "even"), (4, 2100, 128, 136, "random"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,rows,ci,co,kind", LINEAR)
def test_grouped_linear(dev, groups, rows, ci, co, kind, dtype):
    dt = DTYPES[dtype]
    sizes = group_sizes(kind, groups, rows, rows)
    offsets = torch.tensor([0] + sizes).cumsum(0)
    x, w = randn((rows, ci), dt, 1), randn((groups, ci, co), dt, 2, ci ** -0.5)
    for b, relu in ((None, False), (randn((groups, co), dt, 3, 0.1), True)):
        y, m = linear_reference(x, w, b, offsets, None, relu)
        got = F.grouped_linear(x.to(dev), w.to(dev), offsets.int().to(dev), bias=None if b is None else b.to(dev),
                               relu=relu)
        close(got, y, m, ci, "y")
        if sum(sizes) < rows:
            assert torch.count_nonzero(got[sum(sizes):]) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("groups,rows,ci,co,kind", LINEAR)
def test_grouped_linear_gradients(dev, groups, rows, ci, co, kind, relu, dtype):
    dt = DTYPES[dtype]
    sizes = group_sizes(kind, groups, rows, rows + 1)
    offsets = torch.tensor([0] + sizes).cumsum(0)
    x, w = randn((rows, ci), dt, 1), randn((groups, ci, co), dt, 2, ci ** -0.5)
    b, dy = randn((groups, co), dt, 3, 0.1), randn((rows, co), dt, 4)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b)]
    y = F.grouped_linear(leaves[0], leaves[1], offsets.int().to(dev), bias=leaves[2], relu=relu)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(dev))
    # (the activation's mask as the outputs have it: a value near zero may fall on either side)
    dz = dy.double() * (y.detach().cpu() > 0) if relu else dy.double()
    for e in range(groups):
        at = slice(offsets[e], offsets[e + 1])
        xe, ze, we = x[at].double(), dz[at], w[e].double()
        close(dx[at], ze @ we.T, ze.abs() @ we.T.abs(), co, f"dx {e}")
        close(dw[e], xe.T @ ze, xe.T.abs() @ ze.abs(), sizes[e], f"dw {e}")
        close(db[e], ze.sum(0), ze.abs().sum(0), sizes[e], f"db {e}")
    assert torch.count_nonzero(dx[sum(sizes):]) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,experts,ci,co,masked", [
    (1, 1, 2, 32, 64, 0), (8, 2, 32, 512, 200, 0), (60, 3, 5, 37, 45, 0.4), (700, 2, 8, 96, 128, 0.1), (5, 2, 3, 16, 16, 1)])
def test_grouped_linear_of_routes(dev, tokens, k, experts, ci, co, masked, dtype):
    """Rows gathered from the tokens, and their gradients summed per token."""
    dt = DTYPES[dtype]
    logits = randn((tokens, experts), torch.float32, 5)
    logits[torch.rand(logits.shape, generator=torch.Generator().manual_seed(6)) < masked] = -math.inf
    routes = F.route_experts(logits.to(dev), k)
    x, w, dy = randn((tokens, ci), dt, 1), randn((experts, ci, co), dt, 2, ci ** -0.5), randn((tokens * k, co), dt, 4)
    offsets, rows, slots = routes.offsets.cpu().long(), routes.rows.cpu(), routes.slots.cpu().long()
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w)]
    y = F.grouped_linear(*leaves, routes)
    ref, m = linear_reference(x, w, None, offsets, rows, False)
    close(y, ref, m, ci, "y")
    with torch.no_grad():
        assert torch.equal(y, F.grouped_linear(*leaves, routes))
    dx, dw = torch.autograd.grad(y, leaves, dy.to(dev))
    share, size = torch.zeros(tokens * k, ci, dtype=torch.float64), torch.zeros(tokens * k, ci, dtype=torch.float64)
    for e in range(experts):
        at = slice(offsets[e], offsets[e + 1])
        xe, ze, we = x[rows[at].long()].double(), dy[at].double(), w[e].double()
        share[at], size[at] = ze @ we.T, ze.abs() @ we.T.abs()
        close(dw[e], xe.T @ ze, xe.T.abs() @ ze.abs(), len(xe), f"dw {e}")
    held = (slots >= 0)[:, :, None]
    parts = share[slots.clamp(min=0)] * held
    # (each share is rounded to the features' type on its way)
    extra = (UNIT[dt] * parts.abs()).sum(1) / (2 * 2.0 ** -24 * (co + k + 16))
    close(dx, parts.sum(1), (size[slots.clamp(min=0)] * held).sum(1) + extra * 1.01, co + k, "dx")


def test_grouped_linear_long_group_and_odd_views(dev):
    """Rows past a part of the weights' gradient, and tensors that start off a chunk's boundary."""
    rows, ci, co = 20_000, 48, 40
    base = randn((rows * ci + 1,), torch.float16, 1).to(dev)
    x = base[1:].view(rows, ci)
    w = randn((2 * ci * co + 3,), torch.float16, 2, ci ** -0.5).to(dev)[3:].view(2, ci, co)
    offsets = torch.tensor([0, 19_000, 19_003], dtype=torch.int32, device=dev)
    dy = randn((rows * co + 5,), torch.float16, 3).to(dev)[5:].view(rows, co)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    y = F.grouped_linear(*leaves, offsets)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    xd, wd, dd = x.detach().double(), w.detach().double(), dy.double()
    for e, (lo, hi) in enumerate(((0, 19_000), (19_000, 19_003))):
        close(y[lo:hi], xd[lo:hi] @ wd[e], xd[lo:hi].abs() @ wd[e].abs(), ci, "y")
        close(dx[lo:hi], dd[lo:hi] @ wd[e].T, dd[lo:hi].abs() @ wd[e].T.abs(), co, "dx")
        close(dw[e], xd[lo:hi].T @ dd[lo:hi], xd[lo:hi].T.abs() @ dd[lo:hi].abs(), hi - lo, "dw")
    assert torch.count_nonzero(y[19_003:]) == 0 and torch.count_nonzero(dx[19_003:]) == 0


@pytest.mark.parametrize("dtype,groups,rows,ci,co", [
    ("bf16", 12, 17_000, 1032, 1032),  # large tiles both ways
    ("f16", 100, 9_000, 256, 328),     # more groups than lanes
    ("f32", 5, 3_000, 320, 260), ("f16", 3, 40_000, 384, 512), ("bf16", 2, 300, 2048, 136)])
def test_grouped_linear_wide(dev, dtype, groups, rows, ci, co):
    """Weights too large for LDS: gathered rows, groups of any size, tokens without an expert."""
    dt = DTYPES[dtype]
    logits = randn((rows, groups), torch.float32, 1) + torch.linspace(2, 0, groups)
    logits[::7] = -math.inf
    routes = F.route_experts(logits.to(dev), 1)
    x, w = randn((rows, ci), dt, 2).to(dev), randn((groups, ci, co), dt, 3, ci ** -0.5).to(dev)
    b, dy = randn((groups, co), dt, 4, 0.1).to(dev), randn((rows, co), dt, 5).to(dev)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = F.grouped_linear(x, w, routes, bias=b, relu=True)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    offsets, at = routes.offsets.tolist(), routes.rows.long()
    used = torch.zeros(rows, dtype=torch.bool, device=dev)
    for e in range(groups):
        lo, hi = offsets[e], offsets[e + 1]
        source = at[lo:hi]
        used[source] = True
        xe, we, be = x[source].detach().double(), w[e].detach().double(), b[e].detach().double()
        ze = dy[lo:hi].double() * (y[lo:hi] > 0)
        close(y[lo:hi], (xe @ we + be).clamp(min=0), xe.abs() @ we.abs() + be.abs(), ci, f"y {e}")
        close(dx[source], ze @ we.T, ze.abs() @ we.T.abs(), co, f"dx {e}")
        close(dw[e], xe.T @ ze, xe.T.abs() @ ze.abs(), hi - lo, f"dw {e}")
        close(db[e], ze.sum(0), ze.abs().sum(0), hi - lo, f"db {e}")
    assert torch.count_nonzero(dx[~used]) == 0 and torch.count_nonzero(y[offsets[-1]:]) == 0


def test_grouped_linear_nonfinite_rows_stay_in_their_rows(dev):
    """Infinities and NaN of one row, or outside the groups, reach no other row."""
    x = randn((200, 72), torch.float16, 1)
    w = randn((3, 72, 80), torch.float16, 2, 0.1)
    offsets = torch.tensor([10, 70, 70, 180], dtype=torch.int32)
    clean = F.grouped_linear(x.to(dev), w.to(dev), offsets.to(dev))
    x[30], x[100], x[5], x[190] = math.nan, math.inf, math.nan, math.inf
    w[1] = math.nan  # (of a group without rows)
    got = F.grouped_linear(x.to(dev), w.to(dev), offsets.to(dev))
    keep = torch.ones(200, dtype=torch.bool)
    keep[[30, 100]] = False
    assert torch.equal(got.cpu()[keep], clean.cpu()[keep])
    assert got[30].isnan().all() and not got[100].isfinite().any()
    assert torch.count_nonzero(got[:10]) == 0 and torch.count_nonzero(got[180:]) == 0


def test_grouped_linear_repeats_bit_for_bit(dev):
    x, w = randn((5000, 96), torch.bfloat16, 1).to(dev), randn((6, 96, 160), torch.bfloat16, 2, 0.1).to(dev)
    offsets = torch.tensor([0, 100, 2900, 2900, 3500, 3501, 5000], dtype=torch.int32, device=dev)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    dy = randn((5000, 160), torch.bfloat16, 3).to(dev)
    first = None
    for _ in range(3):
        y = F.grouped_linear(*leaves, offsets, relu=True)
        out = [y, *torch.autograd.grad(y, leaves, dy)]
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_grouped_linear_offsets_out_of_range_are_clamped(dev):
    """Offsets that leave the rows give the rows they share with them, nothing else."""
    x, w = randn((50, 16), torch.float16, 1).to(dev), randn((2, 16, 24), torch.float16, 2, 0.25).to(dev)
    y = F.grouped_linear(x, w, torch.tensor([-7, 20, 1000], dtype=torch.int32, device=dev))
    good = F.grouped_linear(x, w, torch.tensor([0, 20, 50], dtype=torch.int32, device=dev))
    assert torch.equal(y, good)


# ---------------------------------------------------------------------------
# route_experts, combine_experts
# ---------------------------------------------------------------------------
def route_reference(logits, k, renormalize):
    """One token at a time, in 64 bits."""
    l = logits.double()
    tokens, experts = l.shape
    weights, chosen = torch.zeros(tokens, k, dtype=torch.float64), torch.full((tokens, k), -1, dtype=torch.int64)
    for t in range(tokens):
        order = sorted((e for e in range(experts) if l[t, e] > -math.inf), key=lambda e: (-l[t, e].item(), e))[:k]
        if not order:
            continue
        over = l[t, order] if renormalize else l[t]
        weights[t, :len(order)] = torch.exp(l[t, order] - torch.logsumexp(over, 0))
        chosen[t, :len(order)] = torch.tensor(order)
    return weights, chosen


def check_order(routes, tokens, k, experts):
    chosen = routes.experts.cpu().long()
    flat = chosen.reshape(-1)
    order = [a for e in range(experts) for a in torch.nonzero(flat == e)[:, 0].tolist()]
    counts = [int((flat == e).sum()) for e in range(experts)]
    assert routes.offsets.tolist() == [0] + torch.tensor(counts).cumsum(0).tolist()
    assert routes.rows.tolist() == [a // k for a in order] + [-1] * (tokens * k - len(order))
    slots = [-1] * (tokens * k)
    for r, a in enumerate(order):
        slots[a] = r
    assert routes.slots.reshape(-1).tolist() == slots


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,k,masked", [
    (1, 1, 1, 0), (1, 8, 8, 0), (8, 32, 2, 0), (63, 9, 3, 0.5), (65, 17, 4, 0.9), (400, 64, 6, 0.1), (130, 200, 16, 0.3),
    (40, 512, 5, 0), (1025, 16, 2, 0.05), (3, 5, 2, 1.0)])
def test_route(dev, tokens, experts, k, masked, renormalize, dtype):
    dt = DTYPES[dtype]
    logits = randn((tokens, experts), torch.float32, 1, 1.5)
    logits[torch.rand(logits.shape, generator=torch.Generator().manual_seed(2)) < masked] = -math.inf
    logits = logits.to(dt)
    leaf = logits.to(dev).requires_grad_(True)
    routes = F.route_experts(leaf, k, renormalize=renormalize)
    weights, chosen = route_reference(logits, k, renormalize)
    assert torch.equal(routes.experts.cpu().long(), chosen)
    # (an exponential is good to two units, its argument to one; sums of up to `experts`)
    close(routes.weights, weights, weights * (1 + 8 / (2.0 * experts)), experts, "weights")
    check_order(routes, tokens, k, experts)
    d = randn((tokens, k), torch.float32, 3)
    (dl,) = torch.autograd.grad(routes.weights, leaf, d.to(dev))
    held = chosen >= 0
    dd = d.double() * held
    p = torch.zeros(tokens, experts + 1, dtype=torch.float64)
    g = torch.zeros_like(p)
    at = torch.where(held, chosen, experts)
    g.scatter_(1, at, dd)
    if renormalize:
        p.scatter_(1, at, weights)
    else:
        l = logits.double()
        p[:, :-1] = torch.where(l > -math.inf, torch.exp(l - torch.logsumexp(l, 1, keepdim=True)), 0)
    p, g = p[:, :-1], g[:, :-1]
    mean = (dd * weights).sum(1, keepdim=True)
    size = p * (g.abs() + (dd.abs() * weights).sum(1, keepdim=True))
    close(dl, p * (g - mean), size, 2 * experts + 4 * k, "dlogits")


@pytest.mark.parametrize("dtype", DTYPES)
def test_route_ties_extremes_and_nan(dev, dtype):
    """Ties and both zeros by the lowest index; the type's lowest value is a number; -inf is not; NaN and inf."""
    dt = DTYPES[dtype]
    low = torch.finfo(dt).min
    n, i = math.nan, math.inf
    logits = torch.tensor([[1, 2, 2, 1], [0.0, -0.0, 0.0, -0.0], [low, low, -i, low], [-i, -i, low, -i], [-i] * 4,
                           [n, 1, 2, 3], [1, i, 2, i], [-n, 5, n, 6]], dtype=dt)
    r = F.route_experts(logits.to(dev), 3)
    assert r.experts.tolist() == [[1, 2, 0], [0, 1, 2], [0, 1, 3], [2, -1, -1], [-1, -1, -1], [0, 3, 2], [1, 3, 2],
                                  [0, 2, 3]]
    w = r.weights.cpu()
    assert torch.equal(w[2:5], torch.tensor([[1 / 3] * 3, [1, 0, 0], [0, 0, 0]]))
    assert torch.equal(w[1], torch.tensor([1 / 3] * 3))
    assert w[5:].isnan().all()
    check_order(r, 8, 3, 4)
    for t in (3, 4):
        full = F.route_experts(logits[t:t + 1].to(dev), 3, renormalize=False)
        assert torch.equal(full.weights.cpu(), w[t:t + 1])


@pytest.mark.parametrize("tokens,k,experts", [(1024, 2, 7), (1025, 2, 7), (70_000, 3, 40), (3, 4, 512), (300_000, 1, 3)])
def test_route_order_of_many(dev, tokens, k, experts):
    """The order over many blocks, against a stable sort."""
    r = F.route_experts(randn((tokens, experts), torch.float16, tokens).to(dev), k)
    flat = r.experts.long().reshape(-1)
    _, order = torch.sort(flat, stable=True)
    assert torch.equal(r.rows.long(), order // k)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(len(order), device=dev)
    assert torch.equal(r.slots.long().reshape(-1), slots)
    assert torch.equal(r.offsets[1:].long(), torch.bincount(flat, minlength=experts).cumsum(0))


def test_route_of_no_tokens(dev):
    leaf = torch.zeros(0, 6, device=dev, requires_grad=True)
    r = F.route_experts(leaf, 2)
    assert r.offsets.tolist() == [0] * 7 and r.rows.numel() == 0 and r.weights.shape == (0, 2)
    w = torch.ones(6, 8, 4, device=dev)
    h = F.grouped_linear(torch.zeros(0, 8, device=dev), w, r)
    y = F.combine_experts(h, r)
    assert h.shape == (0, 4) and y.shape == (0, 4)
    (d,) = torch.autograd.grad(r.weights.sum() + y.sum(), leaf)
    assert d.shape == (0, 6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,experts,c,masked", [
    (1, 1, 2, 1, 0), (8, 2, 32, 512, 0), (77, 3, 6, 96, 0.5), (300, 2, 5, 33, 0.2), (20, 4, 4, 1000, 0), (6, 2, 3, 16, 1)])
def test_combine(dev, tokens, k, experts, c, masked, dtype):
    dt = DTYPES[dtype]
    logits = randn((tokens, experts), torch.float32, 5)
    logits[torch.rand(logits.shape, generator=torch.Generator().manual_seed(6)) < masked] = -math.inf
    routes = F.route_experts(logits.to(dev), k)
    h, dy = randn((tokens * k, c), dt, 1), randn((tokens, c), dt, 2)
    hl, wl = h.to(dev).requires_grad_(True), routes.weights.clone().requires_grad_(True)
    y = F.combine_experts(hl, routes._replace(weights=wl))
    slots, w = routes.slots.cpu().long(), routes.weights.cpu().double()
    held = slots >= 0
    taken = h.double()[slots.clamp(min=0)] * held[:, :, None]
    close(y, (w[:, :, None] * taken).sum(1), (w[:, :, None] * taken).abs().sum(1), k, "y")
    dh, dw = torch.autograd.grad(y, (hl, wl), dy.to(dev))
    ref = torch.zeros(tokens * k + 1, c, dtype=torch.float64)
    ref[torch.where(held, slots, tokens * k)] = w[:, :, None] * dy.double()[:, None]
    close(dh, ref[:-1], ref[:-1].abs(), 1, "dh")
    close(dw, (taken * dy.double()[:, None]).sum(2), (taken * dy.double()[:, None]).abs().sum(2), c, "dw")


# ---------------------------------------------------------------------------
# gated_residual_norm, rms_norm
# ---------------------------------------------------------------------------
def norm_reference(x, h, w, gate, sigmoid, scale, w_next, eps):
    z = h
    if w is not None:
        z = h / torch.sqrt(h.pow(2).mean(1, keepdim=True) + eps) * w
    if gate is not None:
        z = z * (torch.sigmoid(gate) if sigmoid else gate)
    r = x + scale * z
    n = None if w_next is None else r / torch.sqrt(r.pow(2).mean(1, keepdim=True) + eps) * w_next
    return r, n


def near(got, ref, c, what, lost=1.0):
    """A value of a norm or its gradient.  Every term of its formula is at most
    `lost` times the row's (or column's) largest result, with sums of up to c
    terms, taken twice over, on the way."""
    dtype = got.dtype
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    top = ref.abs().amax(tuple(range(1, ref.dim())) if ref.dim() > 1 else None, keepdim=ref.dim() > 1)
    tol = UNIT[dtype] * ref.abs() * 1.001 + (4 * c + 64) * 2.0 ** -24 * lost * top + TINY[dtype]
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), torch.nonzero(bad)[0].tolist(), got[bad][0].item(), ref[bad][0].item())


NORMS = [(1, 1), (1, 512), (7, 16), (33, 63), (100, 96), (257, 200), (65, 512), (12, 1000), (9, 1024), (5, 2048),
         (3, 4095), (3, 8192), (2, 16384), (1500, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate,sigmoid", [("none", False), ("channel", False), ("row", True), ("full", True)])
@pytest.mark.parametrize("n,c", NORMS)
def test_gated_residual_norm(dev, n, c, gate, sigmoid, dtype):
    dt = DTYPES[dtype]
    x, h = randn((n, c), dt, 1, 2.0), randn((n, c), dt, 2)
    w, w_next = 1 + randn((c,), dt, 3, 0.1), 1 + randn((c,), dt, 4, 0.1)
    shape = {"none": None, "channel": (c,), "row": (n, 1), "full": (n, c)}[gate]
    g = None if shape is None else randn(shape, dt, 5)
    tensors = [x, h, w, w_next] + ([] if g is None else [g])
    leaves = [t.to(dev).requires_grad_(True) for t in tensors]
    exact = [t.double().requires_grad_(True) for t in tensors]

    def call(f, v, **kw):
        return f(v[0], v[1], v[2], v[4] if g is not None else None, v[3], **kw)

    r, nx = call(lambda a, b, w, g, wn: F.gated_residual_norm(a, b, weight=w, gate=g, gate_sigmoid=sigmoid, scale=0.5,
                                                              next_weight=wn, eps=1e-6), leaves)
    rr, nr = call(lambda a, b, w, g, wn: norm_reference(a, b, w, g, sigmoid, 0.5, wn, 1e-6), exact)
    near(r, rr, c, "r")
    near(nx, nr, c, "n")
    with torch.no_grad():
        r2, n2 = call(lambda a, b, w, g, wn: F.gated_residual_norm(a, b, weight=w, gate=g, gate_sigmoid=sigmoid,
                                                                   scale=0.5, next_weight=wn, eps=1e-6), leaves)
        assert torch.equal(r, r2) and torch.equal(nx, n2)
    dr, dn = randn((n, c), dt, 6), randn((n, c), dt, 7)
    got = torch.autograd.grad((r, nx), leaves, (dr.to(dev), dn.to(dev)))
    ref = torch.autograd.grad((rr, nr), exact, (dr.double(), dn.double()))
    # (sums over the rows of terms up to a few times their rows' result; one channel's norm has a gradient of zero
    # but for eps, the difference of terms of the gradient's own size)
    for name, a, b in zip(("dx", "dh", "dw", "dw_next", "dgate"), got, ref):
        lost = 4.0 if a.dim() == 2 and a.shape[1] > 1 else 4.0 * max(1, n) ** 0.5
        if c == 1:
            a, b = a.double() / 64, b / 64
            assert (a.cpu() - b).abs().max() <= UNIT[dt] * b.abs().max() * 1.01 + 256 * 2.0 ** -24 * n, name
        else:
            near(a, b, c + n, name, lost)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", [(1, 8), (40, 96), (3, 3000)])
def test_norm_parts(dev, n, c, dtype):
    """Without a norm, a gate or a next norm; and the entry norm alone."""
    dt = DTYPES[dtype]
    x, h, w = randn((n, c), dt, 1), randn((n, c), dt, 2), 1 + randn((c,), dt, 3, 0.1)
    d = randn((n, c), dt, 4)
    xl, hl, wl = (t.to(dev).requires_grad_(True) for t in (x, h, w))
    xe, he, we = (t.double().requires_grad_(True) for t in (x, h, w))
    r, none = F.gated_residual_norm(xl, hl, scale=-2.0)
    assert none is None
    near(r, xe - 2 * he, 1, "r")
    dx, dh = torch.autograd.grad(r, (xl, hl), d.to(dev))
    assert torch.equal(dx.cpu(), d) and torch.equal(dh.cpu(), -2 * d)
    r, _ = F.gated_residual_norm(xl, hl, weight=wl)
    rr, _ = norm_reference(xe, he, we, None, False, 1.0, None, 1e-6)
    near(r, rr, c, "r")
    for a, b in zip(torch.autograd.grad(r, (xl, hl, wl), d.to(dev)), torch.autograd.grad(rr, (xe, he, we), d.double())):
        near(a, b, c + n, "gradient", 4.0 * n ** 0.5)
    y = F.rms_norm(xl, wl, 1e-5)
    yr = xe / torch.sqrt(xe.pow(2).mean(1, keepdim=True) + 1e-5) * we
    near(y, yr, c, "rms_norm")
    for a, b in zip(torch.autograd.grad(y, (xl, wl), d.to(dev)), torch.autograd.grad(yr, (xe, we), d.double())):
        near(a, b, c + n, "rms_norm gradient", 4.0 * n ** 0.5)
    # only one of the two outputs is used, or one leaf wants a gradient
    r, nx = F.gated_residual_norm(xl, hl, weight=wl, next_weight=wl)
    rr, nr = norm_reference(xe, he, we, None, False, 1.0, we, 1e-6)
    near(torch.autograd.grad(nx, hl, d.to(dev))[0], torch.autograd.grad(nr, he, d.double())[0], c, "dh of n", 4.0)
    r, nx = F.gated_residual_norm(xl.detach(), hl.detach(), weight=wl, next_weight=wl.detach())
    rr, nr = norm_reference(xe.detach(), he.detach(), we, None, False, 1.0, we.detach(), 1e-6)
    near(torch.autograd.grad(r, wl, d.to(dev))[0], torch.autograd.grad(rr, we, d.double())[0], c + n, "dw", 4.0 * n ** 0.5)


def test_norm_of_no_rows_zeros_and_nonfinite(dev):
    w = torch.ones(40, device=dev, requires_grad=True)
    r, n = F.gated_residual_norm(torch.zeros(0, 40, device=dev), torch.zeros(0, 40, device=dev), weight=w, next_weight=w)
    assert r.shape == n.shape == (0, 40)
    (dw,) = torch.autograd.grad(r.sum() + n.sum(), w)
    assert torch.count_nonzero(dw) == 0
    x = torch.zeros(3, 40, device=dev)
    h = torch.zeros(3, 40, device=dev)
    h[1, 3] = math.nan
    x[2, 5] = math.inf
    r, n = F.gated_residual_norm(x, h, weight=w.detach(), next_weight=w.detach())
    assert torch.count_nonzero(r[0]) == 0 and torch.count_nonzero(n[0]) == 0
    assert r[1].isnan().all() and n[1].isnan().all()
    assert r[2, 5] == math.inf and torch.count_nonzero(r[2]) == 1 and n[2, 5].isnan() and torch.count_nonzero(n[2]) == 1


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
def keep_reference(count, p, seed, offset):
    """Philox-4x32 with 7 rounds in Python's integers."""
    keep = []
    for i in range((count + 3) // 4):
        c = [i & 0xFFFFFFFF, i >> 32, offset & 0xFFFFFFFF, offset >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(7):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        keep += [v >= int(p * 2 ** 32) for v in c]
    return torch.tensor(keep[:count])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,p,seed,offset", [((1, 1), 0.5, 1, 0), ((37, 51), 0.1, 2 ** 64 - 1, 2 ** 40 + 3),
                                                 ((9, 1000), 0.9, 12345, 7), ((4, 6, 10), 0.3, 0, 2 ** 64 - 1)])
def test_dropout(dev, shape, p, seed, offset, dtype):
    dt = DTYPES[dtype]
    x, res, dy = (randn(shape, dt, s) for s in (1, 2, 3))
    keep = keep_reference(x.numel(), p, seed, offset).view(shape)
    scale = 1 / (1 - p)
    xl, rl = x.to(dev).requires_grad_(True), res.to(dev).requires_grad_(True)
    y = F.dropout(xl, p, seed, offset)
    ref = x.double() * keep * scale
    close(y, ref, ref.abs(), 1, "y")
    assert torch.equal((y != 0).cpu(), keep & (x != 0))
    z = F.dropout(xl, p, seed, offset, residual=rl)
    close(z, ref + res.double(), ref.abs() + res.double().abs(), 2, "with residual")
    dx, dres = torch.autograd.grad(z, (xl, rl), dy.to(dev))
    close(dx, dy.double() * keep * scale, dy.double().abs() * scale, 1, "dx")
    assert torch.equal(dres.cpu(), dy)


def test_dropout_ends_and_dropped_values(dev):
    x = torch.full((1000,), math.nan, device=dev)
    assert torch.count_nonzero(F.dropout(x, 1.0, 5)) == 0
    x = randn((1000,), torch.float32, 1).to(dev)
    assert torch.equal(F.dropout(x, 0.0, 5), x)
    assert F.dropout(x[:0], 0.5, 5).shape == (0,)
    keep = keep_reference(1000, 0.5, 5, 0)
    y = F.dropout(torch.where(keep.to(dev), x, math.inf), 0.5, 5)
    assert y.isfinite().all() and torch.equal((y == 0).cpu(), ~keep)
    # seeds and offsets make other masks; their share of kept values is binomial: within 6 deviations
    n = 1 << 20
    ones = torch.ones(n, device=dev)
    masks = [F.dropout(ones, 0.25, s, o) != 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 << 32, 0), (1, 1 << 32))]
    for i, m in enumerate(masks):
        assert abs(int(m.sum()) - 0.75 * n) < 6 * (n * 0.1875) ** 0.5
        for q in masks[:i]:
            assert abs(int((m & q).sum()) - 0.5625 * n) < 6 * (n * 0.25) ** 0.5


# ---------------------------------------------------------------------------
# gradients against differences, refusals
# ---------------------------------------------------------------------------
def test_gradients_against_differences(dev):
    """A directional derivative of each operator in fp32: central differences of
    step 2^-6.  The operators are linear in each leaf or smooth with third
    derivatives of the size of the function, so that the differences are off by
    step^2 and by the outputs' rounding over the step."""
    step = 2.0 ** -6
    routes = F.route_experts(randn((40, 6), torch.float32, 1).to(dev), 2)

    def check(f, *leaves):
        leaves = [t.to(dev).requires_grad_(True) for t in leaves]
        y = f(*leaves)
        c = randn(tuple(y.shape), torch.float32, 50).to(dev)
        grads = torch.autograd.grad(y, leaves, c)
        for i, (leaf, g) in enumerate(zip(leaves, grads)):
            v = randn(tuple(leaf.shape), torch.float32, 60 + i).to(dev)
            with torch.no_grad():
                moved = [f(*(t + s * step * v if j == i else t for j, t in enumerate(leaves))).double() for s in (1, -1)]
            terms = c.double() * (moved[0] - moved[1]) / (2 * step)
            size = terms.abs().sum() + (c.double() * moved[0]).abs().sum()
            assert abs(terms.sum() - (g.double() * v.double()).sum()) <= (4 * step ** 2 + 2.0 ** -20 / step) * size, i

    check(lambda x, w, b: F.grouped_linear(x, w, routes, bias=b), randn((40, 20), torch.float32, 2),
          randn((6, 20, 12), torch.float32, 3, 0.2), randn((6, 12), torch.float32, 4))
    check(lambda h, w: F.combine_experts(h, routes._replace(weights=w)), randn((80, 20), torch.float32, 5),
          routes.weights.cpu())
    # (logits far enough apart that a step changes no choice)
    logits = torch.stack([torch.randperm(6, generator=torch.Generator().manual_seed(i)) for i in range(40)]).float() * 0.5
    check(lambda l: F.route_experts(l, 6).weights, logits)
    check(lambda l: F.route_experts(l, 6, renormalize=False).weights, logits)
    for sigmoid in (False, True):
        check(lambda x, h, w, g, wn: torch.cat(F.gated_residual_norm(x, h, weight=w, gate=g, gate_sigmoid=sigmoid,
                                                                     scale=0.7, next_weight=wn)),
              *(randn(s, torch.float32, 7 + i) for i, s in enumerate(((30, 24), (30, 24), (24,), (30, 24), (24,)))))
    check(lambda x, r: F.dropout(x, 0.3, 9, residual=r), randn((30, 7), torch.float32, 20), randn((30, 7), torch.float32, 21))


def test_views_orders_and_other_streams(dev):
    """Transposed and strided arguments, and calls on a stream of their own."""
    x = randn((64, 90), torch.float16, 1).to(dev).t()[::2, :]  # [45, 64], neither order contiguous
    w = randn((3, 40, 64), torch.float16, 2, 0.1).to(dev).transpose(1, 2)
    offsets = torch.tensor([0, 9, 0, 9, 30, 9, 45, 9], dtype=torch.int32, device=dev)[::2]
    assert offsets.tolist() == [0, 0, 30, 45]
    y = F.grouped_linear(x, w, offsets)
    assert torch.equal(y, F.grouped_linear(x.contiguous(), w.contiguous(), offsets.contiguous()))
    assert torch.equal(F.rms_norm(x, x[0]), F.rms_norm(x.contiguous(), x[0].contiguous()))
    assert torch.equal(F.dropout(x, 0.5, 1), F.dropout(x.contiguous(), 0.5, 1))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        logits = (x @ w[0]).float()
        r = F.route_experts(logits, 2)
        h = F.grouped_linear(x, randn((40, 64, 32), torch.float16, 3, 0.1).to(dev), r)
        z = F.combine_experts(h, r)
    torch.cuda.current_stream().wait_stream(stream)
    again = F.route_experts(logits, 2)
    assert all(torch.equal(a, b) for a, b in zip(r, again))
    assert torch.equal(z, F.combine_experts(h, r))


def test_refusals(dev):
    f16, f32 = torch.float16, torch.float32
    x, w = torch.zeros(10, 16, device=dev, dtype=f16), torch.zeros(3, 16, 8, device=dev, dtype=f16)
    off = torch.tensor([0, 3, 6, 10], dtype=torch.int32, device=dev)
    routes = F.route_experts(torch.zeros(10, 3, device=dev), 2)

    def refused(f, match=r"\[Spira\]"):
        with pytest.raises(RuntimeError, match=match):
            f()

    refused(lambda: F.grouped_linear(x, w.float(), off))                       # other types
    refused(lambda: F.grouped_linear(x.double(), w.double(), off), "dtype")    # a type without a kernel
    refused(lambda: F.grouped_linear(x, w[:, :8], off), "shape")               # other widths
    refused(lambda: F.grouped_linear(x, w, off.long()), "offsets")             # offsets of another type
    refused(lambda: F.grouped_linear(x, w, off[:3]), "offsets")                # groups without weights
    refused(lambda: F.grouped_linear(x, w, off.cpu()), "offsets")              # on another device
    refused(lambda: F.grouped_linear(x, w, off, bias=torch.zeros(8, device=dev, dtype=f16)), "bias")
    refused(lambda: F.grouped_linear(x[:9], w, routes), "do not fit")          # routes of other tokens
    refused(lambda: F.grouped_linear(x[0], w, off), "features")
    refused(lambda: F.route_experts(x, 0), "choices")
    refused(lambda: F.route_experts(x, 17), "choices")
    refused(lambda: F.route_experts(torch.zeros(2, 600, device=dev), 2), "experts")
    refused(lambda: F.route_experts(torch.zeros(2, 4, device=dev, dtype=torch.int32), 2), "dtype")
    refused(lambda: F.combine_experts(torch.zeros(20, 8, device=dev), routes._replace(weights=routes.weights.half())))
    refused(lambda: F.gated_residual_norm(x, x[:5]), "update")
    refused(lambda: F.gated_residual_norm(x, x, weight=torch.zeros(16, device=dev, dtype=f32)), "weight")
    refused(lambda: F.gated_residual_norm(x, x, gate=torch.zeros(10, device=dev, dtype=f16)), "gate")
    refused(lambda: F.gated_residual_norm(x, x, gate=torch.zeros(5, 16, device=dev, dtype=f16)), "gate")
    refused(lambda: F.rms_norm(torch.zeros(1, 16385, device=dev), torch.zeros(16385, device=dev)), "channels")
    refused(lambda: F.dropout(x, 1.5, 0), "p must be")
    refused(lambda: F.dropout(x, math.nan, 0), "p must be")
    refused(lambda: F.dropout(x, 0.5, 0, residual=x[:5]), "residual")
    for f in (lambda: F.grouped_linear(x.cpu(), w.cpu(), off.cpu()), lambda: F.route_experts(x.cpu(), 2),
              lambda: F.rms_norm(x.cpu(), x[0].cpu()), lambda: F.dropout(x.cpu(), 0.5, 0)):
        with pytest.raises(NotImplementedError):
            f()
