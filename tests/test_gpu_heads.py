"""Norms and rotation of attention's heads, and the router's balance loss, against
their formulas in 64 bits.

Tolerances follow from the arithmetic, with u half a step of the features' type
and e = 2^-24.  Heads: a normed value is off by (D + 24) e of itself (the mean of D
squares, its inverse root, three products), a turned pair by that and 6 e of the pair's size (its sines, two
products, a sum); the output rounds once.  The gradients' sums over D, and those of
the weights over N rows, by n e of their terms' sizes."""
import math

import pytest
import torch

from spira_amd.nn import functional as F

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}
E = 2.0 ** -24


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def close(got, ref, error, what):
    tol = UNIT[got.dtype] * ref.abs() * 1.001 + error + TINY[got.dtype]
    got = got.detach().double()
    bad = ~((got - ref).abs() <= tol)
    assert got.shape == ref.shape and not bad.any(), (
        what, int(bad.sum()), torch.nonzero(bad)[0].tolist(), got[bad][0].item(), ref[bad][0].item(), tol[bad][0].item())


def angles(positions, d, base):
    """[N, 1, D / 2] in 64 bits."""
    at = positions.double() if positions.dim() == 2 else positions.double()[:, None]
    pairs, axes = d // 2, at.shape[1]
    columns = []
    for a in range(axes):
        lo, hi = a * pairs // axes, (a + 1) * pairs // axes
        columns += [at[:, a] * base ** (-j / (hi - lo)) for j in range(hi - lo)]
    return torch.stack(columns, 1)[:, None]


def pairs_of(x, interleaved):
    half = (x.shape[-1] + 1) // 2
    return (x[..., ::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])


def joined(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def turn(x, t, interleaved):
    if t is None:
        return x
    a, b = pairs_of(x, interleaved)
    return joined(a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos(), interleaved)


def size(x, t, interleaved):
    """Of a value's pair."""
    if t is None:
        return x.abs()
    a, b = pairs_of(x, interleaved)
    s = a.abs() + b.abs()
    return joined(s, s, interleaved)


def one_side(x, w, t, g, eps, interleaved):
    """Per output: (value, error): y, dx, dw."""
    d = x.shape[-1]
    x, g = x.double(), g.double()
    inv = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) if w is not None else 1.0
    hat = x * inv
    n = hat * w.double() if w is not None else hat
    c = (d + 24) * E
    y = turn(n, t, interleaved)
    ey = (c + 6 * E) * size(n, t, interleaved)
    back, eb = turn(g, None if t is None else -t, interleaved), 6 * E * size(g, t, interleaved)
    if w is None:
        return (y, ey), (back, eb), None
    dn = back * w.double()
    en = (eb + 2 * E * back.abs()) * w.double().abs()
    mean, sizes = (dn * hat).mean(-1, keepdim=True), (dn * hat).abs().mean(-1, keepdim=True)
    dx = inv * (dn - hat * mean)
    ex = inv * (en + hat.abs() * ((en * hat.abs()).mean(-1, keepdim=True) + 4 * c * sizes) + 4 * c * (dn.abs() + hat.abs() * sizes))
    rows = x.shape[0] * x.shape[1]
    dw = (back * hat).sum((0, 1))
    ew = (eb * hat.abs() + c * (back * hat).abs()).sum((0, 1)) + 2 * (rows + 16) * E * (back * hat).abs().sum((0, 1))
    return (y, ey), (dx, ex), (dw, ew)


HEADS = [
    # rows, heads, key heads, values, axes, farthest position
    (1, 1, 1, 2, 1, 10), (8, 8, 2, 64, 1, 1_000_000), (300, 3, 3, 32, 3, 1000), (65, 4, 1, 128, 1, 2 ** 31 - 1),
    (33, 2, 2, 36, 2, 100), (7, 5, 3, 16, 8, 77), (0, 2, 1, 32, 1, 5), (100, 2, 1, 7, 0, 0), (40, 1, 2, 1, 0, 0),
    (29, 3, 1, 127, 0, 0), (5000, 4, 2, 96, 3, 4000), (31, 2, 1, 10, 5, 50), (3, 40, 40, 80, 1, 9)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,kv,d,axes,far", HEADS)
def test_norm_rotate_heads(dev, n, heads, kv, d, axes, far, interleaved, weighted, dtype):
    dt = DTYPES[dtype]
    x = randn((n, heads + 2 * kv, d), dt, 1, 1.5).to(dev)
    leaves = [x[:, :heads].detach().requires_grad_(True), x[:, heads:heads + kv].detach().requires_grad_(True)]
    weights = [(1 + randn((d,), torch.float32, i, 0.2)).to(dt).to(dev).requires_grad_(True) for i in (2, 3)]
    positions = t = None
    if axes:
        g = torch.Generator().manual_seed(4)
        positions = torch.randint(-far, far, (n, axes) if axes > 1 else (n,), generator=g, dtype=torch.int32).to(dev)
        t = angles(positions, d, 100.0)
    w = weights if weighted else [None, None]
    grads = [randn((n, h, d), dt, i).to(dev) for i, h in ((5, heads), (6, kv))]
    kw = dict(query_weight=w[0], key_weight=w[1], positions=positions, base=100.0, interleaved=interleaved)
    out = F.norm_rotate_heads(*leaves, **kw)
    got = torch.autograd.grad(out, leaves + (weights if weighted else []), grads)
    with torch.no_grad():
        for a, b in zip(out, F.norm_rotate_heads(*leaves, **kw)):
            assert torch.equal(a, b)
    for i in range(2):
        y, dx, dw = one_side(leaves[i].detach(), None if w[i] is None else w[i].detach(), t, grads[i], 1e-6, interleaved)
        close(out[i], *y, f"y {i}")
        close(got[i], *dx, f"dx {i}")
        if dw is not None:
            close(got[2 + i], *dw, f"dw {i}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_heads_strides(dev, dtype):
    """Views at any stride give what their copies give, forward and in the gradients."""
    dt, n, d = DTYPES[dtype], 77, 48
    x = randn((n, 6, d), dt, 1).to(dev)
    flat = torch.cat([torch.zeros(3, dtype=dt, device=dev), x.reshape(-1)])[3:].view(x.shape)
    w = randn((d,), dt, 2).to(dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    g = [randn((n, h, d), dt, 5 + h).to(dev) for h in (4, 2)]
    for v in (x, flat, x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2)):
        out = []
        for q, k in ((v[:, :4], v[:, 4:]), (v[:, :4].contiguous(), v[:, 4:].contiguous())):
            leaves = [q.detach().requires_grad_(True), k.detach().requires_grad_(True)]
            y = F.norm_rotate_heads(*leaves, query_weight=w, key_weight=w, positions=pos)
            out.append((*y, *torch.autograd.grad(y, leaves, [t.transpose(0, 1).contiguous().transpose(0, 1) for t in g])))
        assert all(torch.equal(a, b) for a, b in zip(*out))


def test_one_output_without_a_gradient(dev):
    q, k = (randn((20, h, 32), torch.float32, h).to(dev).requires_grad_(True) for h in (2, 1))
    wq, wk = (torch.ones(32, device=dev, requires_grad=True) for _ in range(2))
    a, _ = F.norm_rotate_heads(q, k, query_weight=wq, key_weight=wk)
    a.sum().backward()
    assert q.grad is not None and wq.grad is not None
    assert k.grad is None or torch.count_nonzero(k.grad) == 0
    assert wk.grad is None or torch.count_nonzero(wk.grad) == 0


def test_heads_gradient_by_differences(dev):
    """Central differences in fp32, h = 2^-7: h^2 of a third derivative, rounding over h."""
    ts = [randn((9, h, 12), torch.float32, h).to(dev) for h in (3, 2)] + [1 + randn((12,), torch.float32, i, 0.2).to(dev) for i in (7, 8)]
    pos = torch.arange(9, dtype=torch.int32, device=dev) * 5
    g = [randn((9, h, 12), torch.float32, 10 + h).to(dev) for h in (3, 2)]

    def call(ts):
        return F.norm_rotate_heads(ts[0], ts[1], query_weight=ts[2], key_weight=ts[3], positions=pos)
    leaves = [t.clone().requires_grad_(True) for t in ts]
    grads = torch.autograd.grad(call(leaves), leaves, g)
    h = 2.0 ** -7
    for i in range(4):
        way = randn(ts[i].shape, torch.float32, 20 + i).to(dev)
        value = []
        for sign in (1, -1):
            moved = list(ts)
            moved[i] = ts[i] + sign * h * way
            value.append(sum((y.double() * x.double()).sum().item() for y, x in zip(call(moved), g)))
        scale = (grads[i].double() * way.double()).abs().sum().item()
        assert abs((value[0] - value[1]) / (2 * h) - (grads[i].double() * way.double()).sum().item()) < 2e-3 * scale


def test_heads_refusals(dev):
    q, k = torch.zeros(8, 4, 16, device=dev), torch.zeros(8, 2, 16, device=dev)
    pos = torch.zeros(8, dtype=torch.int32, device=dev)

    def refused(text, *args, **kw):
        with pytest.raises(RuntimeError, match=r"\[Spira\].*" + text):
            F.norm_rotate_heads(*args, **kw)
    refused("rows, heads", q[0], k)
    refused("queries' rows", q, k[:4])
    refused("queries' rows", q, k[:, :, :8])
    refused("1 to 128", torch.zeros(2, 1, 130, device=dev), torch.zeros(2, 1, 130, device=dev))
    refused("even number", q[:, :, :15], k[:, :, :15], positions=pos)
    refused("axes", q, k, positions=torch.zeros(8, 9, dtype=torch.int32, device=dev))
    refused("Int", q, k, positions=pos.long())
    refused("shape", q, k, positions=pos[:4])
    refused("without an axis", q, k, positions=torch.zeros(8, 0, dtype=torch.int32, device=dev))
    refused("base", q, k, positions=pos, base=0.0)
    refused("query_weight must have", q, k, query_weight=torch.ones(8, device=dev))
    refused("key_weight must be Float", q, k, key_weight=torch.ones(16, device=dev).half())
    refused("must be Float", q, k.half())


# ---------------------------------------------------------------------------
# balance_loss
# ---------------------------------------------------------------------------
def routed(logits, k):
    """Offsets of the k largest, as a router gives them."""
    top, chosen = torch.topk(logits.float(), k, 1)
    chosen = torch.where(top > -math.inf, chosen, logits.shape[1])
    counts = torch.bincount(chosen.reshape(-1), minlength=logits.shape[1] + 1)[:-1]
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts,k,masked", [
    (1, 1, 1, 0), (8, 32, 2, 0), (0, 4, 1, 0), (700, 8, 1, 0.3), (3000, 16, 2, 0.1), (513, 512, 8, 0), (20_000, 3, 1, 0.6),
    (5, 17, 3, 1.0), (9000, 256, 8, 0.2), (4096, 511, 4, 0), (50_000, 64, 6, 0.1)])
def test_balance_loss(dev, tokens, experts, k, masked, dtype):
    """A probability is off by the relative c = (experts + 40) e (its exponential within 2 e and its
    argument's rounding, a sum, a division), sums over T tokens by T e more (less: they are trees)."""
    dt = DTYPES[dtype]
    logits = randn((tokens, experts), torch.float32, 1, 2.0)
    logits[torch.rand(logits.shape, generator=torch.Generator().manual_seed(2)) < masked] = -math.inf
    logits = logits.to(dt).to(dev)
    offsets = routed(logits, k)
    leaf = logits.clone().requires_grad_(True)
    r = F.balance_loss(leaf, offsets)
    by = 3000.0
    (d,) = torch.autograd.grad(r.loss, leaf, torch.tensor(by, device=dev))
    assert torch.equal(r.counts, offsets.diff()) and r.counts.dtype == torch.int32
    l = logits.double()
    some = (l > -math.inf).any(1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, l, 0), 1), 0)
    n = max(int(some.sum()), 1)
    share = offsets.diff().double() / max(int(offsets[-1]), 1)
    mean = p.sum(0) / n
    c = (experts + 60) * E
    many = c + (tokens / 64 + 40) * E
    close(r.probabilities, mean, many * mean, "probabilities")
    close(r.loss, experts * (share * mean).sum(), (many + 40 * E) * experts * (share * mean).sum(), "loss")
    along, sizes = (p * share).sum(1, keepdim=True), (p * share).sum(1, keepdim=True)
    close(d, by * experts / n * p * (share - along), by * experts / n * p * 4 * c * (share + sizes), "gradient")
    with torch.no_grad():
        again = F.balance_loss(logits, offsets)
    assert all(torch.equal(a, b) for a, b in zip(r, again))


def test_balance_loss_of_a_router(dev):
    """1 where all experts are used alike, and its gradient moves the router that way."""
    even = torch.eye(8, device=dev).repeat(100, 1) * 5
    r = F.balance_loss(even, F.route_experts(even, 1))
    assert abs(r.loss.item() - 1) < 1e-5 and (r.counts == 100).all()
    one = torch.zeros(64, 8, device=dev)
    one[:, 3] = 10
    leaf = one.clone().requires_grad_(True)
    r = F.balance_loss(leaf, F.route_experts(leaf, 1))
    assert r.loss.item() > 7.9
    r.loss.backward()
    assert (leaf.grad[:, 3] > 0).all() and (leaf.grad[:, :3] < 0).all()
    strided = one.t().contiguous().t()
    assert torch.equal(F.balance_loss(strided, F.route_experts(strided, 1)).loss, r.loss)


def test_balance_loss_of_nan(dev):
    """NaN is in the loss and in its token's gradient, not in the others'."""
    logits = randn((50, 6), torch.float32, 1).to(dev)
    logits[7, 2] = math.nan
    leaf = logits.clone().requires_grad_(True)
    r = F.balance_loss(leaf, torch.arange(0, 56, 8, dtype=torch.int32, device=dev))
    assert torch.isnan(r.loss) and torch.isnan(r.probabilities).all()
    r.loss.backward()
    assert torch.isnan(leaf.grad[7]).all() and torch.isfinite(leaf.grad[:7]).all() and torch.isfinite(leaf.grad[8:]).all()


def test_balance_refusals(dev):
    l, off = torch.zeros(8, 4, device=dev), torch.zeros(5, dtype=torch.int32, device=dev)

    def refused(text, *args):
        with pytest.raises(RuntimeError, match=r"\[Spira\].*" + text):
            F.balance_loss(*args)
    refused("1 to 512", torch.zeros(2, 513, device=dev), torch.zeros(514, dtype=torch.int32, device=dev))
    refused("offsets must have the shape", l, off[:4])
    refused("Int", l, off.long())
    refused("dtype", l.double(), off)
    refused("shape", l[0], off)
