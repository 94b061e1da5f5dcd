"""Attention over packed sequences against its formulas in 64 bits.

Tolerances follow from the arithmetic.  u is half a step of the features' type:
2^-11 (fp16), 2^-8 (bf16), 2^-24 (fp32); e = 2^-24 is that of the sums.

* a score is off by at most es = scale (D + 16) e sum |q||k| + 4 e |s|, so a
  weight p by the relative w = 2 max es + 2 (n + 16) e (its exponential, the
  running sum of n terms); in 16 bits it is rounded before its product, by u more
  (fp16 numbers below 2^-14 by 2^-25 as they are, under a sum of at least 1); a
  weight or a ds below 2^-126 is no normal number of fp32, in which it is held, and
  may be 0: 2^-126 of each term;
* o: u |o| + sum (w + u) p |v|;
* ds = p (dp - delta): delta has the rounded o (sum |do| tol(o)), dp a sum of D
  terms; then ds is rounded as p is;
* gradients: u of the value and the terms' errors, by the sums' own formulas."""
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


def offsets_of(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int32).cumsum(0, dtype=torch.int32)


def reference(q, k, v, q_at, k_at, causal, scale, dout=None):
    """(values, tolerances) of o and, with dout, dq, dk, dv; q_at, k_at: a sequence's (first, number)."""
    dt = q.dtype
    u, low = UNIT[dt], 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126
    pu = u if dt != torch.float32 else 0.0
    q, k, v = q.double(), k.double(), v.double()
    out = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    tol = [torch.full_like(t, TINY[dt]) for t in out]
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    for (q0, nq), (k0, nk) in zip(q_at, k_at):
        if nq == 0 or nk == 0:
            continue
        rows, cols = slice(q0, q0 + nq), slice(k0, k0 + nk)
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(nk - nq)
        some = seen.any(1, keepdim=True)
        for h in range(q.shape[1]):
            x, y, z = q[rows, h], k[cols, h // group], v[cols, h // group]
            s = torch.where(seen, scale * (x @ y.t().contiguous()), -math.inf)
            es = scale * (d + 16) * E * (x.abs() @ y.abs().t().contiguous()) + 4 * E * s.abs()
            w = 2 * torch.where(seen, es, 0).amax(1, keepdim=True) + 2 * (nk + 16) * E
            p = torch.where(some, torch.softmax(torch.where(some, s, 0), 1), 0)
            ep = (w + pu) * p + low * seen
            o = p @ z
            to = u * o.abs() + ep @ z.abs()
            out[0][rows, h], tol[0][rows, h] = o, tol[0][rows, h] + to
            if dout is None:
                continue
            g = dout[rows, h].double()
            dp, delta = g @ z.t().contiguous(), (g * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            edp = (d + 16) * E * (g.abs() @ z.abs().t().contiguous() + (g * o).abs().sum(1, keepdim=True))
            edp = edp + (g.abs() * to).sum(1, keepdim=True)
            eds = pu * ds.abs() + w * ds.abs() + p * (1 + w) * edp + low * seen
            pt, dst, ept, edst = (t.t().contiguous() for t in (p, ds, ep, eds))
            n = 2 * (max(nq * group, nk) + 16) * E  # (the long sums' own error)
            for i, value, size, error in (
                    (1, scale * ds @ y, scale * ds.abs() @ y.abs(), scale * eds @ y.abs()),
                    (2, scale * dst @ x, scale * dst.abs() @ x.abs(), scale * edst @ x.abs()),
                    (3, pt @ g, pt @ g.abs(), ept @ g.abs())):
                at = (rows, h) if i == 1 else (cols, h // group)
                out[i][at] += value
                tol[i][at] += error + n * size
    if dout is not None:
        for i in (1, 2, 3):
            tol[i] += u * out[i].abs()
    return out, tol


def close(got, ref, tol, what):
    bad = ~((got.detach().double() - ref).abs() <= tol * 1.001)
    assert got.shape == ref.shape and not bad.any(), (
        what, int(bad.sum()), torch.nonzero(bad)[0].tolist(), got[bad][0].item(), ref[bad][0].item(), tol[bad][0].item())


def check(dev, q, k, v, q_lengths, *, k_lengths=None, counts=None, causal, scale=None, train=True, dout=None):
    """A call, and with `train` its gradients, against the reference."""
    offsets = offsets_of(q_lengths)
    key_offsets = None if k_lengths is None else offsets_of(k_lengths)
    by = q.shape[2] ** -0.5 if scale is None else scale
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    starts = (offsets if key_offsets is None else key_offsets).tolist()
    room = q_lengths if k_lengths is None else k_lengths
    used = room if counts is None else counts
    dout = dout if dout is not None else randn(q.shape, q.dtype, 9)
    dout = dout.to(dev) if train else None
    ref, tol = reference(q, k, v, list(zip(offsets.tolist(), q_lengths)), list(zip(starts, used)), causal, by, dout)
    kw = dict(key_offsets=None if key_offsets is None else key_offsets.to(dev),
              key_counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev),
              causal=causal, scale=scale)
    with torch.no_grad():
        y = F.attention(q, k, v, offsets.to(dev), **kw)
        again = F.attention(q, k, v, offsets.to(dev), **kw)
    close(y, ref[0], tol[0], "o")
    assert torch.equal(y, again)
    if not train:
        return y
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = F.attention(*leaves, offsets.to(dev), **kw)
    close(y, ref[0], tol[0], "o with gradients")
    grads = torch.autograd.grad(y, leaves, dout)
    for i, name in enumerate(("dq", "dk", "dv")):
        close(grads[i], ref[i + 1], tol[i + 1], name)
    y2 = F.attention(*leaves, offsets.to(dev), **kw)
    for a, b in zip(grads, torch.autograd.grad(y2, leaves, dout)):
        assert torch.equal(a, b)
    return y


LENGTHS = [
    # sequences' lengths, query heads, key heads, values
    ([1], 1, 1, 16), ([1, 1, 1], 2, 1, 64), ([5, 0, 17, 64], 2, 2, 32), ([130], 4, 2, 64), ([33, 0, 0, 95, 128], 6, 2, 128),
    ([257, 63], 3, 1, 96), ([200, 31, 32], 4, 4, 36), ([70, 3], 2, 1, 1), ([65, 66], 5, 1, 63), ([300], 2, 2, 80),
    ([64, 128], 8, 1, 128), ([90, 0], 2, 2, 7), ([0, 0], 2, 1, 32), ([1, 2, 3] * 30, 4, 2, 40), ([700], 2, 1, 127)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,heads,kv,d", LENGTHS)
def test_sequences(dev, lengths, heads, kv, d, causal, dtype):
    n, dt = sum(lengths), DTYPES[dtype]
    check(dev, randn((n, heads, d), dt, 1), randn((n, kv, d), dt, 2), randn((n, kv, d), dt, 3), lengths, causal=causal)


@pytest.mark.parametrize("causal", [False, True])
def test_many_sequences(dev, causal):
    """More than a wave looks at at once, of uneven lengths and none: themselves, and a token each
    against caches in parts."""
    lengths = [(i * 7) % 11 for i in range(700)]
    n = sum(lengths)
    check(dev, randn((n, 2, 16), torch.float16, 1), randn((n, 1, 16), torch.float16, 2), randn((n, 1, 16), torch.float16, 3),
          lengths, causal=causal)
    room = [(i * 37) % 300 for i in range(300)]
    m = sum(room)
    check(dev, randn((300, 2, 16), torch.float16, 1), randn((m, 1, 16), torch.float16, 2), randn((m, 1, 16), torch.float16, 3),
          [1] * 300, k_lengths=room, causal=causal)


def test_thousands_of_sequences(dev):
    """More than 64 times 64 of them, each found in three steps, some with nothing; in windows, and a
    token each against caches of few keys and of more room."""
    lengths = [(i * 5) % 8 if i % 9 else 0 for i in range(4500)]
    n = sum(lengths)
    check(dev, randn((n, 1, 8), torch.float16, 1), randn((n, 1, 8), torch.float16, 2), randn((n, 1, 8), torch.float16, 3),
          lengths, causal=True)
    room = [(i * 37) % 20 for i in range(4500)]
    m = sum(room)
    check(dev, randn((4500, 1, 8), torch.float16, 1), randn((m, 1, 8), torch.float16, 2), randn((m, 1, 8), torch.float16, 3),
          [1] * 4500, k_lengths=room, counts=[r // 2 for r in room], causal=False)


@pytest.mark.parametrize("dtype,causal", [("f16", False), ("bf16", True)])
def test_a_long_sequence(dev, dtype, causal):
    """Weights of some 1e-4 each, many tiles, and parts of the keys' steps."""
    dt, n = DTYPES[dtype], 9001
    check(dev, randn((n, 2, 24), dt, 1), randn((n, 1, 24), dt, 2), randn((n, 1, 24), dt, 3), [n], causal=causal)


CROSS = [
    # queries, keys (room), keys in use, heads, key heads, values
    ([1, 1], [40, 700], None, 8, 2, 64), ([1] * 5, [300, 64, 128, 1024, 70], [299, 0, 128, 1000, 1], 4, 1, 128),
    ([3, 2, 0, 9], [20, 1, 5, 9], [20, 1, 5, 4], 4, 2, 32),          # (more queries than keys: some see none)
    ([40, 100], [2, 1300], None, 2, 2, 36), ([1], [5000], [4993], 16, 2, 96), ([2] * 40, [100] * 40, [97] * 40, 2, 1, 64),
    ([1, 1, 1], [3000, 0, 50], [2990, 0, 50], 3, 3, 63), ([150], [400], None, 4, 2, 64), ([7], [0], None, 2, 1, 32),
    ([1] * 70, [100] * 70, [99] * 70, 2, 1, 40), ([70], [9000], [8999], 8, 1, 64), ([40, 33], [4100, 5000], None, 4, 2, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,room,used,heads,kv,d", CROSS)
def test_keys_of_their_own(dev, queries, room, used, heads, kv, d, causal, dtype):
    """A cache: keys longer or shorter than the queries, with room behind them that holds NaN."""
    n, m, dt = sum(queries), sum(room), DTYPES[dtype]
    k, v = randn((m, kv, d), dt, 2), randn((m, kv, d), dt, 3)
    if used is not None:
        at = 0
        for r, c in zip(room, used):
            k[at + c:at + r], v[at + c:at + r] = math.nan, math.inf
            at += r
    check(dev, randn((n, heads, d), dt, 1), k, v, queries, k_lengths=room, counts=used, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale,size", [(2.0, 3.0), (1e-3, 1.0), (30.0, 4.0)])
def test_scores_far_apart(dev, scale, size, dtype):
    """From even weights to one that takes all, with scores that rise along the keys (the running maximum moves)."""
    dt, n, d = DTYPES[dtype], 400, 32
    q, v = randn((n, 2, d), dt, 1, size), randn((n, 1, d), dt, 3)
    k = (randn((n, 1, d), torch.float32, 2) * torch.linspace(0.01, 1, n)[:, None, None] * size).to(dt)
    check(dev, q, k, v, [150, 250], causal=True, scale=scale / 10)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["projection", "heads first", "odd start", "expanded", "columns"])
def test_strides(dev, layout, dtype):
    dt, n, h, hk, d = DTYPES[dtype], 190, 4, 2, 64
    x = randn((n, h + 2 * hk, d), dt, 1)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    if layout == "heads first":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    elif layout == "odd start":
        flat = torch.cat([torch.zeros(3, dtype=dt), x.reshape(-1)]).to(dev)[3:].view(x.shape)
        q, k, v = flat[:, :h], flat[:, h:h + hk], flat[:, h + hk:]
    elif layout == "expanded":
        k, v = k[:, :1].to(dev).expand(-1, hk, -1), v[:1].to(dev).expand(n, -1, -1)
    elif layout == "columns":
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "projection":
        x = x.to(dev)
        q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    check(dev, q, k, v, [100, 90], causal=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["key", "value", "query", "gradient"])
@pytest.mark.parametrize("d", [64, 128, 36])
def test_not_finite_where_hidden(dev, what, d, dtype):
    """NaN and infinities late in a sequence leave the rows that do not see them as they are, forward
    and in the gradients, with their own tile's rows among them."""
    dt, n, at = DTYPES[dtype], 200, 150
    q, k, v = randn((n, 4, d), dt, 1), randn((n, 2, d), dt, 2), randn((n, 2, d), dt, 3)
    dout = randn((n, 4, d), dt, 9)
    offsets = torch.tensor([0, n], dtype=torch.int32, device=dev)

    def run(*ts):
        leaves = [t.to(dev).requires_grad_(True) for t in ts[:3]]
        y = F.attention(*leaves, offsets, causal=True)
        with torch.no_grad():
            assert torch.equal(F.attention(*leaves, offsets, causal=True)[:at], y[:at])
        return (y, *torch.autograd.grad(y, leaves, ts[3].to(dev)))
    clean = run(q, k, v, dout)
    dirty = [t.clone() for t in (q, k, v, dout)]
    t = dirty[{"query": 0, "key": 1, "value": 2, "gradient": 3}[what]]
    t[at, :, ::3], t[at + 1, :, 1], t[at + 7, :, :] = math.nan, math.inf, -math.inf
    got = run(*dirty)
    if what in ("key", "value"):  # hidden from the queries before them
        assert torch.equal(got[0][:at], clean[0][:at]) and torch.equal(got[1][:at], clean[1][:at])
        assert torch.isnan(got[0][at]).any() and not torch.isfinite(got[0][at + 8:]).all(2).any()
    else:  # what those give to the keys behind them: nothing
        last = at + 8
        assert torch.equal(got[2][last:], clean[2][last:]) and torch.equal(got[3][last:], clean[3][last:])
        assert not torch.isfinite(got[3][:at]).all(2).any()


def test_infinite_values_reach_the_rows_that_see_them(dev):
    """An infinite value is the output of the rows that see it, under weights that are all positive."""
    n, d = 100, 32
    q, k, v = (randn((n, 1, d), torch.float32, i, 0.1).to(dev) for i in (1, 2, 3))
    v[70, 0, 5], v[70, 0, 6] = math.inf, -math.inf
    y = F.attention(q, k, v, torch.tensor([0, n], dtype=torch.int32, device=dev), causal=True)
    assert torch.isfinite(y[:70]).all()
    assert (y[70:, 0, 5] == math.inf).all() and (y[70:, 0, 6] == -math.inf).all()
    assert torch.isfinite(y[70:, 0, 7:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_sequence(dev, dtype):
    """Zeros before the first sequence and behind the last, in outputs and gradients."""
    dt, n = DTYPES[dtype], 300
    leaves = [randn((n, h, 32), dt, i).to(dev).requires_grad_(True) for i, h in ((1, 4), (2, 2), (3, 2))]
    for lo, mid, hi in ((40, 100, 250), (0, 0, 0), (299, 300, 300)):
        offsets = torch.tensor([lo, mid, hi], dtype=torch.int32, device=dev)
        y = F.attention(*leaves, offsets, causal=False)
        grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
        with torch.no_grad():
            plain = F.attention(*leaves, offsets, causal=False)
        ref, tol = reference(*(t.detach() for t in leaves), [(lo, mid - lo), (mid, hi - mid)],
                             [(lo, mid - lo), (mid, hi - mid)], False, 32 ** -0.5)
        for t in (y, plain, *grads):
            assert torch.count_nonzero(t[:lo]) == 0 and torch.count_nonzero(t[hi:]) == 0
        close(plain, ref[0], tol[0], "o")


def test_offsets_that_are_no_rows(dev):
    """Whatever the numbers are, nothing outside the tensors is touched, and the calls return."""
    q, k = randn((50, 2, 32), torch.float16, 1).to(dev), randn((60, 1, 32), torch.float16, 2).to(dev)
    for a, b, c in (([0, -5, 99], [0, 30, 2 ** 31 - 1], [1000, -3]), ([2 ** 31 - 1, 3, 50], [-2 ** 31, 61, 20], [5, 5])):
        offsets, keys, counts = (torch.tensor(t, dtype=torch.int32, device=dev) for t in (a, b, c))
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, k)]
        y = F.attention(*leaves, offsets, key_offsets=keys, key_counts=counts, causal=True)
        torch.autograd.grad(y, leaves, torch.ones_like(y))
        with torch.no_grad():
            F.attention(q, k, k, offsets, key_offsets=keys, key_counts=counts)
    torch.cuda.synchronize()


def test_offsets_past_32_bits(dev):
    """Sequences at the end of a cache of more than 2^32 bytes, and rows 32 MB apart: what the same rows
    give close together."""
    d, lengths = 64, [300, 200]
    n = sum(lengths)
    q, k, v = (randn((n, h, d), torch.float16, i).to(dev) for i, h in ((1, 2), (2, 1), (3, 1)))
    at, dout = offsets_of(lengths), randn((n, 2, d), torch.float16, 4).to(dev)
    far = 34_000_000
    big = [torch.empty(far, 1, d, dtype=torch.float16, device=dev) for _ in range(2)]
    wide = [torch.empty(n, 1 << 24, dtype=torch.float16, device=dev)[:, None, :d] for _ in range(2)]
    for t, x in zip((*big, *wide), (k, v, k, v)):
        t[-n:] = x
    offsets = at.to(dev)
    for causal in (False, True):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        ref = F.attention(*leaves, offsets, causal=causal)
        grads = torch.autograd.grad(ref, leaves, dout)
        for keys, first in ((big, far - n), (wide, 0)):
            moved = [q.detach().requires_grad_(True), *(t.detach().requires_grad_(True) for t in keys)]
            kw = dict(key_offsets=(at + first).to(dev), causal=causal)
            y = F.attention(*moved, offsets, **kw)
            got = torch.autograd.grad(y, moved, dout)
            assert torch.equal(y, ref) and torch.equal(got[0], grads[0])
            for a, b in zip(got[1:], grads[1:]):
                # (in how many parts a tile's steps are summed goes by the number of keys: 16 bits apart by a step)
                assert torch.allclose(a[-n:].float(), b.float(), rtol=2.0 ** -10, atol=1e-4)
                assert torch.count_nonzero(a[:-n]) == 0
            del y, got, moved
            last = torch.tensor([n - 1, n], dtype=torch.int32, device=dev)  # one token, in parts
            ends = torch.tensor([first + 300, first + n], dtype=torch.int32, device=dev)
            with torch.no_grad():
                one = F.attention(q[-1:], *keys, last - (n - 1), key_offsets=ends, causal=causal)
            assert torch.allclose(one.float(), ref[-1:].float(), rtol=2.0 ** -9, atol=2e-3)


def test_gradients_by_differences(dev):
    """Central differences of sum(w o) along random directions in fp32: their own error is a
    third derivative's h^2 (h = 2^-6, some 1e-4 of the value) and the outputs' rounding, 2^-24 of 200 terms
    over h."""
    n, d = 24, 16
    ts = [randn((n, h, d), torch.float32, i, 0.5).to(dev) for i, h in ((1, 4), (2, 2), (3, 2))]
    w = randn((n, 4, d), torch.float32, 4).to(dev)
    offsets = torch.tensor([0, 10, n], dtype=torch.int32, device=dev)
    leaves = [t.clone().requires_grad_(True) for t in ts]
    grads = torch.autograd.grad(F.attention(*leaves, offsets, causal=True), leaves, w)
    h = 2.0 ** -6
    for i in range(3):
        way = randn(ts[i].shape, torch.float32, 20 + i).to(dev)
        value = []
        for sign in (1, -1):
            moved = list(ts)
            moved[i] = ts[i] + sign * h * way
            value.append((F.attention(*moved, offsets, causal=True).double() * w.double()).sum().item())
        along = (grads[i].double() * way.double()).sum().item()
        scale = (grads[i].double().abs() * way.double().abs()).sum().item()
        assert abs((value[0] - value[1]) / (2 * h) - along) < 2e-3 * scale, i


@pytest.mark.parametrize("need", range(1, 8))
def test_some_gradients(dev, need):
    """Those that are asked for, as all of them together."""
    ts = [randn((90, h, 40), torch.bfloat16, i).to(dev) for i, h in ((1, 4), (2, 2), (3, 2))]
    offsets = torch.tensor([0, 50, 90], dtype=torch.int32, device=dev)
    dout = randn((90, 4, 40), torch.bfloat16, 5).to(dev)
    leaves = [t.clone().requires_grad_(True) for t in ts]
    ref = torch.autograd.grad(F.attention(*leaves, offsets, causal=True), leaves, dout)
    some = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate(ts)]
    got = torch.autograd.grad(F.attention(*some, offsets, causal=True), [t for t in some if t.requires_grad], dout)
    for a, b in zip(got, [r for i, r in enumerate(ref) if need >> i & 1]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens", [True, False])
def test_captured_in_a_graph(dev, tokens):
    """Replays on new features, lengths and counts equal the eager calls, with eager work between them."""
    n, m = (4, 6000) if tokens else (300, 300)
    q, k, v = (randn((r, h, 64), torch.float16, i).to(dev) for i, (r, h) in enumerate(((n, 4), (m, 2), (m, 2))))
    offsets = torch.tensor([0, n // 2, n], dtype=torch.int32, device=dev)
    keys = torch.tensor([0, m // 2, m], dtype=torch.int32, device=dev)
    counts = torch.tensor([m // 2, m // 2], dtype=torch.int32, device=dev)

    def call():
        return F.attention(q, k, v, offsets, key_offsets=keys, key_counts=counts, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for i in range(4):
        q.copy_(randn(q.shape, q.dtype, 30 + i))
        counts.copy_(torch.tensor([m // 2 - 7 * i, 11 * i]))
        graph.replay()
        got = y.clone()
        assert torch.equal(got, call()), i
        torch.cuda.synchronize()


def test_two_calls_on_two_streams(dev):
    q, k, v = (randn((r, h, 128), torch.bfloat16, i).to(dev) for i, (r, h) in enumerate(((8, 8), (20000, 2), (20000, 2))))
    offsets = torch.arange(9, dtype=torch.int32, device=dev)
    keys = torch.arange(9, dtype=torch.int32, device=dev) * 2500
    ref = F.attention(q, k, v, offsets, key_offsets=keys)
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                out.append(F.attention(q, k, v, offsets, key_offsets=keys))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in out)


def test_refusals(dev):
    q, k = torch.zeros(8, 4, 16, device=dev), torch.zeros(8, 2, 16, device=dev)
    off = torch.tensor([0, 8], dtype=torch.int32, device=dev)

    def refused(text, *args, **kw):
        with pytest.raises(RuntimeError, match=r"\[Spira\].*" + text):
            F.attention(*args, **kw)
    refused("rows, heads", q[0], k, k, off)
    refused("multiple", q[:, :3], k, k, off)
    refused("1 to 128", torch.zeros(8, 4, 129, device=dev), torch.zeros(8, 2, 129, device=dev),
            torch.zeros(8, 2, 129, device=dev), off)
    refused("heads of 16", q, k[:, :, :8], k[:, :, :8], off)
    refused("shape", q, k, k[:4], off)
    refused("must be Float", q, k.half(), k, off)
    refused("dtype", q.double(), k.double(), k.double(), off)
    refused("Int", q, k, k, off.long())
    refused(r"sequences \+ 1", q, k, k, off[:1])
    refused("key_offsets must have the shape", q, k, k, off, key_offsets=torch.zeros(3, dtype=torch.int32, device=dev))
    refused("key_counts must have the shape", q, k, k, off, key_counts=off)
    refused("as many as the queries", q, k[:4], k[:4], off)
    refused("as many as the queries", q, k[:4], k[:4], off, key_counts=off[1:])
    refused("must be a GPU tensor", q, k.cpu(), k, off)
    refused("must be a GPU tensor", q, k, k, off.cpu())
    for scale in (0.0, -1.0, math.inf, math.nan):
        refused("scale", q, k, k, off, scale=scale)
    x = q.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(F.attention(x, k, k, off).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        d.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        refused("forward mode", torch.autograd.forward_ad.make_dual(q, q), k, k, off)
