"""Attention where its kernels' shortcuts end: values that are not finite behind the mask
(in narrow heads among others), rows that overlap, small weights and gradients in fp16, common
parts that cancel, large scores.  Units and
the reference are those of test_gpu_attention.py."""
import math

import pytest
import torch

from spira_amd.nn import functional as F
from test_gpu_attention import DTYPES, E, UNIT, check, offsets_of, randn

pytestmark = pytest.mark.gpu


def gradients(leaves, offsets, dout, **kw):
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    y = F.attention(*leaves, offsets, **kw)
    return (y.detach(), *torch.autograd.grad(y, leaves, dout))


# ---------------------------------------------------------------------------
# not finite behind the mask
# ---------------------------------------------------------------------------
def columns_fill_blocks(rows, heads, kv, sequences, dtype):
    """Whether a block owns 128 columns of queries (else 32): the kernels' own rule."""
    return (rows * (heads // kv) // 128 + sequences) * kv >= (512 if dtype == torch.float32 else 192)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["key", "value", "query", "gradient"])
@pytest.mark.parametrize("d", [8, 16, 32, 64, 100])
@pytest.mark.parametrize("many", [False, True])
def test_not_finite_where_hidden(dev, many, d, what, dtype):
    """NaN and infinities leave the rows that do not see them as they are, forward and in the gradients:
    for heads of every width of tile, in blocks of 32 columns and of 128."""
    dt = DTYPES[dtype]
    n, at, kv = (1000, 150, 32 if dtype == "f32" else 12) if many else (200, 150, 2)
    assert columns_fill_blocks(n, 2 * kv, kv, 1, dt) == many
    clean = [randn((n, h, d), dt, i).to(dev) for i, h in ((1, 2 * kv), (2, kv), (3, kv), (9, 2 * kv))]
    dirty = [t.clone() for t in clean]
    t = dirty[("query", "key", "value", "gradient").index(what)]
    t[at, :, ::3], t[at + 1, :, 1], t[at + 7] = math.nan, math.inf, -math.inf
    offsets = torch.tensor([0, n], dtype=torch.int32, device=dev)
    ref, got = (gradients(x[:3], offsets, x[3], causal=True) for x in (clean, dirty))
    assert all(torch.isfinite(r).all() for r in ref)
    if what in ("key", "value"):  # hidden from the queries before them
        assert torch.equal(got[0][:at], ref[0][:at]) and torch.equal(got[1][:at], ref[1][:at])
        assert torch.isnan(got[0][at]).any() and not torch.isfinite(got[0][at + 8:]).all(2).any()
    else:  # what those give to the keys behind them: nothing
        last = at + 8
        assert torch.equal(got[2][last:], ref[2][last:]) and torch.equal(got[3][last:], ref[3][last:])
        assert not torch.isfinite(got[3][:at]).all(2).any()


INFINITE = [
    # queries, keys (None: as many), heads, key heads, causal
    (1, 700, 8, 2, False), (1, 6000, 2, 1, True), (3, 45, 4, 1, False), (100, None, 2, 1, True), (100, None, 2, 2, False),
    (1000, None, 24, 24, True), (1000, None, 24, 24, False), (90, 5000, 4, 4, False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,m,heads,kv,causal", INFINITE)
def test_infinite_values_are_the_output(dev, n, m, heads, kv, causal, dtype):
    """Of the rows that see them, under weights that are all positive, in whole tiles, the last and those on the
    mask's edge; of both signs NaN."""
    dt, d, m, own = DTYPES[dtype], 32, m or n, m is None
    q, k, v = (randn((r, h, d), dt, i, 0.1).to(dev) for i, (r, h) in enumerate(((n, heads), (m, kv), (m, kv))))
    at = [m // 2, m - 1]
    for a in at:
        v[a, :, 5], v[a, :, 6] = math.inf, -math.inf
    v[at[0], :, 7], v[at[1], :, 7] = math.inf, -math.inf
    offsets, keys = (torch.tensor([0, r], dtype=torch.int32, device=dev) for r in (n, m))
    kw = {} if own else dict(key_offsets=keys)
    with torch.no_grad():
        y = F.attention(q, k, v, offsets, causal=causal, **kw)
    for y in (y, F.attention(q.requires_grad_(True), k, v, offsets, causal=causal, **kw).detach()):
        sees = torch.arange(n, device=dev) >= n - m + at[0] if causal else torch.ones(n, dtype=torch.bool, device=dev)
        both = torch.arange(n, device=dev) >= n - m + at[1] if causal else sees
        assert torch.isfinite(y[~sees]).all() and torch.isfinite(y[..., :5]).all() and torch.isfinite(y[..., 8:]).all()
        assert (y[sees][..., 5] == math.inf).all() and (y[sees][..., 6] == -math.inf).all()
        assert torch.isnan(y[both][..., 7]).all() and (y[sees & ~both][..., 7] == math.inf).all()


# ---------------------------------------------------------------------------
# rows that overlap
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[1] * 5, [70], [3, 0, 129, 33]])
def test_a_query_expanded_over_rows(dev, lengths, causal, dtype):
    """One query for all rows (a row stride of 0), with scores far above those that exp2 takes in 16 bits."""
    n, room = sum(lengths), [m * 3 + 60 for m in lengths]
    m = sum(room)
    q = (randn((1, 4, 64), DTYPES[dtype], 1) * 3).to(dev).expand(n, -1, -1)
    assert q.stride(0) == 0
    k, v = randn((m, 2, 64), DTYPES[dtype], 2) * 3, randn((m, 2, 64), DTYPES[dtype], 3)
    check(dev, q, k, v, lengths, k_lengths=room, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("step", [0, 8, 32])
def test_rows_closer_than_their_width(dev, step, dtype):
    """Queries, keys and values whose rows lie `step` values apart, less than a head has; infinities in the
    room behind a cache's keys."""
    dt, n, d = DTYPES[dtype], 150, 64

    def rows(seed, size):
        flat = (randn(((n - 1) * step + d,), dt, seed) * size).to(dev)
        return flat.as_strided((n, 1, d), (step, d, 1))
    q, k, v = rows(1, 3.0), rows(2, 3.0), rows(3, 1.0)
    check(dev, q, k, v, [60, 90], causal=True)
    used = n - 20
    if step:
        v.as_strided(((n - 1) * step + d,), (1,))[(used - 1) * step + d:] = math.inf
    check(dev, q[:4], k, v, [4], k_lengths=[n], counts=[used], causal=False)


# ---------------------------------------------------------------------------
# small weights in fp16
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("queries,kv,train", [(3, 1, False), (3, 1, True), (200, 96, False)])
def test_many_small_weights(dev, queries, kv, train):
    """fp16, few keys that take nearly all with values of 0, and 8000 others with e^-17 each, whose part is the
    output: by a token's waves and by blocks of 128 columns.  In the product a weight is off by 2^-11 of itself or, lifted
    by 2^11, by 2^-25 under that; sums and scores as in the reference's docstring."""
    n, gap, d, large = 8000, 17.0, 16, [0, 32, 64, 96]
    q = torch.zeros(queries, kv, d, dtype=torch.float16)
    q[..., 0] = 1.0
    k, v = torch.zeros(n, kv, d, dtype=torch.float16), 1 + randn((n, kv, d), torch.float16, 5).abs() / 4
    k[large, :, 0], v[large] = gap, 0.0
    y = F.attention(q.to(dev).requires_grad_(train), k.to(dev), v.to(dev),
                    torch.tensor([0, queries], dtype=torch.int32, device=dev),
                    key_offsets=torch.tensor([0, n], dtype=torch.int32, device=dev), scale=1.0).detach().cpu().double()
    each = math.exp(-gap) / (len(large) + (n - len(large)) * math.exp(-gap))
    small = v.double().sum(0)
    ref = each * small
    w = 2 * 4 * E * gap + 2 * (n + 16) * E
    tol = 2.0 ** -11 * ref + ((w + 2.0 ** -11) * each + 2.0 ** -36) * small
    assert ((y - ref).abs() <= tol).all(), ((y - ref).abs() / ref).max()


# ---------------------------------------------------------------------------
# small gradients in fp16
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("size", [64.0, 1.0, 2.0 ** -7, 2.0 ** -13])
@pytest.mark.parametrize("kv,causal", [(1, False), (1, True), (24, True)])
def test_small_gradients(dev, kv, causal, size):
    """fp16, even weights of 4000 keys, and gradients of the outputs down to what fp16 holds few bits of: ds is
    some sqrt(n) below dq and dk.  Each ds is off by half a step, 2^-11 of itself (but 2^-39, half a step under the
    lift of 2^14, or 2^-34 of the largest of its column, which that is lowered by), dp and delta by their sums'
    2 (d + 16) e, and the outputs round once."""
    n, d = 4000, 64
    u = UNIT[torch.float16]
    v, dout = randn((n, kv, d), torch.float16, 3), (randn((n, kv, d), torch.float32, 4) * size).half()
    small, large = randn((n, kv, d), torch.float32, 1) * 2.0 ** -6, randn((n, kv, d), torch.float32, 2) * 16
    offsets = torch.tensor([0, n], dtype=torch.int32, device=dev)
    heads = slice(0, min(kv, 2))
    for which in ("dq", "dk"):
        q, k = (t.half() for t in ((small, large) if which == "dq" else (large, small)))
        got = gradients([t.to(dev) for t in (q, k, v)], offsets, dout.to(dev), causal=causal)[1 if which == "dq" else 2]
        for h in range(heads.start, heads.stop):
            x, y, z, g = (t[:, h].to(dev).double() for t in (q, k, v, dout))
            seen = torch.ones(n, n, dtype=torch.bool, device=dev)
            seen = seen.tril() if causal else seen
            s = torch.where(seen, d ** -0.5 * (x @ y.t()), -math.inf)
            p = torch.softmax(s, 1)
            dp = g @ z.t()
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta)
            es = d ** -0.5 * (d + 16) * E * (x.abs() @ y.abs().t()) + 4 * E * torch.where(seen, s, 0).abs()
            w = 2 * es.amax(1, keepdim=True) + 2 * (n + 16) * E
            # (delta by way of the outputs in two pieces, whose weights round by u each, at random: 6 of their deviation)
            to = 6 * u * (p.square() @ z.square()).sqrt() + 2.0 ** -36 * (seen.double() @ z.abs())
            edp = (d + 16) * E * (g.abs() @ z.abs().t() + (p * dp.abs()).sum(1, keepdim=True)) + (g.abs() * to).sum(1, keepdim=True)
            eds = w * ds.abs() + p * edp
            if which == "dq":
                low = 2.0 ** -39 + 2.0 ** -34 * ds.abs().amax(1, keepdim=True)
                eds = torch.where(seen, eds + u * ds.abs() + low, 0)
                ref, tol = d ** -0.5 * ds @ y, d ** -0.5 * eds @ y.abs()
            else:
                low = 2.0 ** -39 + 2.0 ** -34 * ds.abs().amax(0, keepdim=True)
                eds = torch.where(seen, eds + u * ds.abs() + low, 0)
                ref, tol = d ** -0.5 * ds.t() @ x, d ** -0.5 * eds.t() @ x.abs()
            tol = tol + u * ref.abs() + 2.0 ** -25 + 2 * n * E * tol
            bad = (got[:, h].double() - ref).abs() > tol
            assert not bad.any(), (which, h, int(bad.sum()), (got[:, h].double() - ref).abs().max().item(), tol.max().item())


# ---------------------------------------------------------------------------
# common parts that cancel
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,part", [("f16", 32.0), ("bf16", 16.0)])
@pytest.mark.parametrize("what", ["values", "keys", "queries"])
@pytest.mark.parametrize("times", [6, 48])
def test_common_parts_cancel(dev, times, what, dtype, part):
    """Few keys a row (all of them on the mask's edge), and values, keys or a pair of heads' queries that have
    a common part of `part` times what tells them apart: it cancels in dq or dk, what the roundings of the outputs, of
    the weights and of ds leave of it does not.  With those kept as second operands an output, a weight of the
    gradients and ds are held to u^2 / 2 and a weight of the outputs to 2 u^2, so a gradient's norm is off by u (its own
    rounding) and by `part` times some of these: below u / 4.  Rounded without, one of them alone is some
    part u / sqrt(12)."""
    dt, lengths = DTYPES[dtype], [9, 12, 7, 11] * times
    u, n, d = UNIT[dt], sum(lengths), 64
    assert columns_fill_blocks(n, 2, 1, len(lengths), dt) == (times > 6)
    q, k, v, g = (randn((n, h, d), torch.float32, i) for i, h in ((1, 2), (2, 1), (3, 1), (4, 2)))
    if what == "values":
        v = 1 + v / part
    elif what == "keys":
        k = 1 + k / part
    else:  # the second head's query is the first's and a little, its gradient the other way
        q[:, 1], g[:, 1] = q[:, 0] + q[:, 1] / part, -g[:, 0]
    q, k, v, g = (t.to(dt).to(dev) for t in (q, k, v, g))
    offsets = offsets_of(lengths)
    got = gradients((q, k, v), offsets.to(dev), g, causal=True)
    refs = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v)]
    for a, b in zip(offsets.tolist(), offsets.tolist()[1:]):
        seen = torch.ones(b - a, b - a, dtype=torch.bool, device=dev).tril()
        for h in range(2):
            x, y, z, w = (t.double() for t in (q[a:b, h], k[a:b, 0], v[a:b, 0], g[a:b, h]))
            p = torch.softmax(torch.where(seen, d ** -0.5 * (x @ y.t()), -math.inf), 1)
            dp = w @ z.t()
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            refs[0][a:b, h] = d ** -0.5 * ds @ y
            refs[1][a:b, 0] += d ** -0.5 * ds.t() @ x
            refs[2][a:b, 0] += p.t() @ w
    for i, name in ((1, "dq"), (2, "dk"), (3, "dv")):
        if (what, name) in (("queries", "dq"), ("values", "dv"), ("keys", "dv")):
            continue  # (nothing cancels)
        off = (got[i].double() - refs[i - 1]).norm() / refs[i - 1].norm()
        assert off <= 1.25 * u, (name, off.item() / u)


# ---------------------------------------------------------------------------
# large scores in fp32
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("queries,keys,kv,rising", [(1, 300, 1, False), (3, 300, 2, True), (1, 5000, 1, False),
                                                    (600, 300, 110, False), (600, 300, 110, True)])
def test_large_scores_in_parts(dev, queries, keys, kv, rising):
    """fp32, scores of 15000 and little more, exact in the type: what waves, parts and the maximum's steps put
    together is of one reference each, rounded once.  A weight is off by its exponential's 2^-23 and its argument's
    2^-24 of the distance from the largest (in exp2, once for the scale, once for the product), sums of n terms by n e, all
    twice (over the weights' sum); joins by 2^-22 each.  By way of a rounded reference of 21640 they are off by some 2^-11."""
    d, g = 16, torch.Generator().manual_seed(3)
    s = 15000 + torch.randint(0, 256, (keys,), generator=g) / 256 + (torch.arange(keys) // 32 * 0.5 if rising else 0)
    q, k = torch.zeros(queries, kv, d), torch.zeros(keys, kv, d)
    q[..., 0], k[..., 0] = 1, s[:, None]
    v = (1 - torch.arange(keys) // 32 % 2 * 2.0)[:, None, None].expand(-1, kv, d).contiguous()
    q, k, v = (t.to(dev).requires_grad_(True) for t in (q, k, v))
    offsets, at = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (queries, keys))
    assert columns_fill_blocks(queries, kv, kv, 1, torch.float32) == (queries > 3)
    with torch.no_grad():
        y = F.attention(q, k, v, offsets, key_offsets=at, scale=1.0)
    z = F.attention(q, k, v, offsets, key_offsets=at, scale=1.0)
    dv = torch.autograd.grad(z, v, torch.ones_like(z))[0]
    s = s.to(dev).double()
    p = torch.softmax(s, 0)
    each = 2 ** -23 + 2 * E * (s.max() - s) * 1.45
    off = 2 * ((p * each).sum() + min(keys, 640) * E + 4 * 2.0 ** -22)
    ref = torch.einsum("n,nhd->hd", p, v.detach().double())
    for out in (y, z):
        assert ((out.double() - ref).abs() <= off).all(), ((out.double() - ref).abs().max() / off).item()
    tol = (queries * p * (each + off + queries * E))[:, None, None]
    bad = (dv.double() - queries * p[:, None, None]).abs() / tol
    assert (bad <= 1).all(), bad.max().item()
