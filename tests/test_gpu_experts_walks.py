"""The row operators where their kernels go round: blocks that walk many rows, with
sums carried from row to row; rows streamed past weights over many tiles; weights'
gradients without parts; long sums of few rows.

Tolerances follow from the arithmetic: an output's own rounding, u |ref|, and
2^-24 for each rounding on the longest way to a value, twice over, times the
magnitude that the formula has with each of its terms taken positive."""
import pytest
import torch

from spira_amd.nn import functional as F

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}


def tolerance(ref, magnitude, roundings, dtype):
    return UNIT[dtype] * ref.abs() * 1.001 + 2 * roundings * 2.0 ** -24 * magnitude + TINY[dtype]


def close(got, ref, magnitude, roundings, what=""):
    got, dtype = got.detach().double(), got.dtype
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tolerance(ref, magnitude, roundings, dtype))
    assert not bad.any(), (what, int(bad.sum()), torch.nonzero(bad)[0].tolist(), got[bad][0].item(), ref[bad][0].item())


def randn(shape, dtype, seed, scale=1.0, device="cpu"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * scale).to(dtype)


# ---------------------------------------------------------------------------
# gated_residual_norm
# ---------------------------------------------------------------------------
# a sum over a row: up to 16 values a lane, ten exchanges; a value's products, roots and gates: up to 38 more
ROW = 64


def column(n):
    """Roundings of a sum over n rows: those of a term; one a row that a lane walks (512 blocks of a row or more,
    counted as one), then over lanes, waves and blocks."""
    return ROW + (n + 511) // 512 + 6 + 16 + 14


def norm_inputs(n, c, dt, gate, device):
    x, h = randn((n, c), dt, 1, 2.0, device), randn((n, c), dt, 2, 1.0, device)
    w, w_next = 1 + randn((c,), dt, 3, 0.1, device), 1 + randn((c,), dt, 4, 0.1, device)
    shape = {"none": None, "channel": (c,), "row": (n, 1), "full": (n, c)}[gate]
    g = None if shape is None else randn(shape, dt, 5, 1.0, device)
    return x, h, w, w_next, g, randn((n, c), dt, 6, 1.0, device), randn((n, c), dt, 7, 1.0, device)


def norm_reference(x, h, w, w_next, gate, dr, dn, sigmoid, scale, eps):
    """{name: (value, magnitude)} of both outputs and all gradients, and {name: the rows' terms} of sums over rows."""
    x, h, w, w_next, dr, dn = (t.double() for t in (x, h, w, w_next, dr, dn))

    def mean(v):
        return v.mean(1, keepdim=True)

    rh = torch.rsqrt(mean(h * h) + eps)
    hh = h * rh
    z = hh * w
    raw = None if gate is None else gate.double()
    g = torch.ones((), dtype=torch.float64, device=x.device) if raw is None else torch.sigmoid(raw) if sigmoid else raw
    r = x + scale * g * z
    r_size = x.abs() + (scale * g * z).abs()
    rr = torch.rsqrt(mean(r * r) + eps)
    rhat, rhat_size = r * rr, r_size * rr
    dnw = dn * w_next
    dx = dr + rr * (dnw - rhat * mean(dnw * rhat))
    dx_size = dr.abs() + rr * (dnw.abs() + rhat_size * mean(dnw.abs() * rhat_size))
    dz, dz_size = scale * g * dx, (scale * g).abs() * dx_size
    dh = rh * (dz * w - hh * mean(dz * w * hh))
    dh_size = rh * (dz_size * w.abs() + hh.abs() * mean(dz_size * (w * hh).abs()))
    out = {"r": (r, r_size), "n": (rhat * w_next, rhat_size * w_next.abs()), "dx": (dx, dx_size), "dh": (dh, dh_size)}
    terms = {"dw": (dz * hh, dz_size * hh.abs()), "dw_next": (dn * rhat, dn.abs() * rhat_size)}
    if gate is not None:
        slope = g * (1 - g) if sigmoid else torch.ones_like(g)
        dg, dg_size = scale * z * dx * slope, scale * z.abs() * dx_size * (g if sigmoid else slope)
        if gate.dim() == 1:
            terms["dgate"] = (dg, dg_size)
        elif gate.shape[1] == 1:
            out["dgate"] = (dg.sum(1, keepdim=True), dg_size.sum(1, keepdim=True))
        else:
            out["dgate"] = (dg, dg_size)
    return out, terms


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate,sigmoid", [("none", False), ("channel", False), ("channel", True), ("row", True),
                                          ("full", True), ("full", False)])
@pytest.mark.parametrize("n,c", [(20_011, 96), (40_013, 20), (2_117, 2048), (2_100, 8200)])
def test_norms_walk_rows(dev, n, c, gate, sigmoid, dtype):
    """More rows than the blocks of either pass hold at once, and not a multiple of a block's; the last two with a row
    to a block, whose sums meet at barriers."""
    x, h, w, w_next, g, dr, dn = norm_inputs(n, c, DTYPES[dtype], gate, dev)
    out, terms = norm_reference(x, h, w, w_next, g, dr, dn, sigmoid, 0.5, 1e-6)
    leaves = {"dx": x, "dh": h, "dw": w, "dw_next": w_next} | ({} if g is None else {"dgate": g})
    for t in leaves.values():
        t.requires_grad_(True)
    r, nx = F.gated_residual_norm(x, h, weight=w, gate=g, gate_sigmoid=sigmoid, scale=0.5, next_weight=w_next, eps=1e-6)
    got = {"r": r, "n": nx} | dict(zip(leaves, torch.autograd.grad((r, nx), list(leaves.values()), (dr, dn))))
    for name, (ref, size) in out.items():
        close(got[name], ref, size, ROW, name)
    for name, (term, size) in terms.items():
        close(got[name], term.sum(0), size.sum(0), column(n), name)


@pytest.mark.parametrize("gate", ["none", "channel"])
@pytest.mark.parametrize("n,c", [(20_011, 96), (2_117, 512)])
def test_a_row_too_many_or_too_few_is_seen(n, c, gate):
    """The tolerance of sums over rows against the formula itself, in fp32: without the first, the last or another row,
    or with one of them twice, no sum passes."""
    _, terms = norm_reference(*norm_inputs(n, c, torch.float32, gate, "cpu"), False, 0.5, 1e-6)
    for name, (term, size) in terms.items():
        limit = tolerance(term.sum(0), size.sum(0), column(n), torch.float32)
        for row in (0, n // 2, n - 1):
            assert (term[row].abs() > 2 * limit).any(), (name, row)


# ---------------------------------------------------------------------------
# grouped_linear
# ---------------------------------------------------------------------------
def sizes_of(kind, groups, rows):
    if kind == "one":
        return [rows if e == groups // 3 else 0 for e in range(groups)]
    g = torch.Generator().manual_seed(groups + rows)
    share = torch.rand(groups, generator=g) ** 3 * (torch.rand(groups, generator=g) > 0.2)
    cuts = (share.cumsum(0) / share.sum() * (rows - 3)).long()  # (three rows of no group at the end)
    return (cuts - torch.cat([cuts.new_zeros(1), cuts[:-1]])).tolist()


def check_linear(dev, dtype, tokens, sizes, ci, co, gathered, relu=True, k=1):
    """Outputs and gradients of groups of these sizes, rows in their order or gathered from shuffled tokens."""
    dt, rows, groups = DTYPES[dtype], tokens * k, len(sizes)
    offsets = torch.tensor([0] + sizes).cumsum(0).tolist()
    held = offsets[-1]
    n = tokens if gathered else rows
    x, w = randn((n, ci), dt, 1, 1.0, dev), randn((groups, ci, co), dt, 2, ci ** -0.5, dev)
    b, dy = randn((groups, co), dt, 3, 0.1, dev), randn((rows, co), dt, 4, 1.0, dev)
    at = torch.arange(rows, device=dev)
    arg = torch.tensor(offsets, dtype=torch.int32, device=dev)
    if gathered:
        # (any assignment will do: choice j of token t has row (t k + j) p mod T k, rows past the groups none)
        slot = torch.arange(rows, device=dev)[torch.randperm(rows, generator=torch.Generator().manual_seed(5)).to(dev)]
        at[slot] = torch.arange(rows, device=dev) // k
        at[held:] = -1
        slots = torch.where(slot < held, slot, -1).view(tokens, k)
        ones = torch.ones(tokens, k, device=dev)
        arg = F.ExpertRoutes(ones, ones.int(), arg, at.int(), slots.int())
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = F.grouped_linear(x, w, arg, bias=b, relu=relu)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    share = torch.zeros(rows, ci, dtype=torch.float64, device=dev)
    size = torch.zeros_like(share)
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        xe, we, be = x.detach()[at[lo:hi]].double(), w[e].detach().double(), b[e].detach().double()
        ref = xe @ we + be
        close(y[lo:hi], ref.clamp(min=0) if relu else ref, xe.abs() @ we.abs() + be.abs(), ci + 16, f"y {e}")
        ze = dy[lo:hi].double() * ((y[lo:hi] > 0) if relu else 1)
        share[lo:hi], size[lo:hi] = ze @ we.T, ze.abs() @ we.T.abs()
        close(dw[e], xe.T @ ze, xe.T.abs() @ ze.abs(), hi - lo + 16, f"dw {e}")
        close(db[e], ze.sum(0), ze.abs().sum(0), hi - lo + 16, f"db {e}")
    assert torch.count_nonzero(y[held:]) == 0
    if gathered:
        sums, sizes_ = (torch.zeros(n, ci, dtype=torch.float64, device=dev).index_add_(0, at[:held], v[:held])
                        for v in (share, size))
        close(dx, sums, sizes_, co + k + 16, "dx")
    else:
        close(dx, share, size, co + 16, "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ci,co", [(32, 64), (33, 70)])
def test_streamed_rows_over_many_tiles(dev, ci, co, dtype):
    """140k gathered rows: three or more tiles of 16 rows to a wave, sources and rows fetched ahead."""
    check_linear(dev, dtype, 70_001, sizes_of("uneven", 8, 140_002), ci, co, True, k=2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gathered", [False, True])
@pytest.mark.parametrize("groups,rows,ci,co", [(300, 5_000, 256, 264), (1100, 6_000, 64, 72), (300, 5_000, 129, 131)])
def test_weights_gradient_without_parts(dev, groups, rows, ci, co, gathered, dtype):
    """1024 tiles of weights and more: whole groups, some of them empty, written at once."""
    check_linear(dev, dtype, rows, sizes_of("uneven", groups, rows), ci, co, gathered)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uneven", "one"])
@pytest.mark.parametrize("groups,rows,ci,co", [(32, 16, 2048, 512), (32, 512, 1000, 136), (20, 300, 4096, 72),
                                               (40, 640, 1024, 1096)])
def test_few_rows_long_sums(dev, groups, rows, ci, co, kind, dtype):
    """Sums past the depth at which each wave's ring of stages is used again; all rows in one of many groups.  The last
    has more blocks of 16 rows than run at once: tiles, in 16 bits."""
    check_linear(dev, dtype, rows, sizes_of(kind, groups, rows), ci, co, False)
    check_linear(dev, dtype, rows, sizes_of(kind, groups, rows), ci, co, True)
