"""Attention where its kernels' shortcuts end: values that are not finite behind the mask,
for narrow heads among others.  Units are those of test_gpu_attention.py."""
import math

import pytest
import torch

from spira_amd.nn import functional as F
from test_gpu_attention import DTYPES, randn

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
