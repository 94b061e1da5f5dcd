"""Angles of norm_rotate_heads against 60 digits, where calls of other bases, widths and axes come in
between.

A sine or cosine is off by 2^-22.7 (its own three roundings of the angle and its series), by 2^31 of the turn's 2^-60 (6 of
them a radian: 2^-26), and rounds once: 2^-22 in all."""
import decimal
import math

import pytest
import torch

from spira_amd.nn import functional as F

pytestmark = pytest.mark.gpu

TWO_PI = "6.28318530717958647692528676655900576839433879875021164194989"


def angles(positions, pairs, axes, base):
    """[rows, pairs], within one turn."""
    rows = []
    with decimal.localcontext() as c:
        c.prec = 60
        whole, log = decimal.Decimal(TWO_PI), decimal.Decimal(base).ln()
        for at in positions.view(len(positions), axes).tolist():
            row = []
            for a in range(axes):
                lo, hi = a * pairs // axes, (a + 1) * pairs // axes
                row += [float(at[a] * (-log * j / (hi - lo)).exp() % whole) for j in range(hi - lo)]
            rows.append(row)
    return torch.tensor(rows, dtype=torch.float64)


def test_calls_in_turn(dev):
    far = torch.tensor([0, 1, -1, 12345, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    calls = [(d, axes, base) for d in (64, 128, 10) for axes in (1, 3) for base in (10000.0, 500000.0, 100.0, 1.5)]
    for d, axes, base in calls + calls[::-1]:
        x = torch.zeros(len(far), 1, d, device=dev)
        x[..., :d // 2] = 1  # (of each pair the first)
        at = far if axes == 1 else torch.stack([far, far.flip(0), far.roll(2)], 1).contiguous()
        y, k = F.norm_rotate_heads(x, x, positions=at.to(dev), base=base)
        t = angles(at, d // 2, axes, base)
        off = (y[:, 0].cpu().double() - torch.cat([t.cos(), t.sin()], 1)).abs().max().item()
        assert torch.equal(y, k) and off <= 2.0 ** -22, (d, axes, base, math.log2(off))
