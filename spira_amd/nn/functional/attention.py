"""Attention over rows of voxel features: packed sequences with grouped heads, and
the norms and rotation of its queries and keys, each with its gradient.  No
reference counterpart.

Types, streams, errors and gradients are those of the other row operators
(``experts.py``).  Heads are [N, H, D] with the D values of a head consecutive;
rows and heads may lie at any stride (views of one projection are read in place).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._native import _C
from .convolution import _gpu

__all__ = ["attention", "norm_rotate_heads"]


def attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, offsets: torch.Tensor, *,
              key_offsets: Optional[torch.Tensor] = None, key_counts: Optional[torch.Tensor] = None,
              causal: bool = False, scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale * queries @ keys^T) @ values`` within each of B packed
    sequences and for each head.

    ``queries`` are [N, H, D], ``keys`` and ``values`` [M, Hk, D], H a multiple of
    Hk (query head h reads key head h * Hk // H), D from 1 to 128.  ``offsets``
    [B + 1] int32 (on the GPU, ascending): sequence b has the queries offsets[b] to
    offsets[b + 1], and the same of the keys.  A cache has ``key_offsets`` [B + 1]
    of its own and, with room behind a sequence's keys, ``key_counts`` [B] int32:
    the keys in use from key_offsets[b] on; what lies behind them is not read and
    gets no gradient.  ``causal``: query i of n sees key j of m if j <= i + m - n,
    the last query all of them.  ``scale`` (positive) is D ** -0.5 unless given.

    Up to 65536 sequences of any lengths, none included.  A query that sees no key, or
    is in no sequence, gets zeros.  Values that are not finite reach the queries
    that see them only.  In 16 bits the softmax's weights, and in the gradients the
    scores' too, are rounded to the features' type before their products; the outputs of
    few tokens, and the rows of tiles in which a causal mask ends, take what that leaves as
    a second term.  In fp32 nothing is rounded.
    """
    _gpu(queries)
    return _C.attention(queries, keys, values, offsets, key_offsets, key_counts, causal, scale)


def norm_rotate_heads(queries: torch.Tensor, keys: torch.Tensor, *, query_weight: Optional[torch.Tensor] = None,
                      key_weight: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                      base: float = 10000.0, interleaved: bool = False,
                      eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries [N, H, D] and keys [N, Hk, D] as attention takes them: each head
    normed, ``x / sqrt(mean(x ** 2) + eps) * weight`` ([D]; as it is without one),
    then rotated by its row's position.

    ``positions`` are int32, [N] or [N, A] for A axes (a voxel's x, y, z).  Pair p
    of the D / 2 pairs is (p, p + D / 2), or (2p, 2p + 1) if ``interleaved``; band a
    of the pairs, from a * (D // 2) // A to the next band's first, belongs to axis
    a, and its pair j of n turns by positions[:, a] * base ** (-j / n) radians
    (exact to the features' type at any position).  D from 1 to 128, even with
    positions.
    """
    _gpu(queries)
    return _C.norm_rotate_heads(queries, keys, query_weight, key_weight, positions, base, interleaved, eps)
