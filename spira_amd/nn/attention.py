"""An attention block on voxel features, with its norms, rotation, gate and
residual.  No reference counterpart."""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from ..tensors import SparseTensor
from . import functional as F

__all__ = ["AttentionBlock"]


class AttentionBlock(nn.Module):
    """``x + scale * gate * norm(project(attention(heads(norm(x)))))`` over the
    voxels of a scene.

    ``heads`` query heads of ``head_channels`` (channels // heads unless given) and
    ``kv_heads`` key heads (as many unless given); queries and keys are normed per
    head and rotated by their voxel's x, y and z (``rotate``, which takes heads of an
    even width from 6 on).  ``gate`` is learned per channel.

    Takes and returns a ``SparseTensor`` of the same coordinates (packed or not).  Its
    rows are one sequence, or with ``window`` sequences of so many consecutive rows
    each: of an ordered tensor, windows along the order of its keys.  A batch of
    scenes behind each other passes their ``offsets`` [scenes + 1] (int32, on the GPU)
    instead of the window.  ``causal``: a voxel sees those before it and itself.  Parameters have
    the features' type (``.half()``, ``.bfloat16()``).
    """

    def __init__(self, channels: int, heads: int, kv_heads: Optional[int] = None, *, head_channels: Optional[int] = None,
                 window: Optional[int] = None, causal: bool = False, rotate: bool = True, base: float = 100.0,
                 scale: float = 1.0, eps: float = 1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
            raise RuntimeError("[Spira] AttentionBlock: the number of heads must be a multiple of the key heads'")
        d = channels // heads if head_channels is None else head_channels
        if not 1 <= d <= 128 or (rotate and (d % 2 or d < 6)):
            raise RuntimeError("[Spira] AttentionBlock: needs heads of 1 to 128 channels, and to rotate them an even "
                               f"number from 6 on, got {d}")
        if window is not None and window <= 0:
            raise RuntimeError(f"[Spira] AttentionBlock: the window must be positive, got {window}")
        self.heads, self.kv_heads, self.head_channels = heads, kv_heads, d
        self.window, self.causal, self.rotate = window, causal, rotate
        self.base, self.scale, self.eps = base, scale, eps
        self.entry = nn.Parameter(torch.ones(channels))
        self.project = nn.Parameter(torch.randn(channels, (heads + 2 * kv_heads) * d) * channels ** -0.5)
        self.query_norm = nn.Parameter(torch.ones(d))
        self.key_norm = nn.Parameter(torch.ones(d))
        self.out = nn.Parameter(torch.randn(heads * d, channels) * (heads * d) ** -0.5)
        self.exit = nn.Parameter(torch.ones(channels))
        self.gate = nn.Parameter(torch.full((channels,), 0.1))

    def _sequences(self, rows: int, device: torch.device) -> torch.Tensor:
        window = max(rows, 1) if self.window is None else self.window
        count = max(1, -(-rows // window))
        # (the last may be shorter; made on the GPU, with nothing to wait for)
        return (torch.arange(count + 1, device=device) * window).clamp_(max=rows).int()

    def forward(self, input: SparseTensor, offsets: Optional[torch.Tensor] = None) -> SparseTensor:
        x, (h, k) = input.features, (self.heads, self.kv_heads)
        if offsets is None:
            offsets = self._sequences(x.shape[0], x.device)
        positions = None
        if self.rotate:
            positions = input.coordinates if input.coordinates.dim() == 2 else F.unflatten(input.coordinates)
        n = F.rms_norm(x, self.entry, self.eps)
        p = (n @ self.project).view(-1, h + 2 * k, self.head_channels)
        q, keys = F.norm_rotate_heads(p[:, :h], p[:, h:h + k], query_weight=self.query_norm, key_weight=self.key_norm,
                                      positions=positions, base=self.base, eps=self.eps)
        y = F.attention(q, keys, p[:, h + k:], offsets, causal=self.causal)
        y, _ = F.gated_residual_norm(x, y.flatten(1) @ self.out, weight=self.exit, gate=self.gate, scale=self.scale,
                                     eps=self.eps)
        return SparseTensor(coordinates=input.coordinates, features=y, stride=input.stride, double=input._double)
