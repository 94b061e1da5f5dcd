"""A mixture-of-experts feed-forward block on voxel features, with its norms,
gate, dropout and residual.  No reference counterpart."""
from __future__ import annotations

import torch
from torch import nn

from ..tensors import SparseTensor
from . import functional as F

__all__ = ["ExpertBlock"]


class ExpertBlock(nn.Module):
    """``x + scale * gate * norm(dropout(experts(norm(x))))`` per voxel.

    A router picks ``choices`` of ``experts`` two-layer networks (C ->
    ``hidden`` -> C, ReLU) for each voxel and adds up their outputs with its
    softmax weights.  ``gate`` is learned per channel.  Takes and returns a
    ``SparseTensor`` of the same coordinates, behind any ``SparseConv`` block;
    parameters have the features' type (``.half()``, ``.bfloat16()``).

    Dropout acts in training mode.  Its mask follows from ``seed`` and the
    number of training calls so far, which is part of the state_dict.
    """

    def __init__(self, channels: int, hidden: int, experts: int, choices: int = 2, *, dropout: float = 0.0,
                 scale: float = 1.0, eps: float = 1e-6, seed: int = 0):
        super().__init__()
        self.choices, self.dropout, self.scale, self.eps, self.seed = choices, dropout, scale, eps, seed
        self.entry = nn.Parameter(torch.ones(channels))
        self.router = nn.Parameter(torch.randn(channels, experts) * channels ** -0.5)
        self.up = nn.Parameter(torch.randn(experts, channels, hidden) * (2 / channels) ** 0.5)
        self.up_bias = nn.Parameter(torch.zeros(experts, hidden))
        self.down = nn.Parameter(torch.randn(experts, hidden, channels) * hidden ** -0.5)
        self.down_bias = nn.Parameter(torch.zeros(experts, channels))
        self.exit = nn.Parameter(torch.ones(channels))
        self.gate = nn.Parameter(torch.full((channels,), 0.1))
        self.register_buffer("calls", torch.zeros((), dtype=torch.int64, device="cpu"))

    def _apply(self, fn, recurse=True):
        # (the count of calls is read on the host: it stays there)
        calls = self._buffers.pop("calls")
        super()._apply(fn, recurse)
        self._buffers["calls"] = calls
        return self

    def forward(self, input: SparseTensor) -> SparseTensor:
        x = input.features
        n = F.rms_norm(x, self.entry, self.eps)
        routes = F.route_experts(n @ self.router, self.choices)
        h = F.grouped_linear(n, self.up, routes, bias=self.up_bias, relu=True)
        h = F.grouped_linear(h, self.down, routes.offsets, bias=self.down_bias)
        h = F.combine_experts(h, routes)
        if self.training and self.dropout > 0:
            h = F.dropout(h, self.dropout, self.seed, int(self.calls))
            self.calls += 1
        y, _ = F.gated_residual_norm(x, h, weight=self.exit, gate=self.gate, scale=self.scale, eps=self.eps)
        return SparseTensor(coordinates=input.coordinates, features=y, stride=input.stride)
