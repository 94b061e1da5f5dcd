"""A mixture-of-experts feed-forward block on voxel features, with its norms,
gate, dropout and residual.  No reference counterpart."""
from __future__ import annotations

from typing import Optional, Tuple

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

    Dropout acts in training mode.  Without a ``seed`` each call's mask is drawn
    from torch's CPU generator: another in every call, block and, where their
    generators differ, process.  With one it follows from the seed and the
    number of training calls so far, which is part of the state_dict; blocks of
    one width (copies among them) and ranks then need seeds of their own, or
    they drop the same positions.

    A call that a backward pass computes again (``torch.utils.checkpoint``) has
    its first mask, by torch's generator, whose state checkpointing restores
    (``preserve_rng_state``, the default).  A captured graph replays the mask
    that it was captured with.
    """

    _KEPT = 4096  # calls whose numbers are kept for a backward pass

    def __init__(self, channels: int, hidden: int, experts: int, choices: int = 2, *, dropout: float = 0.0,
                 scale: float = 1.0, eps: float = 1e-6, seed: Optional[int] = None):
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
        # (no buffer: it is read on the host and stays there, where a data-parallel wrapper over RCCL could not send it)
        self.calls = torch.zeros((), dtype=torch.int64, device="cpu")
        self._numbers = {}  # of recent training calls, by their draws

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "calls"] = self.calls.detach()

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)
        key = prefix + "calls"
        if key in state_dict:
            self.calls.fill_(int(state_dict[key]))
        elif strict:
            missing_keys.append(key)
        if key in unexpected_keys:
            unexpected_keys.remove(key)

    def _mask(self) -> Tuple[int, int]:
        """Seed and offset of this training call's mask."""
        draw = tuple(torch.randint(2 ** 63 - 1, (2,), dtype=torch.int64, device="cpu").tolist())
        again = torch._C._current_graph_task_id() >= 0  # within a backward pass: a call computed again
        if not again:
            self._numbers.pop(draw, None)
            self._numbers[draw] = int(self.calls)
            if len(self._numbers) > self._KEPT:
                del self._numbers[next(iter(self._numbers))]
            self.calls += 1
        if draw not in self._numbers:
            raise RuntimeError("[Spira] ExpertBlock: a training call within a backward pass that repeats none before it "
                               "(checkpointing has to preserve the state of torch's generator)")
        return draw if self.seed is None else (self.seed, self._numbers[draw])

    def forward(self, input: SparseTensor) -> SparseTensor:
        x = input.features
        n = F.rms_norm(x, self.entry, self.eps)
        routes = F.route_experts(n @ self.router, self.choices)
        h = F.grouped_linear(n, self.up, routes, bias=self.up_bias, relu=True)
        h = F.grouped_linear(h, self.down, routes.offsets, bias=self.down_bias)
        h = F.combine_experts(h, routes)
        if self.training and self.dropout > 0:
            h = F.dropout(h, self.dropout, *self._mask())
        y, _ = F.gated_residual_norm(x, h, weight=self.exit, gate=self.gate, scale=self.scale, eps=self.eps)
        return SparseTensor(coordinates=input.coordinates, features=y, stride=input.stride)
