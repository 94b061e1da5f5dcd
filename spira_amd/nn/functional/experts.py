"""Row operators of a mixture-of-experts block over voxel features [N, C]:
products grouped by expert, the router and the sum of its experts' rows, the
norms around the block with its gate and residual, and dropout, each with its
gradient.  No reference counterpart.

fp16, bf16 and fp32 features (all floating inputs of a call share one type, the
routing weights are fp32); sums are taken in fp32 and outputs rounded once.
Calls run on the current stream, read nothing back and give identical results
when repeated.  Errors are ``RuntimeError("[Spira] ...")``; CPU tensors raise
``NotImplementedError``.  Gradients are of first order; tangents of forward
mode are refused.
"""
from __future__ import annotations

from operator import index
from typing import NamedTuple, Optional, Tuple, Union

import torch

from ._native import _C
from .convolution import _gpu

__all__ = ["ExpertRoutes", "route_experts", "grouped_linear", "combine_experts", "gated_residual_norm", "rms_norm",
           "dropout", "BalanceLoss", "balance_loss"]


_LOW = (1 << 64) - 1


class ExpertRoutes(NamedTuple):
    """A router's choice for T tokens of E experts, k each, and the order of
    its T * k assignments by expert (tokens ascending within an expert).

    Where a token has fewer than k experts to choose from, the rest of its
    choices hold expert -1, slot -1 and weight 0, and as many rows at the end
    belong to no expert.
    """
    weights: torch.Tensor  # [T, k] fp32, differentiable
    experts: torch.Tensor  # [T, k] int32
    offsets: torch.Tensor  # [E + 1] int32: expert e has rows offsets[e] to offsets[e + 1]
    rows: torch.Tensor     # [T * k] int32: the token of each row, or -1
    slots: torch.Tensor    # [T, k] int32: the row of each choice, or -1


def route_experts(logits: torch.Tensor, k: int, *, renormalize: bool = True) -> ExpertRoutes:
    """The k largest of each token's ``logits`` [T, E] (the lowest index first
    among equals) with their softmax weights, over the chosen ones or, without
    ``renormalize``, over all, and the order of the tokens by expert.

    A logit of -inf masks its expert for that token.  NaN ranks above every
    number and makes its token's weights NaN.  Up to 512 experts and 16
    choices.
    """
    _gpu(logits)
    return ExpertRoutes(*_C.route_experts(logits, k, renormalize))


class BalanceLoss(NamedTuple):
    """What a router's choices over T tokens say of its E experts' use."""
    loss: torch.Tensor           # [] fp32, differentiable: 1 where all are used alike, up to E
    counts: torch.Tensor         # [E] int32: assignments to each expert
    probabilities: torch.Tensor  # [E] fp32: mean of the router's softmax over the tokens


def balance_loss(logits: torch.Tensor, groups: Union[torch.Tensor, ExpertRoutes]) -> BalanceLoss:
    """``E * sum_e share[e] * probabilities[e]``: the loss that keeps a router's
    experts in use.

    ``logits`` [T, E] are the router's, ``groups`` its ``ExpertRoutes`` or their
    offsets [E + 1] int32.  share[e] is expert e's part of the assignments (it has
    no gradient), probabilities[e] the mean of softmax(logits)[:, e] over the
    tokens that have an expert (a logit above -inf).  Up to 512 experts.
    """
    _gpu(logits)
    return BalanceLoss(*_C.balance_loss(logits, groups.offsets if isinstance(groups, ExpertRoutes) else groups))


def grouped_linear(features: torch.Tensor, weight: torch.Tensor, groups: Union[torch.Tensor, ExpertRoutes], *,
                   bias: Optional[torch.Tensor] = None, relu: bool = False) -> torch.Tensor:
    """``relu(features[r] @ weight[e] + bias[e])`` for the rows r of each group e.

    ``weight`` is [E, C_in, C_out], ``bias`` [E, C_out].  ``groups``: offsets
    [E + 1] int32 (on the GPU, ascending), group e being the rows offsets[e] to
    offsets[e + 1] of ``features``; or a router's ``ExpertRoutes``, in which
    case ``features`` are its tokens [T, C_in] and the rows [T * k] are gathered
    by the kernel (and their gradients summed per token).  Groups may have any
    number of rows, none included; rows in no group are zero.
    """
    _gpu(features)
    if isinstance(groups, ExpertRoutes):
        return _C.grouped_linear(features, weight, groups.offsets, groups.rows, groups.slots, bias, relu)
    return _C.grouped_linear(features, weight, groups, None, None, bias, relu)


def combine_experts(features: torch.Tensor, routes: ExpertRoutes) -> torch.Tensor:
    """The weighted sum of each token's rows: ``sum_j weights[t, j] *
    features[slots[t, j]]`` over its choices, ``features`` [T * k, C] in the
    routes' order.  Zero for a token without any."""
    _gpu(features)
    return _C.combine_experts(features, routes.weights, routes.rows, routes.slots)


def gated_residual_norm(residual: torch.Tensor, update: torch.Tensor, *, weight: Optional[torch.Tensor] = None,
                        gate: Optional[torch.Tensor] = None, gate_sigmoid: bool = False, scale: float = 1.0,
                        next_weight: Optional[torch.Tensor] = None,
                        eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The end of a residual block and the entry of the next, in one pass:

        z = update / sqrt(mean(update ** 2) + eps) * weight   (or update)
        r = residual + scale * gate * z
        n = r / sqrt(mean(r ** 2) + eps) * next_weight        (or None)

    Returns (r, n).  ``weight`` and ``next_weight`` are [C]; ``gate`` is [C],
    [N, 1] or [N, C], taken as it is or through a sigmoid.  Up to 16384
    channels.
    """
    _gpu(residual)
    return _C.gated_residual_norm(residual, update, weight, gate, gate_sigmoid, scale, next_weight, eps)


def rms_norm(features: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``features / sqrt(mean(features ** 2) + eps) * weight`` over the channels:
    the entry of a first block."""
    _gpu(features)
    return _C.gated_residual_norm(features, None, None, None, False, 1.0, weight, eps)[1]


def dropout(features: torch.Tensor, p: float, seed: int, offset: int = 0, *,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``features / (1 - p)`` where a value is kept (with probability 1 - p),
    else 0, plus ``residual``.

    Value i (in row-major order) is kept if word i % 4 of Philox-4x32 with 7
    rounds, counter (i // 4, offset) and key ``seed`` (64 bits each), is at
    least floor(p * 2**32): the same mask whenever these are the same, on
    which the gradient relies (no mask is stored).  A program counts
    ``offset`` up by one per call, and a captured graph replays the mask that
    it was captured with.
    """
    _gpu(features)
    return _C.dropout(features, p, index(seed) & _LOW, index(offset) & _LOW, residual)
