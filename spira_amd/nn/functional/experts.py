"""Row operators of a mixture-of-experts block over voxel features [N, C]:
products grouped by expert, the router and the sum of its experts' rows, the
norms around the block with its gate and residual, and dropout, each with its
gradient.  No reference counterpart.

fp16, bf16 and fp32 features (all floating inputs of a call share one type, the
routing weights are fp32); sums are taken in fp32 and outputs rounded once.
Calls run on the current stream, read nothing back and give identical results
when repeated.  Errors are ``RuntimeError("[Spira] ...")``; CPU tensors raise
``NotImplementedError``.  Gradients are of first order.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from ._native import _C
from .convolution import _c, _gpu

__all__ = ["ExpertRoutes", "route_experts", "grouped_linear", "combine_experts", "gated_residual_norm", "rms_norm",
           "dropout"]


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


def _tracked(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize):
        out = _C.route_experts(logits, k, renormalize)
        ctx.save_for_backward(logits, out[0], out[1])
        ctx.renormalize = renormalize
        ctx.mark_non_differentiable(*out[1:])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, *_):
        logits, weights, experts = ctx.saved_tensors
        return _C.route_experts_backward(logits, weights, experts, _c(dweights), ctx.renormalize), None, None


def route_experts(logits: torch.Tensor, k: int, *, renormalize: bool = True) -> ExpertRoutes:
    """The k largest of each token's ``logits`` [T, E] (the lowest index first
    among equals) with their softmax weights, over the chosen ones or, without
    ``renormalize``, over all, and the order of the tokens by expert.

    A logit of -inf masks its expert for that token.  NaN ranks above every
    number and makes its token's weights NaN.  Up to 512 experts and 16
    choices.
    """
    _gpu(logits)
    logits, k = _c(logits), int(k)
    if _tracked(logits):
        return ExpertRoutes(*_Route.apply(logits, k, bool(renormalize)))
    return ExpertRoutes(*_C.route_experts(logits, k, bool(renormalize)))


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, rows, slots, relu):
        y = _C.grouped_linear(x, weight, offsets, rows, bias, relu)
        ctx.save_for_backward(x, weight, offsets, rows, slots, y if relu else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, offsets, rows, slots, y = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*_C.grouped_linear_backward(x, weight, offsets, rows, slots, y, _c(dy), *need[:3]), None, None, None,
                None)


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
    rows = slots = None
    offsets = groups
    if isinstance(groups, ExpertRoutes):
        offsets, rows, slots = groups.offsets, _c(groups.rows), _c(groups.slots)
        if slots.dim() != 2 or slots.size(0) != features.size(0) or slots.numel() != rows.numel():
            raise RuntimeError(f"[Spira] grouped_linear: routes of {tuple(slots.shape)} choices and "
                               f"{rows.numel()} rows do not fit {features.size(0)} tokens")
    args = _c(features), _c(weight), _c(bias)
    if _tracked(*args):
        return _GroupedLinear.apply(*args, _c(offsets), rows, slots, bool(relu))
    return _C.grouped_linear(args[0], args[1], _c(offsets), rows, args[2], bool(relu))


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weights, rows, slots):
        ctx.save_for_backward(h, weights, rows, slots)
        return _C.combine_experts(h, slots, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        h, weights, rows, slots = ctx.saved_tensors
        return (*_C.combine_experts_backward(h, rows, slots, weights, _c(dy), *ctx.needs_input_grad[:2]), None, None)


def combine_experts(features: torch.Tensor, routes: ExpertRoutes) -> torch.Tensor:
    """The weighted sum of each token's rows: ``sum_j weights[t, j] *
    features[slots[t, j]]`` over its choices, ``features`` [T * k, C] in the
    routes' order.  Zero for a token without any."""
    _gpu(features)
    h, weights, slots = _c(features), _c(routes.weights), _c(routes.slots)
    if _tracked(h, weights):
        return _Combine.apply(h, weights, _c(routes.rows), slots)
    return _C.combine_experts(h, slots, weights)


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, weight, gate, next_weight, gate_sigmoid, scale, eps):
        r, n, inv_h, inv_r = _C.gated_residual_norm(x, h, weight, gate, gate_sigmoid, scale, next_weight, eps, True)
        ctx.save_for_backward(x, h, weight, gate, next_weight, inv_h, inv_r)
        ctx.options = gate_sigmoid, scale
        ctx.set_materialize_grads(False)
        return r, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dn):
        x, h, weight, gate, next_weight, inv_h, inv_r = ctx.saved_tensors
        need = [bool(v) for v in ctx.needs_input_grad[:5]]
        dx, dh, dw, dg, dnw = _C.gated_residual_norm_backward(
            x, h, weight, gate, ctx.options[0], ctx.options[1], next_weight, inv_h, inv_r, _c(dr), _c(dn), need)
        return dx, dh, dw, dg, dnw, None, None, None


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
    args = _c(residual), _c(update), _c(weight), _c(gate), _c(next_weight)
    if _tracked(*args):
        return _GatedResidualNorm.apply(*args, bool(gate_sigmoid), float(scale), float(eps))
    x, h, weight, gate, next_weight = args
    return _C.gated_residual_norm(x, h, weight, gate, bool(gate_sigmoid), float(scale), next_weight, float(eps),
                                  False)[:2]


def rms_norm(features: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``features / sqrt(mean(features ** 2) + eps) * weight`` over the channels:
    the entry of a first block."""
    _gpu(features)
    x, weight = _c(features), _c(weight)
    if _tracked(x, weight):
        return _GatedResidualNorm.apply(x, None, None, None, weight, False, 1.0, float(eps))[1]
    return _C.gated_residual_norm(x, None, None, None, False, 1.0, weight, float(eps), False)[1]


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.mask = p, seed, offset
        return _C.dropout(x, p, seed, offset, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = _C.dropout(_c(dy), *ctx.mask, None) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


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
    low = (1 << 64) - 1
    args = _c(features), _c(residual), float(p), int(seed) & low, int(offset) & low
    if _tracked(*args[:2]):
        return _Dropout.apply(*args)
    return _C.dropout(args[0], *args[2:], args[1])
