"""Rows moved by scores instead of by a seed (addition to the reference API).

``route`` assigns every row to ``top_k`` experts, ``plan_rows`` turns the choices into an order that brings
the rows of an expert together, ``dispatch_rows`` moves rows into that order and ``combine_rows`` sums
them back, weighted.  As in the shuffle, a row is one instance: everything behind axis 0.  All run
on the tensors' current stream, give the same result on every run, and have gradients (of first
order, by backward passes: tangents of forward-mode differentiation are refused).  All can be captured into CUDA graphs; as for any PyTorch backward pass, capture one with
leaves of its own, not those of an eager graph that is still alive.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _native

SCORINGS = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"top2": 0, "max": 1}


class Routing(NamedTuple):
    """``experts`` int32 (rows, top_k), best first, -1 where none is left; ``weights`` float32 (rows, top_k)."""

    experts: torch.Tensor
    weights: torch.Tensor


class RowPlan(NamedTuple):
    """An order of rows * top_k entries by expert.

    ``slots`` int32 (rows, top_k): the place of each entry, -1 for an entry without an expert.
    ``sources`` int32 (rows * top_k,): the entry (row * top_k + j) at each place; -1 behind the last one.
    ``offsets`` int32 (n_experts + 1,): the first place of each expert, and the number of places in use.

    ``plan_rows`` names every place in use once.  With a plan made by hand that does not, a place named twice holds
    pieces of either row (or gradient), and a place below ``offsets[-1]`` that no entry names holds anything.
    """

    slots: torch.Tensor
    sources: torch.Tensor
    offsets: torch.Tensor


def route(
    logits: torch.Tensor,
    top_k: int,
    *,
    scoring: str = "softmax",
    bias: torch.Tensor | None = None,
    n_groups: int = 1,
    top_groups: int | None = None,
    group_score: str = "top2",
    renormalize: bool = False,
    scale: float = 1.0,
) -> Routing:
    """Choose ``top_k`` experts for every row.

    With ``s`` the softmax or sigmoid of a row's logits, the experts with the highest ``s + bias`` are
    chosen (equal ones by the lowest index; scores are compared in 64 bits, or by their logits where
    there is neither bias nor group), and their weights are
    ``scale * s``, divided by the sum of the chosen ``s`` with ``renormalize``.  The weights have a gradient
    with respect to ``logits``; ``bias`` moves the choice alone and gets none.  An expert whose logit or
    biased score is -inf is never chosen; a row with fewer than ``top_k`` others ends with experts -1
    of weight 0.

    :param logits: CUDA tensor (rows, n_experts) of float32, bfloat16 or float16; up to 1024 experts,
        contiguous within a row, any row stride.
    :param top_k: Experts per row, up to 32.
    :param bias: float32 (n_experts,) on the same device, added to the scores for the choice.
    :param n_groups: Groups of neighbouring experts, up to 32, a divisor of the number of experts.
    :param top_groups: Groups whose experts can be chosen (default: all), those with the best scores.
    :param group_score: A group's score: ``"top2"``, the sum of its two highest ``s + bias``, or ``"max"``.
    """
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise TypeError("route takes a CUDA tensor of logits")
    _native.score_dtype(logits)
    logits = _native.plain(logits)
    assert logits.dim() == 2, f"logits must have shape (rows, n_experts), got {tuple(logits.shape)}"
    n = logits.shape[1]
    assert 1 <= n <= _native.MAX_ROUTE_EXPERTS, f"number of experts ({n}) must be in [1, {_native.MAX_ROUTE_EXPERTS}]"
    assert n == 1 or logits.stride(1) == 1, "logits of a row must be contiguous"
    assert scoring in SCORINGS, f"scoring ({scoring!r}) must be one of {tuple(SCORINGS)}"
    assert group_score in GROUP_SCORES, f"group_score ({group_score!r}) must be one of {tuple(GROUP_SCORES)}"
    assert 1 <= n_groups <= 32 and n % n_groups == 0, f"n_groups ({n_groups}) must divide {n} experts and be at most 32"
    top_groups = n_groups if top_groups is None else top_groups
    assert 1 <= top_groups <= n_groups, f"top_groups ({top_groups}) must be in [1, n_groups = {n_groups}]"
    reach = min(n // n_groups * top_groups, _native.MAX_TOP_K)
    assert 1 <= top_k <= reach, f"top_k ({top_k}) must be in [1, {reach}] (the kept groups' experts, at most {_native.MAX_TOP_K})"
    assert math.isfinite(scale), f"scale ({scale}) must be finite"
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.device != logits.device or bias.dtype != torch.float32:
            raise TypeError(f"bias must be a float32 tensor on the device of logits ({logits.device})")
        bias = _native.plain(bias)
        assert bias.shape == (n,) and bias.is_contiguous(), f"bias must be contiguous with shape ({n},), got {tuple(bias.shape)}"
    _no_tangents(logits)
    spec = (int(top_k), SCORINGS[scoring], int(n_groups), int(top_groups), GROUP_SCORES[group_score], bool(renormalize),
            float(scale))
    if logits.requires_grad and torch.is_grad_enabled():
        return Routing(*_Route.apply(logits, bias, spec))
    return Routing(*_native.route(logits, bias, *spec))


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, spec):
        experts, weights = _native.route(logits, bias, *spec)
        ctx.mark_non_differentiable(experts)
        ctx.set_materialize_grads(False)  # or every backward pass would fill a gradient of experts
        ctx.save_for_backward(logits, experts)
        ctx.spec = spec
        return experts, weights

    @staticmethod
    def backward(ctx, _, grad_weights):
        _first_order()
        if grad_weights is None:
            return None, None, None
        logits, experts = ctx.saved_tensors
        top_k, scoring, _, _, _, renormalize, scale = ctx.spec
        return _native.route_backward(logits, experts, _native.plain(grad_weights).contiguous(), scoring, renormalize, scale), None, None


def plan_rows(experts: torch.Tensor, n_experts: int) -> RowPlan:
    """The order that brings entries of the same expert together, entries of one expert in their order.

    :param experts: CUDA tensor (rows, top_k) of int32 or int64, contiguous.  Entries outside
        0 .. n_experts-1 (-1 by convention) take no place.
    :param n_experts: Number of experts, up to 4096.
    """
    if not isinstance(experts, torch.Tensor) or not experts.is_cuda or experts.dtype not in (torch.int32, torch.int64):
        raise TypeError("plan_rows takes a CUDA tensor of int32 or int64 expert numbers")
    assert experts.dim() == 2, f"experts must have shape (rows, top_k), got {tuple(experts.shape)}"
    assert experts.shape[1] >= 1, "experts must have at least one column"
    assert experts.is_contiguous(), "experts must be contiguous"
    assert 1 <= n_experts <= _native.MAX_PLAN_EXPERTS, f"n_experts ({n_experts}) must be in [1, {_native.MAX_PLAN_EXPERTS}]"
    assert experts.numel() < 2**31, f"rows * top_k ({experts.numel()}) must be below 2**31"
    return RowPlan(*_native.plan_rows(experts, int(n_experts)))


def dispatch_rows(data: torch.Tensor, plan: RowPlan) -> torch.Tensor:
    """Rows copied into the plan's order: a tensor (rows * top_k, ...), zeros behind the places in use.

    :param data: CUDA tensor (rows, ...) of any dtype (rows are moved as bytes; a gradient needs float32,
        bfloat16 or float16).  Each row is contiguous; any row stride.
    """
    data = _check_moved(data, plan, "dispatch_rows")
    assert data.shape[0] == plan.slots.shape[0], f"data has {data.shape[0]} rows, the plan {plan.slots.shape[0]}"
    _no_tangents(data)
    if data.requires_grad and torch.is_grad_enabled():
        _native.score_dtype(data)
        return _Dispatch.apply(data, plan.slots, plan.offsets)
    return _native.dispatch_rows(data, plan.slots, plan.offsets)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, data, slots, offsets):
        ctx.save_for_backward(slots)
        return _native.dispatch_rows(data, slots, offsets)

    @staticmethod
    def backward(ctx, grad):
        _first_order()
        (slots,) = ctx.saved_tensors
        return _native.combine_rows(_native.plain(grad).contiguous(), slots, None), None, None


def combine_rows(data: torch.Tensor, plan: RowPlan, weights: torch.Tensor | None = None) -> torch.Tensor:
    """Each row's places summed back: ``out[r] = sum over j of weights[r, j] * data[slots[r, j]]``.

    Sums are taken in 32 bits in the order of j and rounded once; entries without a place are left
    out.  Gradients go to ``data`` and to ``weights``.

    :param data: CUDA tensor (rows * top_k, ...) of float32, bfloat16 or float16 in the plan's order.  Each
        row is contiguous; any row stride.
    :param weights: float32 (rows, top_k), contiguous, on the same device; None sums without weights.
    """
    data = _check_moved(data, plan, "combine_rows")
    _native.score_dtype(data)
    slots = plan.slots
    assert data.shape[0] == slots.numel(), f"data has {data.shape[0]} rows, the plan {slots.numel()} places"
    if weights is not None:
        if not isinstance(weights, torch.Tensor) or weights.device != data.device or weights.dtype != torch.float32:
            raise TypeError(f"weights must be a float32 tensor on the device of data ({data.device})")
        weights = _native.plain(weights)
        assert weights.shape == slots.shape, f"weights must have shape {tuple(slots.shape)}, got {tuple(weights.shape)}"
        assert weights.is_contiguous(), "weights must be contiguous"
    _no_tangents(data, weights)
    if torch.is_grad_enabled() and (data.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(data, weights, slots, plan.offsets)
    return _native.combine_rows(data, slots, weights)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, data, weights, slots, offsets):
        # The rows are read again for the weights' gradient alone.
        ctx.save_for_backward(data if ctx.needs_input_grad[1] else None, weights, slots, offsets)
        return _native.combine_rows(data, slots, weights)

    @staticmethod
    def backward(ctx, grad):
        _first_order()
        data, weights, slots, offsets = ctx.saved_tensors
        return (*_native.combine_backward(_native.plain(grad).contiguous(), data, slots, weights, offsets, *ctx.needs_input_grad[:2]),
                None, None)


def _first_order() -> None:
    """The gradients' kernels have no gradients: refuse ``create_graph=True``, under which a backward
    pass runs with gradients enabled."""
    if torch.is_grad_enabled():
        raise RuntimeError("povs gradients are once differentiable: call backward without create_graph=True")


def _no_tangents(*tensors: torch.Tensor | None) -> None:
    """Refuse dual tensors: the kernels would return their outputs without a tangent."""
    if forward_ad._current_level >= 0:  # inside a dual_level
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("povs gradients are for backward passes: forward-mode differentiation is not supported")


def _check_moved(data: torch.Tensor, plan: RowPlan, what: str) -> torch.Tensor:
    if not isinstance(data, torch.Tensor) or not data.is_cuda:
        raise TypeError(f"{what} takes a CUDA tensor of rows")
    data = _native.plain(data)
    assert data.dim() >= 1, f"data must have at least one dimension, but has {data.dim()}"
    assert data.is_contiguous() or data[:1].is_contiguous(), "rows of data must be contiguous"
    slots, offsets = plan.slots, plan.offsets
    if slots.device != data.device or offsets.device != data.device or slots.dtype != torch.int32 or offsets.dtype != torch.int32:
        raise TypeError(f"plan.slots and plan.offsets must be int32 tensors on the device of data ({data.device})")
    assert slots.is_contiguous() and offsets.is_contiguous(), "plan.slots and plan.offsets must be contiguous"
    assert slots.dim() == 2 and slots.shape[1] >= 1, f"plan.slots must have shape (rows, top_k), got {tuple(slots.shape)}"
    assert offsets.dim() == 1 and offsets.numel() >= 2, "plan.offsets must have shape (n_experts + 1,)"
    return data
