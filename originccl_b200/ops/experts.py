"""Tokens sorted by expert and back, with weights applied (``csrc/kernels/experts.cu``).

What goes before and after the exchange of expert parallelism (:meth:`Communicator.all_to_all`,
or ``dist.all_to_all_single`` with uneven splits on the torch backend)::

    order = experts.sort_by_expert(expert_ids, num_experts)        # expert_ids [tokens, top]
    rows = experts.dispatch(x, order)                              # [tokens * top, h], expert by expert
    answers = ...                                                  # expert e: rows offsets[e]:offsets[e + 1]
    y = experts.combine(answers, order, weights)                   # y[t] = sum_j weights[t, j] * answer of (t, j)

The order is stable: an expert's rows stay in the order of the tokens. Ids outside
``[0, num_experts)`` (conventionally -1) drop the assignment: no row, weight zero, gradient zero. The rows
behind the last kept one are zeros. Types: float32, bfloat16, float16; weights have the rows' type
or are float32; sums are kept in 32 bits. Nothing synchronises with the host. The reference has
neither AllToAll nor compute operators.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native
from ._capture import apply

MAX_EXPERTS = 1023
MAX_TOP = 64

_ops = _native.ops()


class ExpertOrder:
    """Where every assignment went; assignment ``t * top + j`` is choice j of token t.

    ``slots`` [tokens, top] int32: its sorted row, -1 if dropped. ``sources`` [tokens * top] int32: the
    assignment of each sorted row, -1 behind the last. ``offsets`` [num_experts + 1] int32: the first row of
    each expert; the last entry counts the kept rows."""

    __slots__ = ("slots", "sources", "offsets")

    def __init__(self, slots, sources, offsets) -> None:
        for t, dim in ((slots, 2), (sources, 1), (offsets, 1)):
            if t.dtype is not torch.int32 or t.dim() != dim or not t.is_contiguous():
                raise ValueError("ExpertOrder: slots, sources and offsets must come from sort_by_expert")
        if not 1 <= slots.shape[1] <= MAX_TOP or not 2 <= offsets.shape[0] <= MAX_EXPERTS + 1 or \
                sources.shape[0] != slots.numel() or slots.device != offsets.device or slots.device != sources.device:
            raise ValueError("ExpertOrder: slots, sources and offsets must come from sort_by_expert")
        self.slots, self.sources, self.offsets = slots, sources, offsets

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    def rank_counts(self, world: int) -> torch.Tensor:
        """Rows for each of ``world`` ranks that hold equal, consecutive shares of the experts (the
        split sizes of the exchange), as an int32 tensor on the device."""
        if world < 1 or self.num_experts % world:
            raise ValueError(f"rank_counts: {self.num_experts} experts do not split over {world} ranks")
        return self.offsets[::self.num_experts // world].diff()


def sort_by_expert(expert_ids, num_experts: int) -> ExpertOrder:
    """expert_ids [tokens, top] (or [tokens]) int32 or int64 -> :class:`ExpertOrder`."""
    order = ExpertOrder.__new__(ExpertOrder)
    order.slots, order.sources, order.offsets = _ops.expert_sort(expert_ids, num_experts)
    return order


def dispatch_forward(x, order: ExpertOrder, out=None):
    """x [tokens, h] -> rows [tokens * top, h] sorted by expert (``out``, contiguous, receives them, e.g. a
    registered send buffer)."""
    return _ops.dispatch(x, order.slots, order.offsets, out)


def dispatch_backward(drows, order: ExpertOrder):
    """The gradient of x: each token's sum over its kept assignments' rows of drows."""
    return _ops.combine(drows, order.slots, order.offsets, None)


def combine_forward(rows, order: ExpertOrder, weights=None):
    """rows [tokens * top, h] in sorted order, weights [tokens, top] (None: ones) -> y [tokens, h]."""
    return _ops.combine(rows, order.slots, order.offsets, weights)


def combine_backward(dy, rows, order: ExpertOrder, weights=None, *, weight_grad: bool = True) -> Tuple:
    """(drows, dweights) of :func:`combine_forward`; dweights is None without weights or where it is not
    asked for."""
    return _ops.combine_backward(dy, rows, order.slots, order.offsets, weights, weight_grad)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.order = order
        return dispatch_forward(x, order)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows):
        return dispatch_backward(drows, ctx.order), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        ctx.save_for_backward(rows, weights)
        ctx.order = order
        return combine_forward(rows, order, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, weights = ctx.saved_tensors
        drows, dw = combine_backward(dy, rows, ctx.order, weights, weight_grad=ctx.needs_input_grad[1])
        return drows, dw, None


def dispatch(x, order: ExpertOrder):
    """Differentiable :func:`dispatch_forward`."""
    return apply("dispatch", _Dispatch, x, order)


def combine(rows, order: ExpertOrder, weights: Optional[torch.Tensor] = None):
    """Differentiable :func:`combine_forward` (gradients of rows and weights)."""
    return apply("combine", _Combine, rows, weights, order)
