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

from ._launch import Entry, float_code, int_code, like_or_f32, one_device, ptr, rows as _rows

MAX_EXPERTS = 1023
MAX_TOP = 64

_sort, _dispatch = Entry("bcclExpertSort"), Entry("bcclExpertDispatch")
_combine, _combine_backward = Entry("bcclExpertCombine"), Entry("bcclExpertCombineBackward")


class ExpertOrder:
    """Where every assignment went; assignment ``t * top + j`` is choice j of token t.

    ``slots`` [tokens, top] int32: its sorted row, -1 if dropped. ``sources`` [tokens * top] int32: the
    assignment of each sorted row, -1 behind the last. ``offsets`` [num_experts + 1] int32: the first row of
    each expert; the last entry counts the kept rows."""

    __slots__ = ("slots", "sources", "offsets", "tokens", "top", "num_experts", "device")

    def __init__(self, slots, sources, offsets) -> None:
        for t, dim in ((slots, 2), (sources, 1), (offsets, 1)):
            if t.dtype is not torch.int32 or t.dim() != dim or not t.is_contiguous():
                raise ValueError("ExpertOrder: slots, sources and offsets must come from sort_by_expert")
        self.slots, self.sources, self.offsets = slots, sources, offsets
        self.tokens, self.top = slots.shape
        self.num_experts = offsets.shape[0] - 1
        if not 1 <= self.top <= MAX_TOP or not 1 <= self.num_experts <= MAX_EXPERTS or sources.shape[0] != slots.numel():
            raise ValueError("ExpertOrder: slots, sources and offsets must come from sort_by_expert")
        self.device = one_device("ExpertOrder", slots, sources, offsets)

    def rank_counts(self, world: int) -> torch.Tensor:
        """Rows for each of ``world`` ranks that hold equal, consecutive shares of the experts (the
        split sizes of the exchange), as an int32 tensor on the device."""
        if world < 1 or self.num_experts % world:
            raise ValueError(f"rank_counts: {self.num_experts} experts do not split over {world} ranks")
        return self.offsets[::self.num_experts // world].diff()


def sort_by_expert(expert_ids, num_experts: int) -> ExpertOrder:
    """expert_ids [tokens, top] (or [tokens]) int32 or int64 -> :class:`ExpertOrder`."""
    op = "sort_by_expert"
    icode = int_code(op, "expert_ids", expert_ids.dtype)
    shape = expert_ids.shape
    if len(shape) not in (1, 2):
        raise ValueError(f"{op}: expert_ids must be [tokens, top], got shape {tuple(shape)}")
    tokens, top = shape if len(shape) == 2 else (shape[0], 1)
    if not 1 <= top <= MAX_TOP:
        raise ValueError(f"{op}: 1 to {MAX_TOP} experts per token, got {top}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"{op}: 1 to {MAX_EXPERTS} experts, got {num_experts}")
    device = one_device(op, expert_ids)
    ids = expert_ids.contiguous()
    slots = ids.new_empty((tokens, top), dtype=torch.int32)
    sources = ids.new_empty(tokens * top, dtype=torch.int32)
    offsets = ids.new_empty(num_experts + 1, dtype=torch.int32)
    _sort(device, ids.data_ptr(), icode, tokens, top, num_experts, slots.data_ptr(), sources.data_ptr(), offsets.data_ptr())
    return ExpertOrder(slots, sources, offsets)


def _rows_of(op, what, t, n, order):
    """Width of ``t``, which must be [n, h] beside the order."""
    shape = t.shape
    if len(shape) != 2 or shape[0] != n or shape[1] < 1:
        raise ValueError(f"{op}: {what} must be [{n}, h], got shape {tuple(shape)}")
    if t.get_device() != order.device:
        raise ValueError(f"{op}: {what} must be a CUDA tensor on the order's device, got {t.device}")
    return shape[1]


def _weights(op, weights, order, dtype, code):
    if weights is None:
        return None, code
    wcode = like_or_f32(op, "weights", weights.dtype, dtype)
    if weights.shape != (order.tokens, order.top) or weights.get_device() != order.device:
        raise ValueError(f"{op}: weights must be ({order.tokens}, {order.top}) on the order's device, got "
                         f"{tuple(weights.shape)} on {weights.device}")
    return weights.contiguous(), wcode


def dispatch_forward(x, order: ExpertOrder, out=None):
    """x [tokens, h] -> rows [tokens * top, h] sorted by expert (``out``, contiguous, receives them, e.g. a
    registered send buffer)."""
    op = "dispatch"
    code = float_code(op, "input", x.dtype)
    h = _rows_of(op, "input", x, order.tokens, order)
    n = order.tokens * order.top
    if out is None:
        out = x.new_empty((n, h))
    elif out.dtype is not x.dtype or _rows_of(op, "out", out, n, order) != h or not out.is_contiguous():
        raise ValueError(f"{op}: out must be a contiguous {x.dtype} tensor of shape ({n}, {h})")
    xr, stride = _rows(x, h)
    _dispatch(order.device, xr.data_ptr(), stride, order.slots.data_ptr(), order.offsets.data_ptr(), order.tokens, order.top,
              order.num_experts, h, out.data_ptr(), code)
    return out


def _combine_rows(op, rows, order, weights):
    code = float_code(op, "rows", rows.dtype)
    h = _rows_of(op, "rows", rows, order.tokens * order.top, order)
    w, wcode = _weights(op, weights, order, rows.dtype, code)
    rows = rows.contiguous()
    y = rows.new_empty((order.tokens, h))
    _combine(order.device, rows.data_ptr(), order.slots.data_ptr(), ptr(w), wcode, order.tokens, order.top, h, y.data_ptr(),
             h, code)
    return y


def dispatch_backward(drows, order: ExpertOrder):
    """The gradient of x: each token's sum over its kept assignments' rows of drows."""
    return _combine_rows("dispatch_backward", drows, order, None)


def combine_forward(rows, order: ExpertOrder, weights=None):
    """rows [tokens * top, h] in sorted order, weights [tokens, top] (None: ones) -> y [tokens, h]."""
    return _combine_rows("combine", rows, order, weights)


def combine_backward(dy, rows, order: ExpertOrder, weights=None, *, weight_grad: bool = True) -> Tuple:
    """(drows, dweights) of :func:`combine_forward`; dweights is None without weights or where it is not
    asked for."""
    op = "combine_backward"
    code = float_code(op, "dy", dy.dtype)
    h = _rows_of(op, "dy", dy, order.tokens, order)
    n = order.tokens * order.top
    if _rows_of(op, "rows", rows, n, order) != h or rows.dtype is not dy.dtype:
        raise ValueError(f"{op}: rows must be {dy.dtype} of width {h}, got {rows.dtype} {tuple(rows.shape)}")
    w, wcode = _weights(op, weights, order, dy.dtype, code)
    rows = rows.contiguous()
    d, stride = _rows(dy, h)
    drows = dy.new_empty((n, h))
    dw = torch.empty_like(w) if w is not None and weight_grad else None
    _combine_backward(order.device, d.data_ptr(), stride, rows.data_ptr(), order.slots.data_ptr(), order.offsets.data_ptr(),
                      ptr(w), wcode, order.tokens, order.top, order.num_experts, h, drows.data_ptr(), ptr(dw), code)
    return drows, dw


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
    return _Dispatch.apply(x, order)


def combine(rows, order: ExpertOrder, weights: Optional[torch.Tensor] = None):
    """Differentiable :func:`combine_forward` (gradients of rows and weights)."""
    return _Combine.apply(rows, weights, order)
