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

from typing import NamedTuple, Optional, Tuple

import torch

from ._launch import float_code, int_code, like_or_f32, one_device, rows as _rows, run

MAX_EXPERTS = 1023
MAX_TOP = 64


class ExpertOrder(NamedTuple):
    """Where every assignment went. Assignment ``t * top + j`` is choice j of token t."""
    slots: torch.Tensor    # [tokens, top] int32: its sorted row, -1 if dropped
    sources: torch.Tensor  # [tokens * top] int32: the assignment of each sorted row, -1 behind the last
    offsets: torch.Tensor  # [num_experts + 1] int32: first row of each expert; the last entry counts the kept rows

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
    op = "sort_by_expert"
    icode = int_code(op, "expert_ids", expert_ids)
    if expert_ids.dim() not in (1, 2):
        raise ValueError(f"{op}: expert_ids must be [tokens, top], got shape {tuple(expert_ids.shape)}")
    tokens, top = expert_ids.shape[0], expert_ids.shape[1] if expert_ids.dim() == 2 else 1
    if not 1 <= top <= MAX_TOP:
        raise ValueError(f"{op}: 1 to {MAX_TOP} experts per token, got {top}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"{op}: 1 to {MAX_EXPERTS} experts, got {num_experts}")
    device = one_device(op, expert_ids)
    ids = expert_ids.contiguous()
    dev = expert_ids.device
    slots = torch.empty((tokens, top), dtype=torch.int32, device=dev)
    sources = torch.empty(tokens * top, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    run("bcclExpertSort", device, ids.data_ptr(), icode, tokens, top, num_experts, slots.data_ptr(), sources.data_ptr(),
        offsets.data_ptr())
    return ExpertOrder(slots, sources, offsets)


def _order(op, order, t):
    """(tokens, top, device) of an order whose tensors lie beside ``t``."""
    slots, offsets = order.slots, order.offsets
    if slots.dtype != torch.int32 or slots.dim() != 2 or not slots.is_contiguous() or offsets.dtype != torch.int32 or \
            offsets.dim() != 1 or not offsets.is_contiguous() or not 2 <= offsets.shape[0] <= MAX_EXPERTS + 1 or \
            not 1 <= slots.shape[1] <= MAX_TOP:
        raise ValueError(f"{op}: order must come from sort_by_expert")
    return slots.shape[0], slots.shape[1], one_device(op, t, slots, offsets)


def _sorted(op, what, t, n):
    if t.dim() != 2 or t.shape[0] != n or t.shape[1] < 1:
        raise ValueError(f"{op}: {what} must be [{n}, h], got shape {tuple(t.shape)}")
    return t.contiguous()


def _weights(op, weights, order, dtype):
    if weights is None:
        return None, 0
    code = like_or_f32(op, "weights", weights, dtype)
    if weights.shape != order.slots.shape:
        raise ValueError(f"{op}: weights must be {tuple(order.slots.shape)}, got {tuple(weights.shape)}")
    one_device(op, weights, order.slots)
    return weights.contiguous(), code


def dispatch_forward(x, order: ExpertOrder, out=None):
    """x [tokens, h] -> rows [tokens * top, h] sorted by expert (``out``, contiguous, receives them, e.g. a
    registered send buffer)."""
    op = "dispatch"
    code = float_code(op, "input", x)
    tokens, top, device = _order(op, order, x)
    if x.dim() != 2 or x.shape[0] != tokens or x.shape[1] < 1:
        raise ValueError(f"{op}: input must be [{tokens}, h], got shape {tuple(x.shape)}")
    h = x.shape[1]
    if out is None:
        out = torch.empty(tokens * top, h, dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype or tuple(out.shape) != (tokens * top, h) or not out.is_contiguous():
        raise ValueError(f"{op}: out must be a contiguous {x.dtype} tensor of shape ({tokens * top}, {h})")
    one_device(op, x, out)
    xr, stride = _rows(x)
    run("bcclExpertDispatch", device, xr.data_ptr(), stride, order.slots.data_ptr(), order.offsets.data_ptr(), tokens, top,
        order.num_experts, h, out.data_ptr(), code)
    return out


def _combine(op, rows, order, weights):
    code = float_code(op, "rows", rows)
    tokens, top, device = _order(op, order, rows)
    rows = _sorted(op, "rows", rows, tokens * top)
    w, wcode = _weights(op, weights, order, rows.dtype)
    h = rows.shape[1]
    y = torch.empty(tokens, h, dtype=rows.dtype, device=rows.device)
    run("bcclExpertCombine", device, rows.data_ptr(), order.slots.data_ptr(), None if w is None else w.data_ptr(),
        code if w is None else wcode, tokens, top, h, y.data_ptr(), h, code)
    return y


def dispatch_backward(drows, order: ExpertOrder):
    """The gradient of x: each token's sum over its kept assignments' rows of drows."""
    return _combine("dispatch_backward", drows, order, None)


def combine_forward(rows, order: ExpertOrder, weights=None):
    """rows [tokens * top, h] in sorted order, weights [tokens, top] (None: ones) -> y [tokens, h]."""
    return _combine("combine", rows, order, weights)


def combine_backward(dy, rows, order: ExpertOrder, weights=None, *, weight_grad: bool = True) -> Tuple:
    """(drows, dweights) of :func:`combine_forward`; dweights is None without weights or where it is not
    asked for."""
    op = "combine_backward"
    code = float_code(op, "dy", dy)
    tokens, top, device = _order(op, order, dy)
    if dy.dim() != 2 or dy.shape[0] != tokens or dy.shape[1] < 1:
        raise ValueError(f"{op}: dy must be [{tokens}, h], got shape {tuple(dy.shape)}")
    h = dy.shape[1]
    rows = _sorted(op, "rows", rows, tokens * top)
    if rows.dtype != dy.dtype or rows.shape[1] != h:
        raise ValueError(f"{op}: rows must be {dy.dtype} of width {h}, got {rows.dtype} {tuple(rows.shape)}")
    one_device(op, dy, rows)
    w, wcode = _weights(op, weights, order, dy.dtype)
    d, stride = _rows(dy)
    drows = torch.empty(tokens * top, h, dtype=dy.dtype, device=dy.device)
    dw = torch.empty_like(w) if w is not None and weight_grad else None
    run("bcclExpertCombineBackward", device, d.data_ptr(), stride, rows.data_ptr(), order.slots.data_ptr(),
        order.offsets.data_ptr(), None if w is None else w.data_ptr(), code if w is None else wcode, tokens, top,
        order.num_experts, h, drows.data_ptr(), None if dw is None else dw.data_ptr(), code)
    return drows, dw


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots, sources, offsets):
        ctx.save_for_backward(slots, sources, offsets)
        return dispatch_forward(x, ExpertOrder(slots, sources, offsets))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows):
        return dispatch_backward(drows, ExpertOrder(*ctx.saved_tensors)), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, slots, sources, offsets):
        ctx.save_for_backward(rows, weights, slots, sources, offsets)
        return combine_forward(rows, ExpertOrder(slots, sources, offsets), weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, weights, *order = ctx.saved_tensors
        drows, dw = combine_backward(dy, rows, ExpertOrder(*order), weights, weight_grad=ctx.needs_input_grad[1])
        return drows, dw, None, None, None


def dispatch(x, order: ExpertOrder):
    """Differentiable :func:`dispatch_forward`."""
    return _Dispatch.apply(x, *order)


def combine(rows, order: ExpertOrder, weights: Optional[torch.Tensor] = None):
    """Differentiable :func:`combine_forward` (gradients of rows and weights)."""
    return _Combine.apply(rows, weights, *order)
