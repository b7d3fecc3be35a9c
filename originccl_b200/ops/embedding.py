"""Embedding lookup with scaling, and its gradient by sorted tokens (``csrc/kernels/embedding.cu``).

``out[i] = scale * weight[ids[i] - first_row]``. ``weight`` may be one rank's rows
``[first_row, first_row + len(weight))`` of a larger table: ids outside them give rows of zeros and no gradient,
so the ranks of a tensor-parallel group add up to the whole lookup with one AllReduce::

    rows = embedding.embedding(ids, shard, first_row=tp.rank * shard.shape[0])
    tp.all_reduce(rows)

The gradient sums, for every token of the table, the rows of dy where it occurs, in 32 bits and in
a fixed order; positions of ``padding_idx`` add nothing. Types: float32, bfloat16, float16; ids
int32 or int64. The reference has no compute operators.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _native
from ._capture import apply

_ops = _native.ops()


def embedding_forward(ids, weight, scale: float = 1.0, first_row: int = 0, out=None):
    """ids [...] (any values), weight [rows, h] -> [..., h] of weight's type."""
    return _ops.embedding_forward(ids, weight, scale, first_row, out)


def embedding_backward(dy, ids, num_rows: int, scale: float = 1.0, first_row: int = 0,
                       padding_idx: Optional[int] = None, out=None, accumulate: bool = False):
    """dy [..., h], ids [...] -> the table's gradient [num_rows, h].

    ``out`` (contiguous, dy's type or float32) receives it; with ``accumulate`` it is added to ``out``,
    rows of absent tokens staying untouched (a step's main gradients, a bucket's view)."""
    return _ops.embedding_backward(dy, ids, num_rows, scale, first_row, padding_idx, out, accumulate)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, first_row):
        ctx.save_for_backward(ids)
        ctx.args = weight.shape[0], scale, first_row, padding_idx
        return embedding_forward(ids, weight, scale, first_row)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        n, scale, first_row, padding_idx = ctx.args
        return None, embedding_backward(dy, ids, n, scale, first_row, padding_idx), None, None, None


def embedding(ids, weight, scale: float = 1.0, padding_idx: Optional[int] = None, first_row: int = 0):
    """Differentiable lookup; the gradient is dense. ``padding_idx`` is an id of the whole table whose
    positions are looked up but add nothing to the gradient."""
    if padding_idx is not None and padding_idx < 0:
        raise ValueError(f"embedding: padding_idx must not be negative, got {padding_idx}")
    return apply("embedding", _Embedding, ids, weight, scale, padding_idx, first_row)
