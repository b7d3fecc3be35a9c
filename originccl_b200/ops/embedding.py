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

import functools
from typing import Optional

import torch

from .. import _native
from ._launch import Entry, float_code, int_code, like_or_f32, one_device, out_rows, rows

_forward, _backward = Entry("bcclEmbeddingForward"), Entry("bcclEmbeddingBackward")


@functools.lru_cache(maxsize=1024)
def _workspace(n: int, num_rows: int, h: int) -> int:
    return _native.lib().bcclEmbeddingBackwardWorkspace(n, num_rows, h)


def _first(op, first_row):
    if first_row < 0:
        raise ValueError(f"{op}: first_row must not be negative, got {first_row}")


def embedding_forward(ids, weight, scale: float = 1.0, first_row: int = 0, out=None):
    """ids [...] (any values), weight [rows, h] -> [..., h] of weight's type."""
    op = "embedding"
    code, icode = float_code(op, "weight", weight.dtype), int_code(op, "ids", ids.dtype)
    shape = weight.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{op}: weight must be 2-D, got shape {tuple(shape)}")
    num_rows, h = shape
    _first(op, first_row)
    device = one_device(op, weight, ids, out)
    ids = ids.contiguous()
    w, stride = rows(weight, h)
    shape = (*ids.shape, h)
    if out is None:
        out, ostride = weight.new_empty(shape), h
    else:
        ostride = out_rows(op, out, shape, weight.dtype)
    _forward(device, ids.data_ptr(), icode, ids.numel(), w.data_ptr(), stride, num_rows, h, first_row, scale,
             out.data_ptr(), ostride, code)
    return out


def embedding_backward(dy, ids, num_rows: int, scale: float = 1.0, first_row: int = 0,
                       padding_idx: Optional[int] = None, out=None, accumulate: bool = False):
    """dy [..., h], ids [...] -> the table's gradient [num_rows, h].

    ``out`` (contiguous, dy's type or float32) receives it; with ``accumulate`` it is added to ``out``,
    rows of absent tokens staying untouched (a step's main gradients, a bucket's view)."""
    op = "embedding_backward"
    code, icode = float_code(op, "dy", dy.dtype), int_code(op, "ids", ids.dtype)
    if dy.dim() < 1 or dy.shape[-1] < 1 or dy.shape[:-1] != ids.shape:
        raise ValueError(f"{op}: dy {tuple(dy.shape)} must be one row per id, ids {tuple(ids.shape)}")
    _first(op, first_row)
    if num_rows < 0 or (padding_idx is not None and padding_idx < 0):
        raise ValueError(f"{op}: num_rows and padding_idx must not be negative")
    if accumulate and out is None:
        raise ValueError(f"{op}: accumulate needs out")
    h = dy.shape[-1]
    device = one_device(op, dy, ids, out)
    if out is None:
        out = dy.new_empty((num_rows, h))
    elif tuple(out.shape) != (num_rows, h) or not out.is_contiguous():
        raise ValueError(f"{op}: out must be a contiguous ({num_rows}, {h}) tensor, got {tuple(out.shape)}")
    ocode = like_or_f32(op, "out", out.dtype, dy.dtype)
    ids = ids.contiguous()
    d, stride = rows(dy, h)
    n = ids.numel()
    size = _workspace(n, num_rows, h)
    ws = dy.new_empty(size, dtype=torch.uint8)
    _backward(device, d.data_ptr(), stride, ids.data_ptr(), icode, n, out.data_ptr(), num_rows, h, first_row, scale,
              padding_idx or 0, padding_idx is not None, accumulate, code, ocode, ws.data_ptr(), size)
    return out


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
    return _Embedding.apply(ids, weight, scale, padding_idx, first_row)
