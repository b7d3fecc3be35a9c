"""Layer norm and RMS norm over the last dimension, forward and backward (``csrc/kernels/norms.cu``).

``y = (x - mean) * rstd * weight + bias`` with ``rstd = 1 / sqrt(var + eps)``; RMS norm has no mean and
no bias. Types: float32, bfloat16, float16; weight and bias have x's type or are float32.
Statistics are float32, sums are kept in 32 bits, outputs are rounded once. Rows may have up
to 2^23 elements; a 2-D input may have any row stride. The weights' gradients are summed in a fixed order.

:func:`layer_norm` and :func:`rms_norm` are differentiable; the ``_forward`` / ``_backward`` pairs are the
same kernels for code that keeps its own activations (pipeline stages, captured steps). The
reference has no compute operators.
"""
from __future__ import annotations

from typing import Tuple

import torch

from .. import _native
from ._capture import apply

_LAYER, _RMS = 0, 1
_ops = _native.ops()


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5, out=None) -> Tuple:
    """x [..., h] -> (y, mean, rstd); mean and rstd (float32, x's leading shape) are what
    :func:`layer_norm_backward` needs. ``out`` (may be x itself) receives y."""
    return _ops.norm_forward(_LAYER, x, weight, bias, eps, out)


def layer_norm_backward(dy, x, mean, rstd, weight=None, *, weight_grad: bool = True, bias_grad: bool = True) -> Tuple:
    """(dx, dweight, dbias) of :func:`layer_norm_forward`; without a weight, or where a gradient is not
    asked for, that entry is None. An expanded dy (one row for all) is read as it is."""
    return _ops.norm_backward(_LAYER, dy, x, mean, rstd, weight, weight_grad, bias_grad)


def rms_norm_forward(x, weight=None, eps: float = 1e-5, out=None) -> Tuple:
    """x [..., h] -> (y, rstd) with ``y = x * rstd * weight``, ``rstd = 1 / sqrt(mean(x^2) + eps)``."""
    return _ops.norm_forward(_RMS, x, weight, None, eps, out)


def rms_norm_backward(dy, x, rstd, weight=None, *, weight_grad: bool = True) -> Tuple:
    """(dx, dweight) of :func:`rms_norm_forward`."""
    return _ops.norm_backward(_RMS, dy, x, None, rstd, weight, weight_grad, False)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, weight_grad=need[1], bias_grad=need[2])
        return dx if need[0] else None, dw, db, None


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        y, rstd = rms_norm_forward(x, weight, eps)
        ctx.save_for_backward(x, weight, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw = rms_norm_backward(dy, x, rstd, weight, weight_grad=need[1])
        return dx if need[0] else None, dw, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """Differentiable layer norm over the last dimension."""
    return apply("layer_norm", _LayerNorm, x, weight, bias, eps)


def rms_norm(x, weight=None, eps: float = 1e-5):
    """Differentiable RMS norm over the last dimension."""
    return apply("rms_norm", _RmsNorm, x, weight, eps)
