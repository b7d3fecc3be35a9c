"""Layer norm and RMS norm over the last dimension, forward and backward (``csrc/kernels/norms.cu``).

``y = (x - mean) * rstd * weight + bias`` with ``rstd = 1 / sqrt(var + eps)``; RMS norm has no mean and
no bias. Types: float32, bfloat16, float16; weight and bias have x's type or are float32.
Statistics are float32, sums are kept in 32 bits, outputs are rounded once. Rows may be of any
length; a 2-D input may have any row stride. The weights' gradients are summed in a fixed order.

:func:`layer_norm` and :func:`rms_norm` are differentiable; the ``_forward`` / ``_backward`` pairs are the
same kernels for code that keeps its own activations (pipeline stages, captured steps). The
reference has no compute operators.
"""
from __future__ import annotations

import functools
from typing import Tuple

import torch

from .. import _native
from ._launch import Entry, float_code, like_or_f32, one_device, out_rows, ptr, rows

_LAYER, _RMS = 0, 1
_norm_forward, _norm_backward = Entry("bcclNormForward"), Entry("bcclNormBackward")


@functools.lru_cache(maxsize=1024)
def _workspace(kind: int, n: int, h: int, code: int) -> int:
    return _native.lib().bcclNormBackwardWorkspace(kind, n, h, code)


def _check(op, x, weight, bias):
    """(dtype code, weight's code, row length, contiguous weight and bias)"""
    dtype = x.dtype
    code = float_code(op, "input", dtype)
    shape = x.shape
    h = shape[-1] if shape else 0
    if h < 1:
        raise ValueError(f"{op}: input needs a last dimension of at least 1, got shape {tuple(shape)}")
    if weight is None:
        if bias is not None:
            raise TypeError(f"{op}: bias needs a weight of its own type")
        return code, 0, h, None, None
    wcode = like_or_f32(op, "weight", weight.dtype, dtype)
    if weight.shape != (h,):
        raise ValueError(f"{op}: weight must have shape ({h},), got {tuple(weight.shape)}")
    if bias is not None:
        if bias.dtype is not weight.dtype:
            raise TypeError(f"{op}: bias needs a weight of its own type")
        if bias.shape != (h,):
            raise ValueError(f"{op}: bias must have shape ({h},), got {tuple(bias.shape)}")
        bias = bias.contiguous()
    return code, wcode, h, weight.contiguous(), bias


def _forward(kind, op, x, weight, bias, eps, out):
    code, wcode, h, weight, bias = _check(op, x, weight, bias)
    if not eps >= 0.0:
        raise ValueError(f"{op}: eps must not be negative, got {eps}")
    device = one_device(op, x, weight, bias, out)
    xr, stride = rows(x, h)
    if out is None:
        out, ystride = torch.empty_like(xr, memory_format=torch.contiguous_format), h
    else:
        ystride = out_rows(op, out, x.shape, x.dtype)
    lead = x.shape[:-1]
    mean = x.new_empty(lead, dtype=torch.float32) if kind == _LAYER else None
    rstd = x.new_empty(lead, dtype=torch.float32)
    _norm_forward(device, kind, xr.data_ptr(), stride, ptr(weight), ptr(bias), out.data_ptr(), ystride, ptr(mean),
                  rstd.data_ptr(), x.numel() // h, h, eps, code, wcode)
    return out, mean, rstd


def _backward(kind, op, dy, x, mean, rstd, weight, weight_grad, bias_grad):
    code, wcode, h, weight, _ = _check(op, x, weight, None)
    shape = x.shape
    if dy.dtype is not x.dtype or dy.shape != shape:
        raise ValueError(f"{op}: dy must be {x.dtype} of shape {tuple(shape)}, got {dy.dtype} {tuple(dy.shape)}")
    for what, t in (("mean", mean), ("rstd", rstd)):
        if t is not None and (t.dtype is not torch.float32 or t.shape != shape[:-1] or not t.is_contiguous()):
            raise ValueError(f"{op}: {what} must be the contiguous float32 tensor that the forward pass returned")
    device = one_device(op, x, dy, mean, rstd, weight)
    n = x.numel() // h
    xr, xstride = rows(x, h)
    dyr, dystride = rows(dy, h)
    dx = torch.empty_like(xr, memory_format=torch.contiguous_format)
    dw = torch.empty_like(weight) if weight is not None and weight_grad else None
    db = torch.empty_like(weight) if weight is not None and bias_grad else None
    ws, size = None, 0
    if dw is not None or db is not None:
        size = _workspace(kind, n, h, code)
        ws = x.new_empty(size, dtype=torch.uint8)
    _norm_backward(device, kind, dyr.data_ptr(), dystride, xr.data_ptr(), xstride, ptr(mean), rstd.data_ptr(), ptr(weight),
                   dx.data_ptr(), h, ptr(dw), ptr(db), n, h, code, wcode, ptr(ws), size)
    return dx, dw, db


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5, out=None) -> Tuple:
    """x [..., h] -> (y, mean, rstd); mean and rstd (float32, x's leading shape) are what
    :func:`layer_norm_backward` needs. ``out`` (may be x itself) receives y."""
    return _forward(_LAYER, "layer_norm", x, weight, bias, eps, out)


def layer_norm_backward(dy, x, mean, rstd, weight=None, *, weight_grad: bool = True, bias_grad: bool = True) -> Tuple:
    """(dx, dweight, dbias) of :func:`layer_norm_forward`; without a weight, or where a gradient is not
    asked for, that entry is None. An expanded dy (one row for all) is read as it is."""
    return _backward(_LAYER, "layer_norm_backward", dy, x, mean, rstd, weight, weight_grad, bias_grad)


def rms_norm_forward(x, weight=None, eps: float = 1e-5, out=None) -> Tuple:
    """x [..., h] -> (y, rstd) with ``y = x * rstd * weight``, ``rstd = 1 / sqrt(mean(x^2) + eps)``."""
    y, _, rstd = _forward(_RMS, "rms_norm", x, weight, None, eps, out)
    return y, rstd


def rms_norm_backward(dy, x, rstd, weight=None, *, weight_grad: bool = True) -> Tuple:
    """(dx, dweight) of :func:`rms_norm_forward`."""
    return _backward(_RMS, "rms_norm_backward", dy, x, None, rstd, weight, weight_grad, False)[:2]


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
    return _LayerNorm.apply(x, weight, bias, eps)


def rms_norm(x, weight=None, eps: float = 1e-5):
    """Differentiable RMS norm over the last dimension."""
    return _RmsNorm.apply(x, weight, eps)
