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

from typing import Tuple

import torch

from .. import _native
from ._launch import float_code, like_or_f32, one_device, out_rows, rows, run

_LAYER, _RMS = 0, 1


def _check(op, x, weight, bias):
    code = float_code(op, "input", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{op}: input needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    wcode = 0 if weight is None else like_or_f32(op, "weight", weight, x.dtype)
    for what, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if weight is None or p.dtype != weight.dtype:
            raise TypeError(f"{op}: bias needs a weight of its own type")
        if p.dim() != 1 or p.shape[0] != x.shape[-1]:
            raise ValueError(f"{op}: {what} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
    return code, wcode


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dense(p):
    return None if p is None else p.contiguous()


def _forward(kind, op, x, weight, bias, eps, out):
    code, wcode = _check(op, x, weight, bias)
    if not eps >= 0.0:
        raise ValueError(f"{op}: eps must not be negative, got {eps}")
    device = one_device(op, x, weight, bias, out)
    h, lead = x.shape[-1], x.shape[:-1]
    xr, stride = rows(x)
    weight, bias = _dense(weight), _dense(bias)
    if out is None:
        out, ystride = torch.empty(x.shape, dtype=x.dtype, device=x.device), h
    else:
        ystride = out_rows(op, out, x.shape, x.dtype)
    mean = torch.empty(lead, dtype=torch.float32, device=x.device) if kind == _LAYER else None
    rstd = torch.empty(lead, dtype=torch.float32, device=x.device)
    run("bcclNormForward", device, kind, xr.data_ptr(), stride, _ptr(weight), _ptr(bias), out.data_ptr(), ystride,
        _ptr(mean), rstd.data_ptr(), x.numel() // h, h, eps, code, wcode)
    return out, mean, rstd


def _backward(kind, op, dy, x, mean, rstd, weight, weight_grad, bias_grad):
    code, wcode = _check(op, x, weight, None)
    if dy.dtype != x.dtype or dy.shape != x.shape:
        raise ValueError(f"{op}: dy must be {x.dtype} of shape {tuple(x.shape)}, got {dy.dtype} {tuple(dy.shape)}")
    for what, t in (("mean", mean), ("rstd", rstd)):
        if t is not None and (t.dtype != torch.float32 or t.shape != x.shape[:-1] or not t.is_contiguous()):
            raise ValueError(f"{op}: {what} must be the contiguous float32 tensor that the forward pass returned")
    device = one_device(op, x, dy, mean, rstd, weight)
    h = x.shape[-1]
    n = x.numel() // h
    xr, xstride = rows(x)
    dyr, dystride = rows(dy)
    weight = _dense(weight)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty_like(weight) if weight is not None and weight_grad else None
    db = torch.empty_like(weight) if weight is not None and bias_grad else None
    ws, size = None, 0
    if dw is not None or db is not None:
        size = _native.lib().bcclNormBackwardWorkspace(kind, n, h, code)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    run("bcclNormBackward", device, kind, dyr.data_ptr(), dystride, xr.data_ptr(), xstride, _ptr(mean), rstd.data_ptr(),
        _ptr(weight), dx.data_ptr(), h, _ptr(dw), _ptr(db), n, h, code, wcode, _ptr(ws), size)
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
