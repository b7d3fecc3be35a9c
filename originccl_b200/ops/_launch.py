"""What the compute ops share: dtype codes, operand checks, the call into the library.

The smallest calls are bound by the host (a kernel of 2 us behind some 10 us of Python), so each
operand property is read once and the entry points look nothing up by name.
"""
from __future__ import annotations

import torch

from .. import _native

FLOATS = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}
INTS = {torch.int32: 2, torch.int64: 3}

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_current_stream = (torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream")
                   else lambda d: torch.cuda.current_stream(d).cuda_stream)


class Entry:
    """A C entry point whose last argument is the stream. Calling it with a device index first runs it
    with that device current, on that device's current torch stream, and raises the library's
    message when it refuses."""

    __slots__ = ("name", "fn")

    def __init__(self, name: str) -> None:
        self.name, self.fn = name, None

    def __call__(self, device: int, *args) -> None:
        if self.fn is None:
            self.fn = getattr(_native.lib(), self.name)
        if _current_device() == device:
            rc = self.fn(*args, _current_stream(device))
        else:
            with torch.cuda.device(device):
                rc = self.fn(*args, _current_stream(device))
        if rc != 0:
            raise RuntimeError(_native.last_error())


def float_code(op: str, what: str, dtype) -> int:
    code = FLOATS.get(dtype)
    if code is None:
        raise TypeError(f"{op}: {what} must be float32, bfloat16 or float16, got {dtype}")
    return code


def int_code(op: str, what: str, dtype) -> int:
    code = INTS.get(dtype)
    if code is None:
        raise TypeError(f"{op}: {what} must be int32 or int64, got {dtype}")
    return code


def like_or_f32(op: str, what: str, got, dtype) -> int:
    """Code of a parameter's type next to operands of ``dtype``: the same type, or float32."""
    if got is not dtype and got is not torch.float32:
        raise TypeError(f"{op}: {what} must be {dtype} or float32, got {got}")
    return FLOATS[got]


def one_device(op: str, *tensors) -> int:
    """Index of the CUDA device that holds every operand (None entries are skipped)."""
    device = tensors[0].get_device()  # -1: host memory
    for t in tensors:
        if t is not None and (t.get_device() != device or device < 0):
            raise ValueError(f"{op}: operands must be CUDA tensors on one device, got "
                             f"{sorted({str(t.device) for t in tensors if t is not None})}")
    return device


def ptr(t):
    return None if t is None else t.data_ptr()


def rows(t, h: int):
    """``t`` as rows of its last dimension, of ``h`` elements: (tensor to read, row stride). Copies only
    layouts whose rows are not evenly spaced with adjacent elements."""
    if t.is_contiguous():
        return t, h
    if t.dim() == 2 and (h == 1 or t.stride(1) == 1):
        return t, t.stride(0)
    return t.contiguous(), h


def out_rows(op: str, out, shape, dtype) -> int:
    """A caller's output of ``shape``: its row stride."""
    if out.dtype is not dtype or tuple(out.shape) != tuple(shape):
        raise ValueError(f"{op}: out must be a {dtype} tensor of shape {tuple(shape)}, got {out.dtype} "
                         f"{tuple(out.shape)}")
    h = shape[-1]
    if out.is_contiguous():
        return h
    if out.dim() == 2 and (h == 1 or out.stride(1) == 1) and out.stride(0) >= h:
        return out.stride(0)
    raise ValueError(f"{op}: out must have rows of adjacent elements, evenly spaced and apart")
