"""What the compute ops share: dtype codes, operand checks, the call into the library."""
from __future__ import annotations

import torch

from .. import _native

FLOATS = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}
INTS = {torch.int32: 2, torch.int64: 3}

_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_stream = (torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream")
           else lambda d: torch.cuda.current_stream(d).cuda_stream)


def run(function: str, device: int, *args) -> None:
    """Calls a C entry point with the current stream of ``device`` as its last argument, with that
    device current; raises what the library says when it refuses."""
    fn = getattr(_native.lib(), function)
    if _device() == device:
        rc = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(device))
    if rc != 0:
        raise RuntimeError(_native.last_error())


def float_code(op: str, what: str, t) -> int:
    code = FLOATS.get(t.dtype)
    if code is None:
        raise TypeError(f"{op}: {what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def int_code(op: str, what: str, t) -> int:
    code = INTS.get(t.dtype)
    if code is None:
        raise TypeError(f"{op}: {what} must be int32 or int64, got {t.dtype}")
    return code


def like_or_f32(op: str, what: str, t, dtype) -> int:
    """Code of a parameter next to operands of ``dtype``: the same type, or float32."""
    if t.dtype != dtype and t.dtype != torch.float32:
        raise TypeError(f"{op}: {what} must be {dtype} or float32, got {t.dtype}")
    return FLOATS[t.dtype]


def one_device(op: str, *tensors) -> int:
    """Index of the CUDA device that holds every operand (None entries are skipped)."""
    device = tensors[0].get_device() if tensors[0].is_cuda else -1
    for t in tensors:
        if t is not None and (not t.is_cuda or t.get_device() != device):
            raise ValueError(f"{op}: operands must be CUDA tensors on one device, got "
                             f"{sorted({str(t.device) for t in tensors if t is not None})}")
    return device


def rows(t):
    """``t`` as rows of its last dimension: (tensor to read, row stride). Copies only layouts whose
    rows are not evenly spaced with adjacent elements."""
    h = t.shape[-1]
    if t.is_contiguous():
        return t, h
    if t.dim() == 2 and (h == 1 or t.stride(1) == 1):
        return t, t.stride(0)
    return t.contiguous(), h


def out_rows(op: str, out, shape, dtype):
    """A caller's output of ``shape``: its row stride."""
    if out.dtype != dtype or tuple(out.shape) != tuple(shape):
        raise ValueError(f"{op}: out must be a {dtype} tensor of shape {tuple(shape)}, got {out.dtype} "
                         f"{tuple(out.shape)}")
    h = shape[-1]
    if out.is_contiguous():
        return h
    if out.dim() == 2 and (h == 1 or out.stride(1) == 1) and out.stride(0) >= h:
        return out.stride(0)
    raise ValueError(f"{op}: out must have rows of adjacent elements, evenly spaced and apart")
