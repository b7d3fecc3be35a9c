"""Global gradient norm over many tensors, and clipping by it (``csrc/kernels/grad_norm.cu``).

``norm = sqrt(sum of g^2 over all tensors)``, ``c = min(1, max_norm / (norm + eps))``, ``g <- c * g``: two launches for up
to 1024 tensors of one type, no synchronisation with the host, the same sum on every run. Where c is
1 nothing is written in place. A norm that is infinite or NaN makes c 0 or NaN, as in
``torch.nn.utils.clip_grad_norm_``.

Gradients are float32, bfloat16 or float16, mixed if need be, each dense in memory (any order of
dimensions). With ``comm`` the tensors are this rank's shards of the parameters (tensor
parallelism) and the norm is that of all ranks' shards: one AllReduce of the partial sums between
the launches; every rank of ``comm`` calls it together. Host tensors (ranks of a host communicator)
run on torch operations. The reference has no compute operators.
"""
from __future__ import annotations

from array import array
from typing import Optional, Sequence

import torch

from ._launch import FLOATS, run

PARTIALS = 592  # doubles that hold the partial sums of squares


def _dense(t) -> bool:
    """Elements fill t's memory without gaps or overlaps, in some order of the dimensions."""
    if t.is_contiguous():
        return True
    n = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != n:
            return False
        n *= size
    return True


class _Group:
    """Pointer and count arrays of the tensors of one type (and of their outputs)."""

    def __init__(self, tensors, outs) -> None:
        first = tensors[0]
        self.code, self.n = FLOATS[first.dtype], len(tensors)
        self.ptrs = array("Q", [t.data_ptr() for t in tensors])
        self.counts = array("Q", [t.numel() for t in tensors])
        self.outs, self.out_code = self.ptrs, self.code
        if outs is not None:
            self.out_code = FLOATS[outs[0].dtype]
            self.outs = array("Q", [t.data_ptr() for t in outs])

    @property
    def inputs(self):
        return self.ptrs.buffer_info()[0], self.counts.buffer_info()[0]


def _groups(op, grads, outs, device, written=True):
    """The tensors by type, checked."""
    for t in grads:
        if t.dtype not in FLOATS:
            raise TypeError(f"{op}: gradients must be float32, bfloat16 or float16, got {t.dtype}")
        if t.get_device() != device:
            raise ValueError(f"{op}: gradients must be CUDA tensors on one device")
        if not t.is_contiguous() and not _dense(t):
            raise ValueError(f"{op}: gradients must be dense in memory, got shape {tuple(t.shape)}, strides {t.stride()}")
    if outs is not None:
        for t, o in zip(grads, outs):
            if o.shape != t.shape or o.get_device() != device or (o.dtype != t.dtype and o.dtype != torch.float32):
                raise ValueError(f"{op}: each out must have its gradient's shape and device, and its type or float32")
            if (o.stride() != t.stride() or not _dense(o)) and not (o.is_contiguous() and t.is_contiguous()):
                raise ValueError(f"{op}: each out must be laid out like its gradient")
            if o.data_ptr() == t.data_ptr() and o.dtype != t.dtype and o.numel():
                raise ValueError(f"{op}: an out in its gradient's place must have its type")
    if written:
        ptrs = [t.data_ptr() for t in (grads if outs is None else outs) if t.numel()]
        if len(set(ptrs)) != len(ptrs):
            raise ValueError(f"{op}: a tensor to be written is listed twice")
    kinds = {}
    for i, t in enumerate(grads):
        key = (t.dtype, None if outs is None else outs[i].dtype)
        kinds.setdefault(key, []).append(i)
    if len(kinds) == 1:
        return [_Group(grads, outs)]
    return [_Group([grads[i] for i in idx], None if outs is None else [outs[i] for i in idx])
            for idx in kinds.values()]


def _partials(groups, device, comm):
    partials = torch.empty(PARTIALS, dtype=torch.float64, device=torch.device("cuda", device))
    for i, g in enumerate(groups):
        run("bcclGradSquares", device, *g.inputs, g.n, g.code, int(i > 0), partials.data_ptr())
    if comm is not None and comm.world_size > 1:
        comm.all_reduce(partials)
    return partials


def _host(grads, comm):
    """The norm of host tensors."""
    total = torch.zeros(1, dtype=torch.float64)
    for t in grads:
        total += t.double().square().sum()
    if comm is not None and comm.world_size > 1:
        comm.all_reduce(total)
    return total.sqrt().float()[0]


def _list(op, grads):
    grads = list(grads)
    if not grads:
        raise ValueError(f"{op}: no gradients")
    return grads, grads[0].is_cuda


def _on_host(op, tensors) -> None:
    for t in tensors:
        if t.is_cuda or t.dtype not in FLOATS:
            raise ValueError(f"{op}: gradients must be float32, bfloat16 or float16 tensors, all on one device")


def grad_norm(grads: Sequence[torch.Tensor], *, comm=None):
    """The global norm, a float32 tensor of no dimensions on the gradients' device."""
    op = "grad_norm"
    grads, cuda = _list(op, grads)
    if not cuda:
        _on_host(op, grads)
        return _host(grads, comm)
    device = grads[0].get_device()
    groups = _groups(op, grads, None, device, written=False)
    partials = _partials(groups, device, comm)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    run("bcclGradClip", device, None, None, None, 0, 0, 0, partials.data_ptr(), 0.0, 0.0, norm.data_ptr())
    return norm


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float, *, eps: float = 1e-6,
                   outs: Optional[Sequence[torch.Tensor]] = None, comm=None):
    """Scales the gradients by ``min(1, max_norm / (norm + eps))`` in place, or into ``outs`` (same shapes; the
    gradients' type or float32), and returns the norm from before."""
    op = "clip_grad_norm"
    grads, cuda = _list(op, grads)
    if not max_norm >= 0.0 or not eps >= 0.0:
        raise ValueError(f"{op}: max_norm and eps must not be negative, got {max_norm} and {eps}")
    if outs is not None:
        outs = list(outs)
        if len(outs) != len(grads):
            raise ValueError(f"{op}: {len(grads)} gradients but {len(outs)} outs")
    if not cuda:
        _on_host(op, grads + (outs or []))
        norm = _host(grads, comm)
        coef = torch.clamp(max_norm / (norm + eps), max=1.0)
        for t, o in zip(grads, grads if outs is None else outs):
            o.copy_(t.float() * coef)
        return norm
    device = grads[0].get_device()
    groups = _groups(op, grads, outs, device)
    partials = _partials(groups, device, comm)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    for i, g in enumerate(groups):
        ptrs, counts = g.inputs
        run("bcclGradClip", device, ptrs, g.outs.buffer_info()[0], counts, g.n, g.code, g.out_code, partials.data_ptr(),
            max_norm, eps, norm.data_ptr() if i == 0 else None)
    return norm
