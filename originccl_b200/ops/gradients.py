"""Global gradient norm over many tensors, and clipping by it (``csrc/kernels/grad_norm.cu``).

``norm = sqrt(sum of g^2 over all tensors)``, ``c = min(1, max_norm / (norm + eps))``, ``g <- c * g``: three launches
for up to 1024 tensors of one type, no synchronisation with the host, the same sum on every run. Where c is
1 nothing is written in place. A norm that is infinite or NaN makes c 0 or NaN, as in
``torch.nn.utils.clip_grad_norm_``.

Gradients are float32, bfloat16 or float16, mixed if need be, each dense in memory (any order of
dimensions). With ``comm`` the tensors are this rank's shards of the parameters (tensor
parallelism) and the norm is that of all ranks' shards: one AllReduce of the sum of squares
between the launches; every rank of ``comm`` calls it together. Parameters that every rank of ``comm`` holds whole, with
the same gradient (norm weights, say), are named by ``replicated``, a truth value for each gradient: their
squares count once, not once per rank. Host tensors (ranks of a host communicator)
run on torch operations, without the package's extension. The reference has no compute operators.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import _native

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _list(op, grads):
    grads = list(grads)
    if not grads:
        raise ValueError(f"{op}: no gradients")
    return grads


def _replicated(op, grads, replicated, comm):
    """The list of truth values, or None where no rank would count anything twice."""
    if replicated is None:
        return None
    replicated = [bool(r) for r in replicated]
    if len(replicated) != len(grads):
        raise ValueError(f"{op}: {len(grads)} gradients but {len(replicated)} truth values in replicated")
    return replicated if comm is not None and comm.world_size > 1 and any(replicated) else None


def _host(op, grads, comm, replicated, outs=()):
    """The norm of host tensors."""
    for t in (*grads, *outs):
        if t.is_cuda or t.dtype not in _FLOATS:
            raise ValueError(f"{op}: gradients must be float32, bfloat16 or float16 tensors, all on one device")
    for t, o in zip(grads, outs):
        if o.shape != t.shape or o.dtype not in (t.dtype, torch.float32):
            raise ValueError(f"{op}: each out must have its gradient's shape, and its type or float32, got "
                             f"{o.dtype} {tuple(o.shape)} for {t.dtype} {tuple(t.shape)}")
    total = torch.zeros(1, dtype=torch.float64)
    for i, t in enumerate(grads):
        share = comm.world_size if replicated is not None and replicated[i] else 1
        total += t.double().square().sum() / share
    if comm is not None and comm.world_size > 1:
        comm.all_reduce(total)
    return total.sqrt().float()[0]


def grad_norm(grads: Sequence[torch.Tensor], *, comm=None, replicated: Optional[Sequence[bool]] = None):
    """The global norm, a float32 tensor of no dimensions on the gradients' device."""
    grads = _list("grad_norm", grads)
    replicated = _replicated("grad_norm", grads, replicated, comm)
    if not grads[0].is_cuda:
        return _host("grad_norm", grads, comm, replicated)
    ops = _native.ops()
    total = ops.grad_squares(grads, replicated, 1 if replicated is None else comm.world_size)
    if comm is not None and comm.world_size > 1:
        comm.all_reduce(total)
    return ops.grad_norm_of(grads[0], total)


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float, *, eps: float = 1e-6,
                   outs: Optional[Sequence[torch.Tensor]] = None, comm=None,
                   replicated: Optional[Sequence[bool]] = None):
    """Scales the gradients by ``min(1, max_norm / (norm + eps))`` in place, or into ``outs`` (same shapes; the
    gradients' type or float32; memory of their own), and returns the norm from before."""
    op = "clip_grad_norm"
    if not max_norm >= 0.0 or not eps >= 0.0:
        raise ValueError(f"{op}: max_norm and eps must not be negative, got {max_norm} and {eps}")
    grads = _list(op, grads)
    outs = None if outs is None else list(outs)
    if outs is not None and len(outs) != len(grads):
        raise ValueError(f"{op}: {len(grads)} gradients but {len(outs)} outs")
    replicated = _replicated(op, grads, replicated, comm)
    if not grads[0].is_cuda:
        norm = _host(op, grads, comm, replicated, outs or ())
        coef = torch.clamp(max_norm / (norm + eps), max=1.0)
        for t, o in zip(grads, grads if outs is None else outs):
            o.copy_(t.float() * coef)
        return norm
    ranks = 1 if comm is None else comm.world_size
    return _native.ops().grad_clip(grads, outs, max_norm, eps, replicated, ranks, comm.all_reduce if ranks > 1 else None)
