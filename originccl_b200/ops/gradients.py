"""Global gradient norm over many tensors, and clipping by it (``csrc/kernels/grad_norm.cu``).

``norm = sqrt(sum of g^2 over all tensors)``, ``c = min(1, max_norm / (norm + eps))``, ``g <- c * g``: three launches
for up to 1024 tensors of one type, no synchronisation with the host, the same sum on every run. Where c is
1 nothing is written in place. A norm that is infinite or NaN makes c 0 or NaN, as in
``torch.nn.utils.clip_grad_norm_``.

Gradients are float32, bfloat16 or float16, mixed if need be, each dense in memory (any order of
dimensions). With ``comm`` the tensors are this rank's shards of the parameters (tensor
parallelism) and the norm is that of all ranks' shards: one AllReduce of the sum of squares
between the launches; every rank of ``comm`` calls it together. Host tensors (ranks of a host communicator)
run on torch operations. The reference has no compute operators.
"""
from __future__ import annotations

from array import array
from operator import attrgetter
from typing import NamedTuple, Optional, Sequence

import torch

from .. import _native
from ._launch import FLOATS, Entry

_squares, _clip = Entry("bcclGradSquares"), Entry("bcclGradClip")


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


def _apart_in_python(written, counts, size, read, read_counts, read_size) -> bool:
    """No tensor written overlaps another one or any of the tensors read (arrays of 64-bit words)."""
    ranges = [(p, p + n * size, True) for p, n in zip(array("Q", written), array("Q", counts)) if n]
    ranges += [(p, p + n * read_size, False) for p, n in zip(array("Q", read), array("Q", read_counts)) if n]
    any_end = written_end = 0
    for start, end, w in sorted(ranges):
        if start < (any_end if w else written_end):
            return False
        any_end = max(any_end, end)
        written_end = max(written_end, end) if w else written_end
    return True


_T = torch.Tensor
_dtype = attrgetter("dtype")
_SIZES = {0: 4, 4: 2, 5: 2}  # of the type codes
_lists = _native.tensor_list()
_describe = _lists.describe if _lists else (lambda tensors: None)
_apart = _lists.apart if _lists else _apart_in_python


class _Group(NamedTuple):
    """The tensors of one type: host arrays of their (and their outputs') pointers and element counts."""
    n: int
    code: int
    ptrs: bytes
    counts: bytes
    total: int
    out_code: int
    outs: bytes


def _check_list(op, tensors, device):
    """Checks types, device and layout of a list; returns the types and whether all are contiguous."""
    dtypes = set(map(_dtype, tensors))
    if not dtypes <= FLOATS.keys():
        raise TypeError(f"{op}: tensors must be float32, bfloat16 or float16, got {sorted(map(str, dtypes))}")
    if set(map(_T.get_device, tensors)) != {device}:
        raise ValueError(f"{op}: gradients and outs must be CUDA tensors on one device")
    plain = all(map(_T.is_contiguous, tensors))
    if not plain:
        for t in tensors:
            if not _dense(t):
                raise ValueError(f"{op}: tensors must be dense in memory, got shape {tuple(t.shape)}, strides "
                                 f"{t.stride()}")
    return dtypes, plain


def _groups(op, grads, outs, device, written=True):
    """The tensors by type, checked."""
    a = _describe(grads)
    b = a if outs is None else _describe(outs)
    if a is not None and b is not None and a[4] == b[4] == device and b[1] == a[1] and (b[3] == a[3] or b[3] == 0):
        group = _Group(len(grads), a[3], a[0], a[1], a[2], b[3], b[0])
        if written:
            size = _SIZES[a[3]]
            if outs is None or (b[0] == a[0] and b[3] == a[3]):
                apart = _apart(a[0], a[1], size, b"", b"", 0)
            else:
                apart = _apart(b[0], a[1], _SIZES[b[3]], a[0], a[1], size)
            if not apart:
                raise ValueError(f"{op}: tensors to be written overlap")
        return [group]
    # Lists of mixed types or layouts, and whatever is to be refused.
    dtypes, plain = _check_list(op, grads, device)
    ptrs, counts = list(map(_T.data_ptr, grads)), list(map(_T.numel, grads))
    optrs, odtypes = ptrs, dtypes
    if outs is not None:
        odtypes, oplain = _check_list(op, outs, device)
        optrs = list(map(_T.data_ptr, outs))
        same = list(map(_T.numel, outs)) == counts
        if not (plain and oplain):  # laid out alike, whatever the order of the dimensions
            same = same and all(o.shape == t.shape and (o.stride() == t.stride() or
                                                        (o.is_contiguous() and t.is_contiguous()))
                                for t, o in zip(grads, outs))
        if not same:
            raise ValueError(f"{op}: each out must have its gradient's shape and layout")
    if len(dtypes) == 1 and len(odtypes) == 1:
        kinds = {(*dtypes, *odtypes): None}
    else:
        kinds = {}
        for i, t in enumerate(grads):
            kinds.setdefault((t.dtype, t.dtype if outs is None else outs[i].dtype), []).append(i)
    result = []
    for (dtype, odtype), idx in kinds.items():
        if odtype != dtype and odtype != torch.float32:
            raise TypeError(f"{op}: an out has its gradient's type or float32, got {odtype} for {dtype}")
        idx = range(len(ptrs)) if idx is None else idx
        pack = lambda v: array("Q", [v[i] for i in idx]).tobytes()  # noqa: E731
        result.append(_Group(len(idx), FLOATS[dtype], pack(ptrs), pack(counts), sum(counts[i] for i in idx), FLOATS[odtype],
                             pack(optrs)))
    if written:  # in bytes, over all types at once
        words = lambda v: array("Q", v).tobytes()  # noqa: E731
        lists = [(words(ptrs), words(c * _SIZES[FLOATS[t.dtype]] for c, t in zip(counts, grads)), 1)]
        if outs is not None:
            lists.insert(0, (words(optrs), words(c * _SIZES[FLOATS[t.dtype]] for c, t in zip(counts, outs)), 1))
        if len(lists) == 1 or lists[0] == lists[1]:
            lists[1:] = [(b"", b"", 0)]
        if not _apart(*lists[0], *lists[1]):
            raise ValueError(f"{op}: tensors to be written overlap")
    return result


def _sum_of_squares(like, groups, device, comm):
    total = like.new_empty(1, dtype=torch.float64)
    for i, g in enumerate(groups):
        # A double per 32 KiB of gradients, two more per tensor for its ends (BCCL_GRAD_WORKSPACE).
        size = 8 * (g.total // 8192 + 2 * g.n + 1)
        ws = like.new_empty(size, dtype=torch.uint8)
        _squares(device, g.ptrs, g.counts, g.n, g.code, i > 0, total.data_ptr(), ws.data_ptr(), size)
    if comm is not None and comm.world_size > 1:
        comm.all_reduce(total)
    return total


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
    total = _sum_of_squares(grads[0], groups, device, comm)
    norm = grads[0].new_empty((), dtype=torch.float32)
    _clip(device, None, None, None, 0, 0, 0, total.data_ptr(), 0.0, 0.0, norm.data_ptr())
    return norm


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float, *, eps: float = 1e-6,
                   outs: Optional[Sequence[torch.Tensor]] = None, comm=None):
    """Scales the gradients by ``min(1, max_norm / (norm + eps))`` in place, or into ``outs`` (same shapes; the
    gradients' type or float32; memory of their own), and returns the norm from before."""
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
    total = _sum_of_squares(grads[0], groups, device, comm)
    norm = grads[0].new_empty((), dtype=torch.float32)
    for i, g in enumerate(groups):
        _clip(device, g.ptrs, g.outs, g.counts, g.n, g.code, g.out_code, total.data_ptr(), max_norm, eps,
              norm.data_ptr() if i == 0 else None)
    return norm
