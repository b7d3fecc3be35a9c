"""A backward pass must not be captured into a CUDA graph while an eager graph of the same leaves lives.

Autograd gives each leaf one accumulation node for as long as any graph refers to it, and runs it on the
stream on which it was made. If an eager forward pass made it on another stream and its output is
still held, a captured backward pass would wait for that stream, which a capture may not do; the
error ends the process. While the current stream captures, :func:`apply` looks up where the nodes of an
operator's leaves were made, by whichever operator, and refuses the capture's forward pass instead.
"""
from __future__ import annotations

import torch

from .. import _native

_ops = _native.ops()
_KEY = "bccl_stream"


def apply(op: str, function, *args):
    """``function.apply(*args)``, behind :func:`guard` where it matters: in a capture, with a graph recorded.
    Without a graph (``no_grad``, ``inference_mode``) no backward pass will wait for anything; without a
    capture it may wait. (Marking the nodes of every eager call took 9 us of host time per parameter.)"""
    if torch.is_grad_enabled() and not torch.is_inference_mode_enabled() and torch.cuda.is_initialized() and \
            torch.cuda.is_current_stream_capturing():
        guard(op, *args)
    return function.apply(*args)


def guard(op: str, *inputs) -> None:
    """Refuses a capture whose backward pass would wait for another stream. A mark in a node's metadata counts
    as the stream on which it was made; one without is marked with what autograd says."""
    for t in inputs:
        if not isinstance(t, torch.Tensor) or not t.requires_grad or not t.is_leaf:
            continue
        stream = torch.cuda.current_stream(t.device).cuda_stream if t.is_cuda else 0
        before = _ops.leaf_stream(t)  # None where no node lives
        marks = torch.autograd.graph.get_gradient_edge(t).node.metadata
        made = marks.setdefault(_KEY, stream if before is None else before)
        if made != stream and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{op}: an eager graph of the same leaf tensors, made on another stream, is still alive; "
                               "release its outputs (the loss) before the backward pass is captured")
