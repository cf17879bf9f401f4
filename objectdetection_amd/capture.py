"""Capture of autograd steps into HIP graphs: a check before the process would end.

PyTorch keeps one gradient accumulator per leaf, bound to the stream on which the first graph that
uses the leaf was built, for as long as any such graph is alive.  A backward pass that is captured on
another stream meanwhile waits for that stream, which is not part of the capture: the capture is
invalidated and the process ends inside the runtime.  guard_leaves notes the stream of the eager
graphs that the differentiable functions of this package build on their leaves (also through a few
views and casts, as `weight.to(dtype).t()`) and refuses the capture instead: when a graph is built
during it, whether or not a backward follows (a forward alone is captured under torch.no_grad()).
Graphs that other functions build on the same leaves are not seen.
"""
from __future__ import annotations

import torch

_KEY = "frcnn_stream"
_DEPTH = 4                    # views and casts looked through between an argument and its leaf


def _accumulator(t: torch.Tensor):
    """The gradient accumulator of the leaf behind t, None if none is near."""
    if t.grad_fn is None:
        return torch.autograd.graph.get_gradient_edge(t).node
    node = t.grad_fn
    for _ in range(_DEPTH):
        nxt = node.next_functions
        if len(nxt) != 1 or nxt[0][0] is None:
            return None
        node = nxt[0][0]
        if hasattr(node, "variable"):
            return node
    return None


def guard_leaves(*tensors):
    """Called before a graph is built; the caller holds the result until it is (the accumulators
    and the notes on them live as long as a graph or this list holds them)."""
    if not torch.is_grad_enabled():
        return None
    held, capturing = [], None
    for t in tensors:
        if not isinstance(t, torch.Tensor) or not t.requires_grad or not t.is_cuda:
            continue
        node = _accumulator(t)
        if node is None:
            continue
        held.append(node)
        stream = torch._C._cuda_getCurrentRawStream(t.device.index)
        if node.metadata.setdefault(_KEY, stream) != stream:
            capturing = torch.cuda.is_current_stream_capturing() if capturing is None else capturing
            if capturing:
                raise RuntimeError(
                    "a backward pass cannot be captured while an autograd graph of the same leaf, built on another "
                    "stream, is alive: release its outputs before the capture, or build it on the capture's stream")
    return held
