"""Capture into a HIP graph that replays as it ran."""

import gc
from typing import Any, Callable, Iterable, Tuple

import torch


def capture_graph(fn: Callable[[], Any]) -> Tuple[torch.cuda.CUDAGraph, Any]:
    """Captures ``fn()``; (the graph, ready to replay, and fn's result).

    Libraries record hipMemsetAsync where they clear workspaces and results.
    Replays after the first get such nodes wrong on this hardware, so they are
    replaced by fill kernels (ops/hip/graph_fill.hip) before the graph is
    instantiated. Where ``fn`` runs a backward pass, no eager graph of the
    same parameters may be alive (``eager_graph_of``)."""
    from .. import ops
    ext = ops._load_extension()
    if ext is None:
        raise RuntimeError('capture_graph: the mgproto_hip extension is '
                           'required: it replaces memset nodes, which replay '
                           'wrongly')
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = fn()
    ext.graph_fill_nodes(graph.raw_cuda_graph())
    graph.instantiate()
    return graph, out


def eager_graph_of(params: Iterable[torch.Tensor]) -> bool:
    """Whether an autograd graph of one of the parameters is alive: its nodes
    belong to the stream it was made on, and a captured backward pass that meets
    them breaks the capture."""
    from .. import ops
    ext = ops._load_extension()
    if ext is None:
        return False                          # and no capture
    params = list(params)
    if ext.grad_graph_alive(params):
        gc.collect()                          # it may hang in a cycle
        return ext.grad_graph_alive(params)
    return False
