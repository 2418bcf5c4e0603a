"""Device time of a call, for tests of the rules that choose between kernels."""
from __future__ import annotations

import statistics

import torch


def device_us(call, operands, nbytes):
    """Median time of call(*operands()) in a CUDA graph of calls on sets of operands, `nbytes` each, that together are
    three times what the L2 holds."""
    sets = [operands() for _ in range(-(-400_000_000 // nbytes))]
    for s in sets:
        call(*s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for s in sets * 2:
            call(*s)
    graph.replay()
    times = []
    for _ in range(15):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end) * 1e3 / (2 * len(sets)))
    return statistics.median(times)
