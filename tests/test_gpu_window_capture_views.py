"""A captured step on views of a leaf, [B, L, H, D] seen as [B, H, L, D]: refused beside a living eager graph of that leaf, right without one."""
import pytest
import torch

import landmark_attention_b200 as P
from test_gpu_window import inputs, run

pytestmark = pytest.mark.gpu


def test_views_of_leaves():
    q, k, v, g = inputs(torch.bfloat16, 1, 4, 2, 200, 200, 64, 9)
    want = run(q, k, v, g, 100, 3)
    leaves = [t.transpose(1, 2).contiguous().requires_grad_(True) for t in (q, k, v)]

    def step():
        o = P.window_attention(*[t.transpose(1, 2) for t in leaves], 100, sinks=3)
        return o, torch.autograd.grad(o, leaves, g)

    alive = P.window_attention(*[t.transpose(1, 2) for t in leaves], 100, sinks=3)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="same leaf"):
        with torch.cuda.graph(graph):
            torch.zeros(1, device="cuda")
            step()
    del alive, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, grads = step()
    graph.replay()
    assert torch.equal(o, want[0]) and all(torch.equal(a.transpose(1, 2), b) for a, b in zip(grads, want[1:]))
