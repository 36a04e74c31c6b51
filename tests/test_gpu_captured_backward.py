"""A captured backward whose leaf lies behind a cast, in the captured graph, the living eager one or both: refused before a gradient
reaches the leaf, and with the eager graph dropped the same capture runs and replays."""
import pytest
import torch

import self_forcing_amd as sfa
from gpu_util import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
l8 = sfa.linear8


def test_a_leaf_behind_a_cast():
    x, dy = randn((1, 40, 128), 1, torch.bfloat16).to(DEV), randn((1, 40, 64), 2, torch.bfloat16).to(DEV)
    w = randn((64, 128), 3).to(DEV).requires_grad_()

    def forward():
        return l8.linear8(x, w.to(torch.bfloat16))

    def step():
        return torch.autograd.grad(forward(), w, dy)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    eager = forward()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        y = forward()
        with pytest.raises(RuntimeError, match="same leaves"):
            torch.autograd.grad(y, w, dy)
        del y
    ref = torch.autograd.grad(eager, w, dy)[0]
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(step(), ref)
        out.zero_()
