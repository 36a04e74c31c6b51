"""Which captured backwards are refused, without a GPU: a leaf counts wherever in either graph it is."""
import pytest
import torch

import self_forcing_amd as sfa

blk = sfa.block_ops


class _Twice(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        blk._noted(ctx, x.device)
        return x * 2 + w

    @staticmethod
    @blk._once
    def backward(ctx, dy):
        return dy * 2, dy


@pytest.fixture
def captured(monkeypatch):
    stream, capturing = [0], [False]
    monkeypatch.setattr(blk, "_raw_stream", lambda index: stream[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])

    def run(make, leaf):
        stream[0], capturing[0] = 5, True
        try:
            return torch.autograd.grad(make().sum(), leaf)[0]
        finally:
            stream[0], capturing[0] = 0, False
    return run


SHAPES = {"itself": lambda w: w, "cast": lambda w: w.double(), "strided": lambda w: w.expand(2, 4).t()[:, 0].contiguous(),
          "through another layer": lambda w: torch.tanh(w * 3)}


@pytest.mark.parametrize("eager", SHAPES)
@pytest.mark.parametrize("graph", SHAPES)
def test_a_leaf_behind_other_operators_counts(captured, eager, graph):
    w, v = (torch.randn(4, requires_grad=True) for _ in range(2))
    lives = _Twice.apply(torch.ones(4), SHAPES[eager](w)).sum()
    make = lambda leaf: lambda: _Twice.apply(torch.ones(4), SHAPES[graph](leaf))
    with pytest.raises(RuntimeError, match="same leaves"):
        captured(make(w), w)
    captured(make(v), v)
    del lives
    captured(make(w), w)


def test_a_deep_graph_is_walked(captured):
    w = torch.randn(4, requires_grad=True)
    y = w
    for _ in range(5000):
        y = y + 1
    lives = _Twice.apply(torch.ones(4), y)
    with pytest.raises(RuntimeError, match="same leaves"):
        captured(lambda: _Twice.apply(torch.ones(4), w), w)
    assert lives is not None


def test_an_operators_own_attributes_are_no_leaves(captured):
    class Named(torch.autograd.Function):
        @staticmethod
        def forward(ctx, w):
            ctx.variable = "mine"
            return w * 2

        @staticmethod
        def backward(ctx, dy):
            return dy * 2
    w = torch.randn(4, requires_grad=True)
    lives = _Twice.apply(torch.ones(4), Named.apply(w))
    with pytest.raises(RuntimeError, match="same leaves"):
        captured(lambda: _Twice.apply(torch.ones(4), w), w)
    assert lives is not None
