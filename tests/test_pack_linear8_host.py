"""When a packed model refuses to run on its 8-bit blocks, without a GPU: the blocks' layout is replaced by a record of the call."""
import copy

import numpy as np
import pytest
import torch

import self_forcing_amd as sfa

cm = sfa.causal_model
TINY = dict(dim=64, ffn_dim=128, num_heads=2, num_layers=2, text_dim=32, text_len=8, frame_hw=(2, 3), total_seq_len=6 * 6)


@pytest.fixture
def model(monkeypatch):
    m = cm.CausalWanModel(ops=cm.HipAttentionOps(), **TINY).to(torch.bfloat16)
    m.init_weights(zero_head=False)
    m.packed = []

    def pack(weight, transposed=True):
        m.packed.append(weight.detach().clone())
        return weight.detach().clone()
    monkeypatch.setattr(cm._l8, "pack", pack)
    monkeypatch.setattr(cm._l8, "linear8", lambda x, w, bias=None, **kw: torch.nn.functional.linear(x, w, bias))
    return m.pack_linear8()


def _runs(block, what):
    with torch.no_grad():
        if what == "qkv":
            return block.self_attn._project_qkv(torch.zeros(1, 2, 64, dtype=torch.bfloat16))
        return cm._packed8(block.ffn[0])


def _param(block, what):
    return block.self_attn.k.bias if what == "qkv" else block.ffn[0].weight


@pytest.mark.parametrize("what", ["qkv", "ffn"])
def test_other_memory_at_the_same_address_is_refused(model, what):
    """p.data replaced twice, the second tensor where the packed one lay."""
    block = model.blocks[0]
    p = _param(block, what)
    memory = np.zeros(p.numel(), dtype=np.int16)
    first = torch.from_numpy(memory).view(torch.bfloat16).view(p.shape)
    p.data = first
    model.pack_linear8()
    assert _runs(block, what) is not None
    p.data = torch.ones_like(first)
    with pytest.raises(RuntimeError, match="pack_linear8"):
        _runs(block, what)
    memory[:] = 17
    p.data = torch.from_numpy(memory).view(torch.bfloat16).view(p.shape)
    assert p.data_ptr() == first.data_ptr()
    with pytest.raises(RuntimeError, match="pack_linear8"):
        _runs(block, what)
    model.pack_linear8()
    assert _runs(block, what) is not None


@pytest.mark.parametrize("what", ["qkv", "ffn"])
@pytest.mark.parametrize("change", ["write", "load", "same memory in another layout", "copy"])
def test_changes_that_are_refused(model, what, change):
    block = model.blocks[1]
    p = _param(block, what)
    assert _runs(block, what) is not None
    if change == "write":
        with torch.no_grad():
            p.add_(1)
    elif change == "load":
        model.load_state_dict(copy.deepcopy(model.state_dict()))
    elif change == "copy":
        block = copy.deepcopy(model).blocks[1]
        assert not block.ffn[0].weight8_of.of                     # and does not keep parameters of the first alive
    else:
        p.data = p.data.flip(0) if p.dim() == 1 else p.data.view(64, 128).t()
    with pytest.raises(RuntimeError, match="pack_linear8"):
        _runs(block, what)


def test_a_write_through_data_is_taken_up_by_the_next_pack(model):
    """It cannot be seen: the blocks are a snapshot until pack_linear8 is called again."""
    w = model.blocks[0].ffn[0].weight
    was = w.detach().clone()
    w.data.mul_(2)
    assert torch.equal(_runs(model.blocks[0], "ffn"), was)
    model.packed.clear()
    model.pack_linear8()
    assert torch.equal(_runs(model.blocks[0], "ffn"), 2 * was)


def test_unpacked_layers_hold_nothing(model):
    model.pack_linear8(False)
    for b in model.blocks:
        assert b.self_attn.qkv8 is None and b.self_attn.qkv8_of is None and b.ffn[0].weight8 is None and b.ffn[0].weight8_of is None


def test_with_gradients_enabled_every_layer_is_the_16_bit_one(model, monkeypatch):
    def reached(*args, **kw):
        raise AssertionError("the 8-bit layer")
    monkeypatch.setattr(cm._l8, "linear8", reached)
    sa, ops = model.blocks[0].self_attn, model.blocks[0].ops
    x = torch.randn(1, 2, 64).to(torch.bfloat16)
    qkv = [sa.q, sa.k, sa.v]
    ref = torch.nn.functional.linear(x, torch.cat([m.weight for m in qkv]), torch.cat([m.bias for m in qkv]))
    assert torch.equal(torch.cat(sa._project_qkv(x), -1), ref)
    assert torch.equal(ops.linear(x, sa.o), sa.o(x))
    for call in (lambda: sa._project_qkv(x), lambda: ops.linear(x, sa.o)):
        with torch.no_grad(), pytest.raises(AssertionError, match="the 8-bit layer"):
            call()


@pytest.mark.parametrize("packed", [False, True])
def test_the_feed_forwards_second_layer_is_the_librarys_unless_packed(monkeypatch, packed):
    """own_gemm="auto" is for the block's square projections, however small the feed-forward is."""
    class Ops(cm.HipAttentionOps):
        def __init__(self):
            super().__init__("auto")
            self.through = []

        def linear(self, x, linear):
            self.through.append(linear)
            return linear(x)

        def linear_gelu(self, x, linear):
            return linear(x)

        def ln_modulate(self, x, scale, shift, eps):
            return x

        def gate_residual_ln(self, x, y, gate, eps, **kw):
            return x + y, x + y
    ops = Ops()
    block = cm.CausalWanAttentionBlock(64, 128, 2, frame_hw=(2, 3), total_seq_len=36, ops=ops)
    monkeypatch.setattr(block.self_attn, "forward", lambda x, *a: x)
    monkeypatch.setattr(block.cross_attn, "forward", lambda x, *a: x)
    if packed:
        block.ffn[2].weight8, block.ffn[2].weight8_of = object(), cm._Snapshot(block.ffn[2].weight)
    x, e = torch.randn(1, 6, 64), torch.randn(1, 1, 6, 64)
    with torch.no_grad():
        block(x, e, None, None, None, None, 0, next_mod=(e[:, :, 0], e[:, :, 1]))
    assert (block.ffn[2] in ops.through) == packed


def test_layers_of_32_bits_are_refused_before_any_is_packed(model):
    was = [b.self_attn.qkv8_of for b in model.blocks]
    model.packed.clear()
    model.blocks[1].ffn[2].float()
    with pytest.raises(ValueError, match="float16 / bfloat16 layers"):
        model.pack_linear8()
    assert not model.packed and was == [b.self_attn.qkv8_of for b in model.blocks]
    model.pack_linear8(False)
    model.half().pack_linear8()
