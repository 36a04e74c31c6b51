"""The training operators of the block's rows under saved-tensor hooks on the GPU: gradients are the same bits with the saved tensors
kept on the host and brought back, or given back in another layout."""
import pytest
import torch

import self_forcing_amd as sfa
from gpu_util import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
blk, l8 = sfa.block_ops, sfa.linear8


def _transposed(t):
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t.clone()


HOOKS = [lambda: torch.autograd.graph.save_on_cpu(), lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, _transposed)]


def _same(step, leaves, dy):
    y = step()
    ref = torch.autograd.grad(y, leaves, dy)
    for hooks in HOOKS:
        with hooks():
            y = step()
        got = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("keep8", [False, True])
def test_layer_norms(keep8):
    B, F, per, C = 2, 3, 10, 256
    x = randn((B, F * per, 768), 1, torch.bfloat16).to(DEV)[..., 256:512].requires_grad_()
    e = randn((B, F, 6, C), 2, torch.bfloat16).to(DEV).requires_grad_()
    dy = randn((B, F * per, C), 3, torch.bfloat16).to(DEV)
    w, b = (randn((C,), 4 + i, torch.bfloat16).to(DEV).requires_grad_() for i in range(2))

    def modulated():
        m = e.chunk(6, dim=2)
        return blk.ln_modulate(x, m[1], m[2], checkpoint8=keep8)
    _same(modulated, (x, e), dy)
    _same(lambda: blk.ln_affine(x, w, b, checkpoint8=keep8), (x, w, b), dy)


def test_linear():
    x, w = (randn(s, 6 + i, torch.bfloat16).to(DEV).requires_grad_() for i, s in enumerate(((1, 70, 200), (130, 200))))
    _same(lambda: l8.linear8(x, w), (x, w), randn((1, 70, 130), 8, torch.bfloat16).to(DEV))


@pytest.mark.parametrize("keep8", [False, True])
def test_gelu(keep8):
    x = randn((1, 300, 1000), 9, torch.bfloat16).to(DEV).requires_grad_()
    _same(lambda: blk.gelu_tanh(x, checkpoint8=keep8), x, randn((1, 300, 1000), 10, torch.bfloat16).to(DEV))
