"""What saved-tensor hooks do to the training operators of the block's rows, without a GPU: the hooks give a tensor's values back in
memory and a layout of their own, and the backward's call has to describe those."""
import contextlib

import pytest
import torch
from torch.multiprocessing.reductions import StorageWeakRef

import self_forcing_amd as sfa

blk, l8 = sfa.block_ops, sfa.linear8


class _Library:
    """Takes every call and remembers the backwards' arguments."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    for m in (blk, l8):
        monkeypatch.setattr(m._l, "load", lambda: lib)
        monkeypatch.setattr(m, "_raw_stream", lambda index: 0)
        monkeypatch.setattr(m, "_stream", lambda t: None)
        monkeypatch.setattr(m, "_on_device", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(m, "_rows", lambda t: (t.shape[0] * t.shape[1], t.shape[2], blk._row_stride(t)))
    monkeypatch.setattr(blk, "_ln_bwd_bytes", lambda *a: 0)
    monkeypatch.setattr(l8, "_bytes", lambda *a: 256)
    return lib


class _Hooks(torch.autograd.graph.saved_tensors_hooks):
    """Gives back copies with contiguous values (as save_on_cpu does), or with transposed ones; remembers them."""

    def __init__(self, transposed=False):
        self.given = []
        given = self.given

        def unpack(t):
            t = t.clone(memory_format=torch.contiguous_format)
            if transposed and t.dim() > 1:
                t = t.transpose(-1, -2).contiguous().transpose(-1, -2)
            given.append(t)
            return t
        super().__init__(lambda t: t, unpack)

    def __enter__(self):
        super().__enter__()
        return self


@pytest.mark.parametrize("transposed", [False, True])
def test_layer_norm_takes_the_strides_of_what_it_gets(library, transposed):
    B, F, per, C = 2, 3, 4, 64
    x = torch.randn(B, F * per, 256)[..., 64:128].requires_grad_()
    scale, shift = torch.randn(B, F, 6, C).requires_grad_().chunk(6, dim=2)[1:3]
    dy = torch.ones(B, F * per, C)
    for hooked in (False, True):
        with _Hooks(transposed) if hooked else contextlib.nullcontext():
            y = blk.ln_modulate(x, scale, shift)
        torch.autograd.grad(y, x, dy)
        args = library.calls["sfm_ln_bwd"]
        assert args[5] == (C if hooked else 256)                 # x_stride
        assert args[13] == (C if hooked else 6 * C)              # mod_stride
    w = torch.randn(C).requires_grad_()
    with _Hooks(transposed):
        y = blk.ln_affine(x, w, w)
    torch.autograd.grad(y, x, dy)
    assert library.calls["sfm_ln_bwd"][5] == C


@pytest.mark.parametrize("op", ["ln", "linear8"])
def test_blocks_come_as_rows_whatever_the_hooks_give(library, monkeypatch, op):
    C, N = 256, 64
    x = torch.randn(1, 40, C).bfloat16().requires_grad_()
    with _Hooks(transposed=True) as hooks:
        if op == "ln":
            w = torch.ones(C).bfloat16()
            y = blk.ln_affine(x, w, w, checkpoint8=True)
            name, at = "sfm_ln_bwd", 6
        else:
            blocks = lambda n, k: (torch.zeros(n, k, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.uint8))
            monkeypatch.setattr(l8, "pack", lambda w, transposed: l8.Weight8(*blocks(N, C), *blocks(C, 128), (N, C), w.dtype))
            w = torch.randn(N, C).bfloat16().requires_grad_()
            y = l8._Linear8Fn.apply(x, w, None, None, None)
            name, at = "sfm_linear8_bwd", 8
    torch.autograd.grad(y, x, torch.ones_like(y))
    given = [t for t in hooks.given if t.dtype == torch.uint8 and t.dim() == 2 and not t.is_contiguous()]
    assert given and library.calls[name][at] not in [t.data_ptr() for t in given]


@pytest.mark.parametrize("keep8", [False, True])
def test_gelu_holds_what_the_hooks_give_until_its_call(library, monkeypatch, keep8):
    """Nobody else holds a tensor that a hook has made: freed before the call, its memory would be the gradient's."""
    x = torch.randn(1, 40, 256).bfloat16().requires_grad_()
    given = []

    def unpack(t):
        t = t.clone()
        given.append((t.data_ptr(), StorageWeakRef(t.untyped_storage())))
        return t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = blk.gelu_tanh(x, checkpoint8=keep8)

    def call(*args):
        library.calls["sfm_gelu_bwd"] = args, [ref.expired() for _, ref in given]
        return 0
    monkeypatch.setattr(library, "sfm_gelu_bwd", call, raising=False)
    torch.autograd.grad(y, x, torch.ones_like(y))
    args, gone = library.calls["sfm_gelu_bwd"]
    assert gone == [False] * (2 if keep8 else 1)
    assert [at for at, _ in given] == list(args[5:7] if keep8 else args[3:4])


def test_gelu_takes_rows_whatever_the_hooks_give(library):
    x = torch.randn(1, 40, 256).bfloat16().requires_grad_()
    with _Hooks(transposed=True):
        y = blk.gelu_tanh(x)
    torch.autograd.grad(y, x, torch.ones_like(y))
    assert library.calls["sfm_gelu_bwd"][4] == 256


WRONG = {"type": lambda t: t.double(), "size": lambda t: t[..., :-1], "device": lambda t: t.to("meta"), "none": lambda t: t}


@pytest.mark.parametrize("how", WRONG)
@pytest.mark.parametrize("op", ["ln", "ln8", "gelu", "gelu8", "linear8"])
def test_what_is_not_the_saved_tensor_is_refused(library, monkeypatch, how, op):
    """Before its address reaches a kernel."""
    x, w = torch.randn(1, 40, 256).bfloat16().requires_grad_(), torch.randn(256).bfloat16().requires_grad_()
    blocks = lambda n, k: (torch.zeros(n, k, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.uint8))
    monkeypatch.setattr(l8, "pack", lambda w, transposed: l8.Weight8(*blocks(64, 256), *blocks(256, 128), (64, 256), w.dtype))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, WRONG[how]):
        y = {"ln": lambda: blk.ln_affine(x, w, w), "ln8": lambda: blk.ln_affine(x, w, w, checkpoint8=True), "gelu": lambda: blk.gelu_tanh(x),
             "gelu8": lambda: blk.gelu_tanh(x, checkpoint8=True),
             "linear8": lambda: l8._Linear8Fn.apply(x, torch.randn(64, 256).bfloat16().requires_grad_(), None, None, None)}[op]()
    library.calls.clear()
    if how == "none":
        torch.autograd.grad(y, x, torch.ones_like(y))
        assert library.calls
    else:
        with pytest.raises(RuntimeError, match="saved-tensor hooks gave back"):
            torch.autograd.grad(y, x, torch.ones_like(y))
        assert not library.calls
