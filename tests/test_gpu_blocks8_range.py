"""8-bit blocks at the top of the fp32 and bf16 range on the GPU: what is finite stays finite wherever the blocks are read."""
import pytest
import torch

import self_forcing_amd as sfa
from gpu_util import randn
from oracle import blocks8 as o

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
blk, l8 = sfa.block_ops, sfa.linear8
TOP = 248 * 2.0 ** 120                                # from here on e4m3 would round up to 2^128


def _rows(dtype):
    """A row per value around the top, alone in its block, among smaller ones, beside one that is not finite."""
    top = torch.finfo(dtype).max
    vals = [top, -top, TOP, -TOP, TOP * (1 - torch.finfo(dtype).eps), 3.0e38, 240 * 2.0 ** 120, 2.0 ** 127]
    x = 0.1 * randn((len(vals), 384), 1) * 2.0 ** 119
    for i, v in enumerate(vals):
        x[i, 0], x[i, 130], x[i, 300:] = v, -v, v
    x[3, 131], x[4, 132] = float("inf"), float("nan")
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values(dtype):
    x = _rows(dtype)
    ref = o.values(x)
    assert ref.nan_to_num(0).abs().max() == 240 * 2.0 ** 120
    for out in (torch.float32, torch.bfloat16):
        v = l8.quantize(x[None].to(DEV)).dequantize(out)[0].double().cpu()
        assert torch.equal(torch.isnan(v), torch.isnan(ref)) and torch.equal(v.nan_to_num(0), ref.nan_to_num(0))
    p = l8.pack(x.to(DEV))
    w = o.values(x, True)
    for v in (p.dequantize(torch.float32), l8.Weight8(p.data_t, p.scale_t, None, None, p.shape[::-1], dtype).dequantize(torch.float32).t()):
        v = v.double().cpu()
        assert torch.equal(torch.isnan(v), torch.isnan(w)) and torch.equal(v.nan_to_num(0), w.nan_to_num(0))


@pytest.mark.parametrize("M", [4, 40])
def test_products_and_gradients(M):
    """Rows of one value, quantised inside the product's kernel (4) and before it (40): a weight of 2^-126 brings them back."""
    dtype = torch.bfloat16
    top = torch.finfo(dtype).max
    x = torch.zeros((1, M, 128), dtype=dtype)
    x[0, 1, 5], x[0, 3, 6] = top, -top
    w = torch.full((64, 128), 2.0 ** -126, dtype=dtype)
    got = l8.linear8(x.to(DEV), w.to(DEV))[0].double().cpu()
    ref = (o.values(x[0]) @ o.values(w, True).t())
    assert torch.equal(got, ref) and got[1, 0] == 240 * 2.0 ** -6
    dy = torch.zeros((1, M, 64), dtype=dtype)
    dy[0, 1], dy[0, 3] = 2.0 ** -126, 2.0 ** -125
    dw, _ = l8.weight_grad(dy.to(DEV), l8.quantize(x.to(DEV)))
    assert torch.equal(dw.double().cpu(), dy[0].double().t() @ o.values(x[0]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gelu(dtype):
    x = torch.full((1, 3, 128), torch.finfo(dtype).max, dtype=dtype)
    x[0, 1] *= -1
    leaf = x.to(DEV).requires_grad_()
    y = blk.gelu_tanh(leaf, checkpoint8=True)
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(leaf))
    assert torch.equal(y[0, 0].cpu(), x[0, 0]) and not y[0, 1].any()
    assert torch.equal(dx.cpu(), (x > 0).to(dtype))


def test_a_weights_values_at_every_scale():
    """The values of a packed weight are the blocks' own, bit for bit, for every exponent a block can have."""
    e = torch.arange(-126, 120)
    w = torch.zeros((128 * len(e), 130))
    w[::128, 0] = torch.pow(2.0, e.double() + 8).float()                # 256 * 2^s: more than 448 * 2^(s - 1)
    w[1::128] = w[::128, :1] * torch.rand((1, 130), generator=torch.Generator().manual_seed(5))
    p = l8.pack(w.to(DEV))
    assert p.scale[:, 0].tolist() == (e + 127).tolist()
    ref = o.values(w, True)
    assert torch.equal(p.dequantize(torch.float32).double().cpu(), ref.float().double())
    assert torch.equal(p.dequantize(torch.bfloat16).double().cpu(), ref.to(torch.bfloat16).double())
