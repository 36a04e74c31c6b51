"""Layouts that say nothing: strides of dimensions of one, in weights and rows of linear8."""
import pytest
import torch

import self_forcing_amd as sfa
from gpu_util import randn
from oracle import blocks8 as o

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
l8 = sfa.linear8


@pytest.mark.parametrize("n,k,view", [(1, 300, lambda t: t.t()), (1, 300, lambda t: t[:, 0].expand(1, 300)), (300, 1, lambda t: t),
                                      (300, 1, lambda t: t.t().contiguous().t()), (1, 1, lambda t: t[:1].as_strided((1, 1), (0, 0)))])
def test_weights_with_a_dimension_of_one(n, k, view):
    w = view(randn((300, 1), 1, torch.bfloat16).to(DEV))
    assert w.shape == (n, k)
    p = l8.pack(w)
    ref = o.values(w.cpu(), True)
    assert torch.equal(p.dequantize(torch.float32).double().cpu(), ref)
    x = torch.zeros((1, 3, k), dtype=torch.bfloat16, device=DEV)
    x[0, 1, 0] = 2.0
    y = l8.linear8(x, w)[0].double().cpu()
    assert torch.equal(y[1], 2 * ref[:, 0]) and not y[0].any() and not y[2].any()
