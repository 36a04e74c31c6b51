"""The tile kernels of linear8 and of its weight's gradient on the GPU, against float64: every size asserts that it takes the kernel it
is here for.  The oracle's blocks come from the CPU (torch's powers of two on the GPU are off by a unit of float64, enough to turn a
tie); their float64 products are formed on the GPU.

Tolerances as in test_gpu_linear8.py; the gated residual besides rounds its product and its sum once each in fp32: 2^-23 of both."""
import ctypes as C
import math

import pytest
import torch

import self_forcing_amd as sfa
from gpu_util import randn
from linear8_sizes import NO_TILE, TILE_128, TILE_256, WGRAD_256, product_plan, wgrad_plan
from oracle import blocks8 as o
from test_gpu_linear8 import near, rows, sum8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
l8 = sfa.linear8


def _values(t, square=False):
    return o.values(t.cpu().view(-1, t.shape[-1]), square).to(DEV)


def _layer(M, K, N, dtype, seed):
    x, w, b = rows((2, M // 2, K), seed, dtype), (randn((N, K), seed + 1) / math.sqrt(K)).to(dtype), randn((N,), seed + 2, dtype)
    return x.to(DEV), w.to(DEV), b.to(DEV)


def _product(x, w, b):
    y, slack = sum8(_values(x), _values(w, True))
    y = y + b.double()
    return y.view(*x.shape[:2], -1), (slack + 2.0 ** -23 * (y.abs() + b.double().abs())).view(*x.shape[:2], -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,plan", [(s, (256, h)) for s, h in TILE_256.items()] + [(s, (128, 0)) for s in TILE_128])
def test_product(dtype, size, plan):
    assert product_plan(*size) == plan
    x, w, b = _layer(*size, dtype, 1)
    y, slack = _product(x, w, b)
    p = l8.pack(w, transposed=False)
    got = l8.linear8(x, p, b)
    near(got, y, dtype, slack)
    assert torch.equal(l8.linear8(l8.quantize(x), p, b), got)
    near(l8.linear8(x, p, b, epilogue="gelu_tanh"), o.gelu(y), dtype, 1.13 * slack + 2.0 ** -16 * o.gelu(y).abs())
    N = size[2]
    for off, width in ((0, N + 3), (5, N + 8), (8, -(-N // 8) * 8 + 24)):       # rows of a wider buffer, at any offset
        buf = torch.full((2, size[0] // 2, width), 7.0, dtype=dtype, device=DEV)
        l8.linear8(x, p, b, out=buf[..., off:off + N])
        assert torch.equal(buf[..., off:off + N], got)
        assert bool((buf[..., :off] == 7).all()) and bool((buf[..., off + N:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,plan", [(s, (256, h)) for s, h in TILE_256.items()] + [(s, (128, 0)) for s in TILE_128] + [(s, (0, 0)) for s in NO_TILE])
def test_gated_residual(dtype, size, plan):
    assert product_plan(*size) == plan
    M, K, N = size
    B, L = 2, M // 2
    F = next(f for f in (3, 4, 5, 2, 1) if L % f == 0)
    x, w, b = _layer(*size, dtype, 11)
    y, slack = _product(x, w, b)
    res, gate = randn((B, L, N), 14, dtype).to(DEV), randn((B, F, 1, N), 15, dtype).to(DEV)
    g = gate.double().expand(B, F, L // F, N).reshape(B, L, N)
    args = (x, l8.pack(w, transposed=False), b, "gate_residual")
    was, out = res.clone(), torch.empty_like(res)
    l8.linear8(*args, res=res, gate=gate, out=out)
    want = res.double() + y * g
    near(out, want, dtype, slack * g.abs() + 2.0 ** -23 * ((y * g).abs() + want.abs()))
    assert torch.equal(res, was)
    inplace = res.clone()
    assert l8.linear8(*args, res=inplace, gate=gate) is inplace and torch.equal(inplace, out)
    ungated = l8.linear8(*args, res=res.clone())
    want = res.double() + y
    near(ungated, want, dtype, slack + 2.0 ** -23 * want.abs())
    # res and out as columns of one buffer, off the 16-byte grid, and in place there
    buf = torch.full((B, L, 2 * N + 7), 7.0, dtype=dtype, device=DEV)
    buf[..., 1:1 + N] = res
    l8.linear8(*args, res=buf[..., 1:1 + N], gate=gate, out=buf[..., N + 4:2 * N + 4])
    assert torch.equal(buf[..., N + 4:2 * N + 4], out) and torch.equal(buf[..., 1:1 + N], res)
    l8.linear8(*args, res=buf[..., 1:1 + N], gate=gate)
    assert torch.equal(buf[..., 1:1 + N], out)
    assert all(bool((buf[..., a:z] == 7).all()) for a, z in ((0, 1), (N + 1, N + 4), (2 * N + 4, 2 * N + 7)))


@pytest.mark.parametrize("size", [(4, 256, 64), (528, 512, 256), TILE_128[1], next(iter(TILE_256))])
@pytest.mark.parametrize("apart", [1, 8])
def test_what_the_sums_of_eight_drop(size, apart):
    """Two products of 2^16 that cancel, and one of 2^(16 - j), among the same 8 neighbouring channels or in the next 8: exact up to j = 13,
    and off by less than 2^-13 of the largest beyond; in another 8 exact."""
    M, K, N = size
    x, w = torch.zeros((1, M, K), dtype=torch.bfloat16), torch.zeros((N, K), dtype=torch.bfloat16)
    j = torch.arange(N) % 18                                          # 2^(8 - j) down to e4m3's least, 2^-9
    x[..., 0] = x[..., 2] = 256
    w[:, 0], w[:, 2] = 256, -256
    k = 1 if apart == 1 else 9
    x[..., k], w[:, k] = 256, torch.pow(2.0, 8.0 - j)
    y, small = l8.linear8(x.to(DEV), w.to(DEV))[0].double().cpu(), torch.pow(2.0, 16.0 - j.double())
    exact = (j <= 13) | (apart == 8)
    assert torch.equal(y[:, exact], small[exact].expand(M, -1))
    assert ((y - small).abs() < 2 * 2.0 ** 16 * 2.0 ** -13).all()


def _wgrad(dy, x):
    d, v = dy.view(-1, dy.shape[-1]).double(), _values(x)
    if dy.dtype == torch.float16:
        v = v.clamp(-65504, 65504)
    M = d.shape[0]
    return (d.t() @ v, M * 2.0 ** -23 * (d.abs().t() @ v.abs())), (d.sum(0), M * 2.0 ** -23 * d.abs().sum(0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,parts", WGRAD_256.items())
def test_weight_gradient(dtype, size, parts):
    assert wgrad_plan(*size) == (256, parts)
    M, K, N = size
    x, dy = rows((1, M, K), 21, dtype).to(DEV), rows((1, M, N), 22, dtype).to(DEV)
    x8 = l8.quantize(x)
    dw, db = l8.weight_grad(dy, x8)
    (rw, sw), (rb, sb) = _wgrad(dy, x)
    near(dw, rw, dtype, sw)
    near(db, rb, dtype, sb)
    wide = torch.full((1, M, N + 5), float("nan"), dtype=dtype, device=DEV)      # rows inside others, off the 16-byte grid
    wide[..., 3:3 + N] = dy
    for d in (dy, wide[..., 3:3 + N]):
        again = l8.weight_grad(d, x8)
        assert torch.equal(again[0], dw) and torch.equal(again[1], db)


@pytest.mark.parametrize("size", [(161, 3900, 4001), (4680, 1500, 1501)])
def test_weight_gradient_writes_its_channels_only(size):
    """Non-finite values reach their channel only, and nothing behind dw and dbias is written."""
    M, K, N = size
    assert wgrad_plan(*size)[0] == 256
    dtype, lib = torch.bfloat16, sfa.lib.load()
    x, dy = rows((1, M, K), 31, dtype).to(DEV), rows((1, M, N), 32, dtype).to(DEV)
    x[0, M // 2, K - 1], x[0, M - 1, 5] = float("nan"), float("inf")
    dy[0, 0, N - 1], dy[0, M - 1, 7] = float("nan"), float("-inf")
    x8 = l8.quantize(x)
    n = C.c_size_t(0)
    sfa.lib.check(lib.sfm_linear8_wgrad_workspace_bytes(M, N, K, C.byref(n)))
    dw, db = (torch.full((k + 4096,), 7.0, dtype=dtype, device=DEV) for k in (N * K, N))
    ws = torch.full((n.value + 65536,), 0xA5, dtype=torch.uint8, device=DEV)
    sfa.lib.check(lib.sfm_linear8_wgrad(0, M, N, K, dy.data_ptr(), N, x8.data.data_ptr(), x8.scale.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                        None, ws.data_ptr(), n.value, None))
    torch.cuda.synchronize()
    assert bool((dw[N * K:] == 7).all()) and bool((db[N:] == 7).all()) and bool((ws[n.value:] == 0xA5).all())
    bad = ~torch.isfinite(dw[:N * K].view(N, K))
    want = torch.zeros_like(bad)
    want[7], want[N - 1], want[:, 5], want[:, K - 1] = True, True, True, True
    assert torch.equal(bad, want)
    assert (~torch.isfinite(db[:N])).nonzero().flatten().tolist() == [7, N - 1]


def test_weight_gradient_in_parts_of_more_than_two_grids_worth():
    """More sums of parts than one grid dimension's 2^21 workgroups take: 600 rows of -1, 0 and 1 over and over, so that every sum is exact
    in any order."""
    n, times, C = 600, 100, 8200
    assert wgrad_plan(n * times, C, C) == (256, 2) and C * C > 32 << 21
    g = torch.Generator().manual_seed(41)
    x, dy = (torch.randint(-1, 2, (1, n, C), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    dw, db = l8.weight_grad(dy.repeat(1, times, 1), l8.quantize(x.repeat(1, times, 1)))
    assert torch.equal(dw, (times * (dy[0].double().t() @ x[0].double())).to(torch.bfloat16))
    assert torch.equal(db, (times * dy[0].double().sum(0)).to(torch.bfloat16))
