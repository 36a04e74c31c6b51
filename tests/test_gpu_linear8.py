"""Linear layers on 8-bit blocks, their gradients and the 8-bit checkpoints on the GPU, against the float64 oracle.

Tolerances.  The blocks are exact.  A product: half a step of the output's type on the value, and for the fp32 sum of K products
K 2^-23 sum |x||w| (every addition off by at most a unit of 2^-23 of the magnitudes summed, whatever the order and
whether the matrix unit rounds or truncates).

The e4m3 matrix instructions align the products of 8 neighbouring k to the largest of the 8 before they add them and drop what
lies below 2^-13 of it.  That is seen directly: with products 2^16 and 2^(16 - j) in one such 8, the sum is exact up to
j = 13 and 2^16 from j = 14 on, for every place of the two; in different 8s it is exact to fp32.  Each of the 7 other products
of an 8 so loses less than 2^-13 of the largest, which is at most max |x| max |w| over the 8: 7 2^-13 sum over the 8s of max |x| max |w|."""
import math

import pytest
import torch

import self_forcing_amd as sfa
from gpu_util import randn
from oracle import blocks8 as o

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
l8 = sfa.linear8
blk = sfa.block_ops
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}      # values below may be anything smaller


def near(got, ref, dtype, slack):
    """|got - ref| within half a step of `dtype` plus `slack` (what happened before the rounding)."""
    got, ref = got.double().cpu(), ref.double().cpu()
    slack = slack.double().cpu() if isinstance(slack, torch.Tensor) else slack
    assert got.dtype == ref.dtype and got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    tol = HALF[dtype] * (ref.abs() + slack) + slack + TINY[dtype]
    top = torch.finfo(dtype).max                             # what rounds past the type's range is infinite in it
    out = (ref.abs() - tol > top) | ((ref.abs() + tol > top) & torch.isinf(got))
    assert torch.equal(torch.isinf(got[out]) & (got[out].sign() == ref[out].sign()), torch.ones_like(got[out], dtype=torch.bool))
    got = torch.where(out, ref, got)
    bad = (got - ref).abs() > tol
    bad &= ~torch.isnan(ref)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off; worst {((got - ref).abs() / tol).nan_to_num().max().item():.2f} tolerances"


def rows(shape, seed, dtype):
    """Channels of different strength, and an outlier in some blocks."""
    x = randn(shape, seed, torch.float32) * torch.exp(0.7 * randn(shape[-1:], seed + 50, torch.float32)) + 0.1
    x[..., ::97] *= 20
    return x.to(dtype)


def sum8(x, w):
    """(x w^T, its slack) of values in 8-bit blocks."""
    top = lambda t: torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8)).view(t.shape[0], -1, 8).amax(2)
    return x @ w.t(), x.shape[1] * 2.0 ** -23 * (x.abs() @ w.abs().t()) + 7 * 2.0 ** -13 * (top(x) @ top(w).t())


def product(x, w, b=None):
    """(float64 product of the blocks, its slack)."""
    y, slack = sum8(o.values(x), o.values(w, True))
    return (y, slack) if b is None else (y + b.double(), slack + 2.0 ** -23 * (y.abs() + b.double().abs()))


# ------------------------------------------------------------------------------------------------ blocks
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,K", [(1, 1, 1), (1, 3, 128), (2, 65, 129), (1, 129, 777), (1, 300, 1536), (3, 128, 256)])
def test_blocks_hold_what_the_definition_says(dtype, B, L, K):
    x = rows((B, L, K), 1, dtype)
    x[0, 0] = 0
    r = l8.quantize(x.to(DEV))
    assert r.shape == x.shape and r.dtype == dtype
    assert torch.equal(r.dequantize(torch.float32).double().cpu().view(-1, K), o.values(x.view(-1, K)))
    assert torch.equal(r.dequantize(torch.bfloat16).double().cpu().view(-1, K), o.values(x.view(-1, K)))
    w = x.view(-1, K)
    p = l8.pack(w.to(DEV))
    assert torch.equal(p.dequantize(torch.float32).double().cpu(), o.values(w, True))
    t = l8.Weight8(p.data_t, p.scale_t, None, None, (K, B * L), dtype)
    assert torch.equal(t.dequantize(torch.float32).double().cpu(), o.values(w, True).t())
    assert l8.pack(w.to(DEV), transposed=False).data_t is None


def test_blocks_of_strided_and_unaligned_rows():
    base = rows((1, 40, 600), 2, torch.bfloat16)
    for a, b in ((0, 520), (1, 300), (3, 131), (8, 264)):
        x = base[..., a:b]
        r = l8.quantize(base.to(DEV)[..., a:b])
        assert torch.equal(r.dequantize(torch.float32)[0].double().cpu(), o.values(x[0]))
        p = l8.pack(base.to(DEV)[0, :, a:b])
        assert torch.equal(p.dequantize(torch.float32).double().cpu(), o.values(x[0], True))


def test_blocks_of_extreme_and_non_finite_values():
    x = torch.zeros((1, 8, 256))
    x[0, 0, :128], x[0, 1, 0], x[0, 2, 3], x[0, 3, 7] = 3.0e38, 1e-42, float("inf"), float("nan")
    x[0, 4, 200], x[0, 5, 128:] = float("-inf"), torch.linspace(-448, 448, 128)
    x[0, 6, :128] = 448.0 * 2 ** 5
    x[0, 7] = 65504
    v = l8.quantize(x.to(DEV)).dequantize(torch.float32).double().cpu()
    ref = o.values(x[0])
    assert torch.equal(torch.isnan(v[0]), torch.isnan(ref))
    assert torch.equal(v[0].nan_to_num(0), ref.nan_to_num(0))
    h = l8.quantize(x[:, 7:].half().to(DEV))            # 65504 rounds up past fp16: its largest value comes back
    assert torch.equal(h.dequantize().cpu(), x[:, 7:].half())
    assert h.dequantize(torch.float32).max().item() == 65536


# ------------------------------------------------------------------------------------------------ product
SIZES = [(1, 1, 1), (1, 128, 16), (3, 1536, 100), (16, 100, 8), (5, 2500, 70), (1, 8960, 33), (16, 2176, 130), (17, 300, 40), (64, 128, 129), (65, 1000, 77), (128, 256, 256), (129, 513, 300),
         (200, 2100, 130), (257, 640, 260), (700, 384, 520),
         (300, 100, 300), (300, 200, 260), (300, 390, 256), (300, 512, 264), (1100, 100, 260), (1100, 200, 300), (1100, 384, 256),
         (1030, 520, 257), (1281, 1300, 300), (1420, 513, 264), (2304, 640, 2100), (4300, 520, 5000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(dtype, M, K, N):
    x, w, b = rows((1, M, K), 3, dtype), (randn((N, K), 4) / math.sqrt(K)).to(dtype), randn((N,), 5, dtype)
    y, slack = product(x[0], w, b)
    xd, wd, bd = x.to(DEV), w.to(DEV), b.to(DEV)
    p = l8.pack(wd)
    got = l8.linear8(xd, p, bd)
    near(got[0], y, dtype, slack)
    assert torch.equal(l8.linear8(xd, wd, bd), got) and torch.equal(l8.linear8(l8.quantize(xd), p, bd), got)
    near(l8.linear8(xd, p)[0], *(lambda t: (t[0], dtype, t[1]))(product(x[0], w)))
    # a GELU moves by at most 1.13 of what its argument does, and is 2^-16 of itself off at most in fp32
    near(l8.linear8(xd, p, bd, epilogue="gelu_tanh")[0], o.gelu(y), dtype, 1.13 * slack + 2.0 ** -16 * o.gelu(y).abs())


@pytest.mark.parametrize("M,K,N", [(6, 256, 64), (8, 130, 33), (264, 512, 256), (300, 200, 130)])
def test_gated_residual(M, K, N):
    dtype, B, F = torch.bfloat16, 2, 2
    x, w, b = rows((B, M, K), 6, dtype), (randn((N, K), 7) / math.sqrt(K)).to(dtype), randn((N,), 8, dtype)
    res, gate = randn((B, M, N), 9, dtype), randn((B, F, 1, N), 10, dtype)
    y, slack = product(x.view(-1, K), w, b)
    y, slack = y.view(B, M, N), slack.view(B, M, N)
    g = gate.double().expand(B, F, M // F, N).reshape(B, M, N)
    args = (x.to(DEV), l8.pack(w.to(DEV)), b.to(DEV), "gate_residual")
    rd, gd = res.to(DEV), gate.to(DEV)
    want, s = res.double() + y * g, slack * g.abs() + 2.0 ** -23 * (y * g).abs()
    out = torch.empty_like(rd)
    assert l8.linear8(*args, res=rd, gate=gd, out=out) is out
    near(out, want, dtype, s)
    assert torch.equal(rd.cpu(), res)
    near(l8.linear8(*args, res=rd.clone()), res.double() + y, dtype, slack)
    inplace = rd.clone()
    assert l8.linear8(*args, res=inplace, gate=gd) is inplace and torch.equal(inplace, out)


def test_product_writes_only_its_rows_and_channels():
    """Strided, unaligned output inside a larger buffer."""
    dtype = torch.bfloat16
    x, w = rows((1, 70, 200), 11, dtype), randn((45, 200), 12, dtype)
    y, slack = product(x[0], w)
    for off in (0, 1, 8):
        buf = torch.full((1, 80, 64), 7.0, dtype=dtype, device=DEV)
        l8.linear8(x.to(DEV), w.to(DEV), out=buf[:, 5:75, off:off + 45])
        near(buf[0, 5:75, off:off + 45], y, dtype, slack)
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask[:, 5:75, off:off + 45] = False
        assert bool((buf[mask] == 7.0).all())


@pytest.mark.parametrize("M", [4, 300])
def test_non_finite_values_reach_their_rows_only(M):
    x, w = rows((1, M, 256), 13, torch.bfloat16), randn((64, 256), 14, torch.bfloat16)
    x[0, 1, 3], x[0, 2, 200] = float("inf"), float("nan")
    y = l8.linear8(x.to(DEV), w.to(DEV))[0].cpu()
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3:]).all()
    w[7, 9] = float("inf")
    y = l8.linear8(x.to(DEV), w.to(DEV))[0].cpu()
    assert torch.isnan(y[:, 7]).all() and torch.isfinite(y[0, :7]).all()


# ------------------------------------------------------------------------------------------------ gradients
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,L,K,N", [(1, 1, 128, 8), (1, 5, 100, 33), (2, 64, 256, 128), (1, 333, 520, 264), (1, 129, 130, 257), (1, 2000, 128, 64),
                                     (1, 2100, 390, 521), (1, 1500, 300, 520), (2, 1031, 640, 768), (1, 700, 130, 5)])
def test_training_step(dtype, B, L, K, N):
    x, w, b = rows((B, L, K), 15, dtype), (randn((N, K), 16) / math.sqrt(K)).to(dtype), randn((N,), 17, dtype)
    dy = rows((B, L, N), 18, dtype)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    out = l8.linear8(*leaves)
    dx, dw, db = torch.autograd.grad(out, leaves, dy.to(DEV))
    M = B * L
    y, slack = product(x.view(M, K), w, b)
    near(out.view(M, N), y, dtype, slack)
    d8, w8, x8, d = o.values(dy.view(M, N)), o.values(w, True), o.values(x.view(M, K)), dy.view(M, N).double()
    if dtype == torch.float16:
        x8 = x8.clamp(-65504, 65504)
    near(dx.view(M, K), *(lambda t: (t[0], dtype, t[1]))(sum8(d8, w8.t().contiguous())))
    near(dw, d.t() @ x8, dtype, M * 2.0 ** -23 * (d.abs().t() @ x8.abs()))
    near(db, d.sum(0), dtype, M * 2.0 ** -23 * d.abs().sum(0))
    dw2, db2 = l8.weight_grad(dy.to(DEV), l8.quantize(x.to(DEV)))
    assert torch.equal(dw2, dw) and torch.equal(db2, db)
    # one gradient at a time, the weight laid out beforehand, the rows quantised beforehand
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(l8.linear8(*some), some[i], dy.to(DEV))[0], (dx, dw, db)[i])
    p, (xl, wl, bl) = l8.pack(w.to(DEV)), leaves
    assert torch.equal(torch.autograd.grad(l8.linear8(xl, p, bl), xl, dy.to(DEV))[0], dx)
    assert torch.equal(torch.autograd.grad(l8.linear8(l8.quantize(x.to(DEV)), wl, bl), wl, dy.to(DEV))[0], dw)


def test_input_gradient_against_differences():
    """Inputs and steps on the blocks' grid make the layer linear where it is looked at: differences give dx for a gradient
    that the blocks hold exactly."""
    K, N = 128, 64
    x = torch.randint(-7, 8, (1, 4, K)).float()
    x[..., 0] = 448.0                                    # scale 1 in every block, small integers exact
    w = torch.randint(-7, 8, (N, K)).float()
    dy = torch.randint(-3, 4, (1, 4, N)).float()
    x[..., 1] = 1.0
    f = lambda t: (l8.linear8(t.bfloat16().to(DEV), w.bfloat16().to(DEV)).double().cpu() * dy.double()).sum().item()
    xl = x.bfloat16().to(DEV).requires_grad_()
    wl = w.bfloat16().to(DEV)
    dx, = torch.autograd.grad(l8.linear8(xl, wl), xl, dy.bfloat16().to(DEV))
    # y is rounded to bf16: differences of y are exact where |y| < 256, which the columns used here keep
    y = l8.linear8(xl.detach(), wl)
    for i, j in ((0, 5), (2, 77), (3, 127)):
        d = torch.zeros_like(x)
        d[0, i, j] = 1.0
        exact = (w[:, j].double() * dy[0, i].double()).sum().item()
        assert dx[0, i, j].item() == torch.tensor(exact).bfloat16().item()
        # half a step of bf16 for each of the two roundings of every y of the row
        slack = 2.0 ** -8 * ((y[0, i].double().abs().cpu() + 7) * dy[0, i].double().abs()).sum().item()
        assert abs((f(x + d) - f(x - d)) / 2 - exact) <= slack


@pytest.mark.parametrize("expanded", ["sum", "transposed"])
def test_gradients_of_any_layout(expanded):
    x, w = rows((1, 40, 256), 19, torch.bfloat16), randn((72, 256), 20, torch.bfloat16)
    leaves = [x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()]
    y = l8.linear8(*leaves)
    if expanded == "sum":
        got, dy = torch.autograd.grad(y.sum(), leaves), torch.ones_like(y)
    else:
        m = randn((72, 40), 21, torch.bfloat16).to(DEV)
        got, dy = torch.autograd.grad((y[0].t() * m).sum(), leaves), m.t()[None].contiguous()
    ref = torch.autograd.grad(l8.linear8(*leaves), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_refusals():
    x, w = rows((1, 4, 128), 22, torch.bfloat16).to(DEV), randn((64, 128), 23, torch.bfloat16).to(DEV)
    p = l8.pack(w, transposed=False)
    xr = x.clone().requires_grad_()
    with pytest.raises(ValueError):
        l8.linear8(xr, p)                                # no transposed form for dx
    with pytest.raises(NotImplementedError):
        l8.linear8(xr, w, epilogue="gelu_tanh")
    for call in (lambda: l8.linear8(x, w[:, :64]), lambda: l8.linear8(x, w, bias=w[0]), lambda: l8.linear8(x, w, w[:, 0].float()),
                 lambda: l8.linear8(x, w, res=x), lambda: l8.linear8(x, w, epilogue="gate_residual"),
                 lambda: l8.linear8(x, w, out=torch.empty((1, 4, 63), dtype=x.dtype, device=DEV)), lambda: l8.linear8(x, w.cpu()),
                 lambda: l8.quantize(x[:, :0]), lambda: l8.quantize(x.transpose(1, 2)), lambda: l8.pack(w[:0]),
                 lambda: l8.weight_grad(x, l8.quantize(x[:, :3])), lambda: l8.weight_grad(x.float(), l8.quantize(x)),
                 lambda: l8.linear8(x.double(), w.double())):
        with pytest.raises(ValueError):
            call()
    x8 = l8.quantize(x)
    with pytest.raises(ValueError):                      # the product would read what it writes
        l8.linear8(x8, l8.pack(w), out=x8.data.view(torch.bfloat16).view(-1)[:4 * 64].view(1, 4, 64))
    y = l8.linear8(xr, w)
    with pytest.raises(RuntimeError):                    # no second derivative
        torch.autograd.grad(torch.autograd.grad(y.sum(), xr, create_graph=True)[0].sum(), xr)


# ------------------------------------------------------------------------------------------------ GELU with its input kept in 8 bits
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("B,L,C", [(1, 1, 1), (1, 3, 128), (2, 77, 1000), (1, 130, 264)])
def test_gelu(dtype, keep8, B, L, C):
    x, dy = rows((B, L, C), 24, dtype), randn((B, L, C), 25, dtype)
    leaf = x.to(DEV).requires_grad_()
    y = blk.gelu_tanh(leaf, checkpoint8=keep8)
    dx, = torch.autograd.grad(y, leaf, dy.to(DEV))
    # fp32: the exponential's argument is off by 2^-22 of itself, which at most 100 is 2^-15 of the small values it gives; the
    # gate p = 1 / (1 + exp(-2u)) is 0 below 2^-126, the smallest normal number, so that x p may lack |x| 2^-126
    near(y, o.gelu(x.double()), dtype, 2.0 ** -15 * o.gelu(x.double()).abs() + 2.0 ** -126 * x.double().abs())
    h = o.values(x.view(-1, C)).view(x.shape) if keep8 else x.double()
    near(dx, dy.double() * o.gelu_slope(h), dtype, 2.0 ** -18 * dy.double().abs() * (1 + h.abs()) * (h.abs() < 20))
    assert torch.equal(blk.gelu_tanh(x.to(DEV)), y.detach())


def test_gelu_of_large_and_non_finite_values():
    x = torch.tensor([[[0.0, -0.0, 1e30, -1e30, 40.0, -40.0, float("inf"), float("nan")]]])
    leaf = x.to(DEV).requires_grad_()
    y = blk.gelu_tanh(leaf)
    dx, = torch.autograd.grad(y.sum(), leaf)
    assert y.flatten()[:6].tolist() == [0.0, 0.0, x[0, 0, 2].item(), 0.0, 40.0, 0.0] and y.flatten()[6].item() == float("inf")
    assert torch.isnan(y.flatten()[7]) and torch.isnan(dx.flatten()[7])
    assert dx.flatten()[:7].tolist() == [0.5, 0.5, 1.0, 0.0, 1.0, 0.0, 1.0]


# ------------------------------------------------------------------------------------------------ as they are used
def test_a_feed_forward_in_training():
    """Norm, up projection, GELU, down projection with every activation kept in 8 bits: one step's gradients against the same
    chain in float64, each operator from the tensors that the GPU chain gave it."""
    dtype, L, C, H = torch.bfloat16, 150, 256, 520
    x, dy = rows((1, L, C), 26, dtype).to(DEV), randn((1, L, C), 27, dtype).to(DEV)
    lw, lb = (1 + 0.1 * randn((C,), 28)).to(dtype).to(DEV), randn((C,), 29, dtype).to(DEV)
    w1, w2 = (randn((H, C), 30) / 16).to(dtype).to(DEV), (randn((C, H), 31) / 23).to(dtype).to(DEV)
    b1, b2 = randn((H,), 32, dtype).to(DEV), randn((C,), 33, dtype).to(DEV)
    leaves = [t.requires_grad_() for t in (x, lw, lb, w1, b1, w2, b2)]
    n = blk.ln_affine(x, lw, lb, checkpoint8=True)
    h = l8.linear8(n, w1, b1)
    a = blk.gelu_tanh(h, checkpoint8=True)
    y = l8.linear8(a, w2, b2)
    for t in (n, h, a):
        t.retain_grad()
    y.backward(dy)
    c = lambda t: t.detach().double().cpu().view(-1, t.shape[-1])
    sub = lambda g, v, s: near(g.cpu().view(v.shape), v, dtype, s)
    prod = lambda p, q: (p @ q, p.shape[1] * 2.0 ** -23 * (p.abs() @ q.abs()))
    prod8 = lambda p, q: sum8(p, q.t().contiguous())
    v2, v1 = o.values(c(w2), True), o.values(c(w1), True)
    sub(a.grad, *prod8(o.values(c(dy)), v2))
    sub(w2.grad, *prod(c(dy).t(), o.values(c(a))))
    hv = o.values(c(h))
    sub(h.grad, c(a.grad) * o.gelu_slope(hv), 2.0 ** -18 * c(a.grad).abs() * (1 + hv.abs()))
    sub(n.grad, *prod8(o.values(c(h.grad)), v1))
    sub(w1.grad, *prod(c(h.grad).t(), o.values(c(n))))
    sub(b1.grad, c(h.grad).sum(0), L * 2.0 ** -23 * c(h.grad).abs().sum(0))
    # the whole chain against autograd's own in float64 without 8-bit values: roundings of 2^-4 each, averaged over the sums
    xs = [t.detach().double().cpu().requires_grad_() for t in leaves]
    F = torch.nn.functional
    r = F.linear(F.gelu(F.linear(F.layer_norm(xs[0], (C,), xs[1], xs[2], 1e-6), xs[3], xs[4]), approximate="tanh"), xs[5], xs[6])
    ref = torch.autograd.grad(r, xs, dy.double().cpu())
    for got, want in zip(leaves, ref):
        cos = F.cosine_similarity(got.grad.double().cpu().flatten(), want.flatten(), dim=0).item()
        assert cos > 0.99, cos


def test_saved_rows_are_not_what_the_user_changes_later():
    x, w = rows((1, 20, 128), 34, torch.bfloat16).to(DEV), randn((64, 128), 35, torch.bfloat16).to(DEV).requires_grad_()
    ref, = torch.autograd.grad(l8.linear8(x, w).sum(), w)
    y = l8.linear8(x, w)
    x.zero_()
    got, = torch.autograd.grad(y.sum(), w)
    assert torch.equal(got, ref)


def test_on_another_stream_and_twice_at_once():
    x, w = rows((1, 300, 640), 36, torch.bfloat16).to(DEV), randn((260, 640), 37, torch.bfloat16).to(DEV)
    dy = randn((1, 300, 260), 38, torch.bfloat16).to(DEV)
    leaves = [t.requires_grad_() for t in (x, w)]
    step = lambda: [*(t := (l8.linear8(*leaves),)), *torch.autograd.grad(t[0], leaves, dy)]
    ref = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, ref))


def test_captured_and_replayed():
    x, dy = rows((1, 200, 384), 39, torch.bfloat16).to(DEV), randn((1, 200, 260), 40, torch.bfloat16).to(DEV)
    w, b = (t.to(DEV).requires_grad_() for t in (randn((260, 384), 41, torch.bfloat16), randn((260,), 42, torch.bfloat16)))
    lw, lb = (randn((384,), 43 + i, torch.bfloat16).to(DEV).requires_grad_() for i in range(2))

    def step():
        y = l8.linear8(blk.gelu_tanh(blk.ln_affine(x, lw, lb, checkpoint8=True), checkpoint8=True), w, b)
        return [y, *torch.autograd.grad(y, (w, b, lw, lb), dy)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (50, 51, 52):
        with torch.no_grad():
            x.copy_(rows((1, 200, 384), seed, torch.bfloat16))
            w.copy_(randn((260, 384), seed + 10, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        ref = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, r) for a, r in zip(out, ref))


@pytest.mark.parametrize("M", [5, 70])
def test_columns_of_one_buffer(M):
    """x, res and out side by side in the rows of one buffer are not an overlap; what lies between stays."""
    buf = randn((1, M, 640), 60, torch.bfloat16).to(DEV)
    w = l8.pack(randn((96, 256), 61, torch.bfloat16).to(DEV))
    was = buf.clone()
    x, res, out = buf[..., :256], buf[..., 256:352], buf[..., 400:496]
    ref = l8.linear8(x.clone(), w, epilogue="gate_residual", res=res.clone())
    l8.linear8(x, w, epilogue="gate_residual", res=res, out=out)
    assert torch.equal(out, ref)
    assert torch.equal(buf[..., :400], was[..., :400]) and torch.equal(buf[..., 496:], was[..., 496:])
    l8.linear8(x, w, epilogue="gate_residual", res=res)
    assert torch.equal(res, ref)
    for bad in (buf[..., 255:351], buf[..., 257:353]):
        with pytest.raises(ValueError, match="overlaps"):
            l8.linear8(x, w, epilogue="gate_residual", res=res, out=bad)


def test_a_captured_backward_refuses_leaves_of_a_living_eager_graph():
    """Refused before a gradient reaches the leaf; with the eager graph dropped the same capture runs and replays."""
    x, dy = rows((1, 40, 128), 63, torch.bfloat16).to(DEV), randn((1, 40, 64), 64, torch.bfloat16).to(DEV)
    w = randn((64, 128), 65, torch.bfloat16).to(DEV).requires_grad_()

    def step():
        return torch.autograd.grad(l8.linear8(x, w), w, dy)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    eager = l8.linear8(x, w)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        y = l8.linear8(x, w)
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


def test_rows_past_4_gib():
    """2.2 million rows of 2048, more than 2^32 elements: the same 4400 rows over and over, of -1, 0 and 1, so that every sum is exact
    in any order (their magnitudes stay under 2^24) and what the last rows give is what the first give."""
    n, times, K, N = 4400, 500, 2048, 64
    g = torch.Generator().manual_seed(70)
    base, dy1 = (torch.randint(-1, 2, (1, n, c), generator=g).to(torch.bfloat16).to(DEV) for c in (K, N))
    w = torch.randint(-1, 2, (N, K), generator=g).to(torch.bfloat16).to(DEV)
    x, dy = base.repeat(1, times, 1), dy1.repeat(1, times, 1)
    assert x.numel() > 1 << 32
    x8, w8 = l8.quantize(x), l8.pack(w)
    assert torch.equal(x8.dequantize()[:, -n:], base)
    ref = torch.nn.functional.linear(base.float(), w.float()).to(torch.bfloat16)
    for y in (l8.linear8(x8, w8), l8.linear8(x, w8)):
        assert torch.equal(y[:, -n:], ref) and torch.equal(y[:, :n], ref)
    dw, db = l8.weight_grad(dy, x8)
    assert torch.equal(dw, (times * (dy1[0].double().T @ base[0].double())).to(torch.bfloat16))
    assert torch.equal(db, (times * dy1[0].double().sum(0)).to(torch.bfloat16))
    del x8, dy, y
    lw, lb = torch.ones(K, dtype=torch.bfloat16, device=DEV), torch.zeros(K, dtype=torch.bfloat16, device=DEV)
    for op in (lambda t: blk.gelu_tanh(t, checkpoint8=True), lambda t: blk.ln_affine(t, lw, lb, checkpoint8=True),
               lambda t: blk.ln_affine(t, lw, lb)):
        few, many = base.clone().requires_grad_(), x.requires_grad_()
        a, b = op(few), op(many)
        assert torch.equal(a, b[:, -n:])
        da, = torch.autograd.grad(a, few, base)
        dm, = torch.autograd.grad(b, many, x.detach())
        assert torch.equal(da, dm[:, -n:])
        del a, b, dm


@pytest.mark.parametrize("N,K", [(1, 1), (130, 300), (700, 513), (512, 512)])
def test_a_weights_scales_are_whole_words(N, K):
    """What lies behind a row's blocks in the scales is written too, whatever was in the memory before."""
    torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV)
    w = randn((N, K), 71, torch.bfloat16).to(DEV)
    p = l8.pack(w)
    for s, n, k in ((p.scale, N, K), (p.scale_t, K, N)):
        assert s.shape == (-(-n // 128), -(-k // 512) * 4)
        assert bool((s[:, :-(-k // 128)] > 0).all()) and not s[:, -(-k // 128):].any()
    q = l8.pack(w)
    assert all(torch.equal(getattr(p, a), getattr(q, a)) for a in ("data", "scale", "data_t", "scale_t"))
