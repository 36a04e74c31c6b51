"""LayerNorm's backward and its 8-bit checkpoint on the GPU against the float64 oracle.

Tolerances.  A row's sums are fp32, at most 64 additions deep in any lane and 10 over lanes and waves: E = 80 * 2^-24 of the
magnitudes summed.  With x off by that of its mean, xh is off by e = E (|xh| + (|mean| + mean|x|) r); what follows from it in
dx and in the column sums is first order in e, and the column sums over R rows add R 2^-24 of theirs.  With the checkpoint,
an xh within e of the border between two e4m3 values may land on either: their distance is allowed where it is so."""
import pytest
import torch

import self_forcing_amd as sfa
from gpu_util import randn
from oracle import blocks8 as o
from test_gpu_linear8 import near, rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
blk = sfa.block_ops
E = 80 * 2.0 ** -24


def reference(x, dy, w, groups, keep8, eps=1e-6):
    """x, dy [R, C], w [R, C] or [C] (double): (dx, dw, db) and their slacks; sums over `groups` equal runs of rows."""
    x, dy = x.double(), dy.double()
    R, C = x.shape
    xh, r = o.ln_parts(x, eps)
    e = E * (xh.abs() + (x.mean(-1, keepdim=True).abs() + x.abs().mean(-1, keepdim=True)) * r)
    if keep8:
        lo, hi = o.values(xh - e), o.values(xh + e)
        xh = o.values(xh)
        e = torch.maximum((hi - xh).abs(), (lo - xh).abs()) + 2.0 ** -30
    dx, dyxh = o.ln_grads(dy, xh, r, w)
    g = (dy * w).abs()
    mgx, mg = (g * xh.abs()).mean(-1, keepdim=True), g.mean(-1, keepdim=True)
    sx = r * (3 * E * (g + mg + xh.abs() * mgx) + e * mgx + xh.abs() * (g * e).mean(-1, keepdim=True))
    per = lambda t: t.view(groups, -1, C).sum(1)
    n = (R // groups + 80) * 2.0 ** -24
    return (dx, per(dyxh), per(dy)), (sx, per(dy.abs() * e) + n * per(dyxh.abs()), n * per(dy.abs()))


def check(got, want, dtype):
    for g, ref, slack in zip(got, *want):
        near(g.reshape(ref.shape), ref, dtype, slack)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("B,L,C", [(1, 1, 8), (1, 3, 1536), (2, 65, 136), (1, 777, 1000), (1, 40, 5120), (1, 9, 8192), (1, 5, 1544)])
def test_affine(dtype, keep8, B, L, C):
    x, dy = rows((B, L, C), 1, dtype), randn((B, L, C), 2, dtype)
    w, b = (1 + 0.3 * randn((C,), 3)).to(dtype), randn((C,), 4, dtype)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = blk.ln_affine(*leaves, checkpoint8=keep8)
    assert torch.equal(y.detach(), blk.ln_affine(x.to(DEV), w.to(DEV), b.to(DEV)))          # the forward is the one there was
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    check(got, reference(x.view(-1, C), dy.view(-1, C), w.double(), 1, keep8), dtype)
    if not keep8:
        raw = blk.ln_affine_backward(dy.to(DEV), x.to(DEV), w.to(DEV))
        assert all(torch.equal(a, r) for a, r in zip(got, raw))
    # the same again: the sums have one order
    assert all(torch.equal(a, r) for a, r in zip(got, torch.autograd.grad(blk.ln_affine(*leaves, checkpoint8=keep8), leaves, dy.to(DEV))))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("B,F,per,C", [(1, 1, 1, 64), (1, 3, 40, 1536), (2, 2, 7, 256), (1, 5, 1, 128), (1, 2, 30, 5120)])
def test_modulated(dtype, keep8, B, F, per, C):
    x, dy = rows((B, F * per, C), 5, dtype), randn((B, F * per, C), 6, dtype)
    e = (0.3 * randn((B, F, 6, C), 7)).to(dtype)
    xd, ed = x.to(DEV).requires_grad_(), e.to(DEV).requires_grad_()
    sh, sc = ed.chunk(6, dim=2)[:2]
    y = blk.ln_modulate(xd, sc, sh, checkpoint8=keep8)
    assert torch.equal(y.detach(), blk.ln_modulate(x.to(DEV), sc.detach(), sh.detach()))
    dx, de = torch.autograd.grad(y, (xd, ed), dy.to(DEV))
    w = (1 + e[:, :, 1:2].double()).expand(B, F, per, C).reshape(-1, C)
    check((dx, de[:, :, 1], de[:, :, 0]), reference(x.view(-1, C), dy.view(-1, C), w, B * F, keep8), dtype)
    assert not de[:, :, 2:].any()
    if not keep8:
        raw = blk.ln_modulate_backward(dy.to(DEV), x.to(DEV), sc.detach())
        assert torch.equal(raw[0], dx) and torch.equal(raw[1], de[:, :, 1:2]) and torch.equal(raw[2], de[:, :, 0:1])


def test_broadcast_modulation_and_shared_leaves():
    """One row of modulation for all frames and videos, and one tensor as both scale and shift."""
    x, dy = rows((2, 30, 64), 8, torch.float32).to(DEV), randn((2, 30, 64), 9).to(DEV)
    m = (0.3 * randn((64,), 10)).to(DEV).requires_grad_()
    e = m.expand(2, 3, 1, 64)
    got, = torch.autograd.grad(blk.ln_modulate(x, e, e), m, dy)
    (_, dw, db), (_, sw, sb) = reference(x.cpu().view(-1, 64), dy.cpu().view(-1, 64), 1 + m.detach().double().cpu(), 6, False)
    near(got, (dw + db).sum(0), torch.float32, (sw + sb).sum(0) + 12 * 2.0 ** -24 * (dw.abs() + db.abs()).sum(0))


def test_gradients_against_differences():
    x, dy = rows((1, 4, 64), 11, torch.float32), randn((1, 4, 64), 12)
    w, b = 1 + 0.3 * randn((64,), 13), randn((64,), 14)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(blk.ln_affine(*leaves), leaves, dy.to(DEV))
    f = lambda *t: (blk.ln_affine(*(v.to(DEV) for v in t)).double().cpu() * dy.double()).sum().item()
    h = 2.0 ** -6
    for which, at in ((0, (0, 1, 5)), (0, (0, 3, 63)), (1, (7,)), (2, (20,))):
        t = [x.clone(), w.clone(), b.clone()]
        d = torch.zeros_like(t[which])
        d[at] = h
        up, down = list(t), list(t)
        up[which], down[which] = t[which] + d, t[which] - d
        num = (f(*up) - f(*down)) / (2 * h)
        # differences: the third derivative's h^2 (a row's values are of order 1 to its spread), and the fp32 outputs' 2^-22 / h
        assert abs(num - grads[which][at].item()) < 2e-2 * max(1.0, abs(num))


def test_other_layouts():
    """Rows inside a wider buffer, gradients expanded from a sum and off the 16-byte grid."""
    dtype, C = torch.bfloat16, 256
    buf, w, b = rows((1, 50, 512), 15, dtype).to(DEV), randn((C,), 16, dtype).to(DEV), randn((C,), 17, dtype).to(DEV)
    x = buf[..., 128:384].requires_grad_()
    xc = x.detach().contiguous().requires_grad_()
    dyb = randn((1, 50, C + 8), 18, dtype).to(DEV)
    for dy in (torch.ones((), dtype=dtype, device=DEV).expand(1, 50, C), dyb[..., 3:3 + C], dyb[..., 8:]):
        for keep8 in (False, True):
            got, = torch.autograd.grad(blk.ln_affine(x, w, b, checkpoint8=keep8), x, dy)
            ref, = torch.autograd.grad(blk.ln_affine(xc, w, b, checkpoint8=keep8), xc, dy.contiguous())
            assert torch.equal(got, ref)


def test_rows_of_one_value_and_non_finite_rows():
    x = torch.zeros((1, 4, 64))
    x[0, 1], x[0, 2, 5], x[0, 3] = 3.0, float("inf"), torch.linspace(-1, 1, 64)
    for keep8 in (False, True):
        xl = x.to(DEV).requires_grad_()
        w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
        y = blk.ln_affine(xl, w, b, checkpoint8=keep8)
        dx, = torch.autograd.grad(y, xl, torch.ones_like(y))
        assert not dx[0, :2].any() and torch.isnan(dx[0, 2]).all() and torch.isfinite(dx[0, 3]).all()


def test_an_input_changed_in_place_is_noticed():
    x, y = (rows((1, 8, 64), 20 + i, torch.bfloat16).to(DEV) for i in range(2))
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV).requires_grad_()
    out = blk.ln_affine(x, w, w.detach())
    blk.gate_residual_(x, y)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.sum(), w)
    out = blk.ln_affine(x, w, w.detach(), checkpoint8=True)      # the checkpoint does not need x
    blk.gate_residual_(x, y)
    torch.autograd.grad(out.sum(), w)


def test_refusals():
    x, w = rows((1, 12, 64), 22, torch.bfloat16).to(DEV), torch.ones(64, dtype=torch.bfloat16, device=DEV)
    m = torch.zeros((1, 3, 1, 64), dtype=torch.bfloat16, device=DEV)
    xl = x.clone().requires_grad_()
    for call in (lambda: blk.ln_affine(xl, w.float(), w), lambda: blk.ln_affine(xl, w, w[:32]), lambda: blk.ln_affine(xl.transpose(1, 2), w[:12], w[:12]),
                 lambda: blk.ln_modulate(xl, m, m[:, :1]), lambda: blk.ln_modulate(x, m[:, :1], m), lambda: blk.ln_modulate(xl, m.float(), m),
                 lambda: blk.ln_affine(xl[..., :12], w[:12], w[:12], checkpoint8=True), lambda: blk.ln_affine_backward(x[:, :4], x, w),
                 lambda: blk.ln_affine_backward(x.float(), x, w), lambda: blk.ln_modulate_backward(x, x, m[..., :32]),
                 lambda: blk.gelu_tanh(xl.transpose(1, 2)), lambda: blk.gelu_tanh(xl.double())):
        with pytest.raises(ValueError):
            call()
