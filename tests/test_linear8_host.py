"""Refusals of the 8-bit block operators at the C boundary and in Python: nothing touches a device."""
import ctypes as C
import os
import re

import pytest
import torch

import self_forcing_amd as sfa
from self_forcing_amd import lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20          # a 16-byte aligned address that no refused call reads


def _rc(rc, code, text):
    assert rc == code and text in L.load().sfm_last_error().decode()


def test_struct_size_matches_the_header():
    assert C.sizeof(L.Linear8Desc) == 2 * 4 + 8 + 2 * 4 + 3 * 8 + 2 * 4


def test_header_macros_are_what_the_host_allocates():
    text = open(os.path.join(ROOT, "include", "sfm_attn.h")).read()
    assert re.search(r"SFM_PAD8\(n\) \(\(\(int64_t\)\(n\) \+ 127\) / 128 \* 128\)", text)
    assert re.search(r"SFM_PITCH8\(n\) \(\(\(int64_t\)\(n\) \+ 511\) / 512 \* 4\)", text)


def test_quantize_dequantize_pack_refusals():
    lib = L.load()
    q = lambda dt=0, r=4, K=128, x=P, xs=128, d=2 * P, s=3 * P, y=None, ys=0, cs=None: lib.sfm_quantize8(dt, r, K, x, xs, d, s, y, ys, cs, None)
    _rc(q(dt=7), -2, "dtype")
    for r, K in ((0, 128), (4, 0), (1 << 31, 128), (4, 1 << 23)):
        _rc(q(r=r, K=K, xs=1 << 24), -3, "rows=")
    _rc(q(x=None), -1, "non-NULL")
    _rc(q(d=None, s=None), -1, "non-NULL")
    _rc(q(s=None), -1, "scale")
    _rc(q(xs=127), -5, "x: rows")
    _rc(q(x=P + 1), -7, "x is not aligned")
    _rc(q(d=2 * P + 8), -7, "16-byte")
    _rc(q(y=P, ys=100), -5, "y: rows")
    _rc(q(cs=P + 2), -7, "colsum")
    _rc(lib.sfm_dequantize8(0, 4, 128, P, 2 * P, None, 128, None), -1, "y must")
    _rc(lib.sfm_dequantize8(0, 4, 128, P, None, 3 * P, 128, None), -1, "scale")
    _rc(lib.sfm_dequantize8(2, 4, 128, P, 2 * P, 3 * P, 127, None), -5, "y: rows")
    _rc(lib.sfm_pack8(0, 4, 128, None, 128, P, P, None, None, None), -1, "w must")
    _rc(lib.sfm_pack8(0, 4, 128, P, 100, P, P, None, None, None), -5, "w: rows")
    _rc(lib.sfm_pack8(0, 4, 128, P, 128, P, P, P, None, None), -1, "transposed")


def _desc(**kw):
    d = L.Linear8Desc(0, L.EPI_NONE, 16, 64, 128, 64, 64, 64, 1, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_product_refusals():
    lib = L.load()

    def f(d=None, x=P, xs=2 * P, w=3 * P, ws=4 * P, b=None, res=None, gate=None, out=5 * P):
        return lib.sfm_linear8(C.byref(_desc() if d is None else d), x, xs, w, ws, b, res, gate, out, None)
    _rc(f(_desc(dtype=2)), -2, "dtype")
    for kw in (dict(M=0), dict(N=0), dict(K=0), dict(M=1 << 31)):
        _rc(f(_desc(**kw)), -3, "rows=")
    _rc(f(_desc(epilogue=9)), -3, "epilogue")
    _rc(f(out=None), -1, "out")
    _rc(f(xs=None), -1, "x8")
    _rc(f(ws=None), -1, "w8")
    _rc(f(w=3 * P + 4), -7, "w8")
    _rc(f(_desc(out_stride=63)), -5, "out")
    _rc(f(out=5 * P + 1), -7, "out")
    _rc(f(b=P + 1), -7, "bias")
    _rc(f(_desc(epilogue=L.EPI_GATE_RESIDUAL)), -1, "res")
    _rc(f(_desc(epilogue=L.EPI_GATE_RESIDUAL, res_stride=1), res=6 * P), -5, "res")
    _rc(f(_desc(epilogue=L.EPI_GATE_RESIDUAL, rows_per_frame=0), res=6 * P, gate=7 * P), -5, "rows_per_frame")
    _rc(f(out=P + 2), -6 + 2, "overlaps")
    _rc(f(out=3 * P + 64 * 128 - 2), -4, "overlaps")


def test_forward_refusals():
    lib = L.load()

    def f(d=None, x=P, xs=128, data=2 * P, scale=3 * P, out=6 * P):
        return lib.sfm_linear8_fwd(C.byref(_desc() if d is None else d), x, xs, data, scale, 4 * P, 5 * P, None, None, None, out, None)
    _rc(f(x=None), -1, "x must")
    _rc(f(xs=127), -5, "x: rows")
    _rc(f(x=P + 1), -7, "x is not")
    _rc(f(data=None), -1, "x8")
    _rc(f(scale=None), -1, "x8")
    _rc(f(_desc(M=17), data=None, scale=None), -1, "x8")
    _rc(f(_desc(dtype=2)), -2, "dtype")
    _rc(f(out=P + 64), -4, "overlaps x")
    _rc(f(out=2 * P + 64), -4, "overlaps x8")
    _rc(f(data=None, scale=None, out=4 * P + 64), -4, "overlaps w8")
    text = open(os.path.join(ROOT, "include", "sfm_attn.h")).read()
    assert f"#define SFM_LINEAR8_FEW_ROWS {L.LINEAR8_FEW_ROWS}\n" in text


def test_gradient_refusals():
    lib = L.load()
    n = C.c_size_t(0)
    assert lib.sfm_linear8_wgrad_workspace_bytes(300, 64, 128, C.byref(n)) == 0 and n.value >= 10 * 64 * 4
    need = n.value
    _rc(lib.sfm_linear8_wgrad_workspace_bytes(300, 64, 128, None), -1, "bytes")
    _rc(lib.sfm_linear8_wgrad_workspace_bytes(0, 64, 128, C.byref(n)), -3, "rows=")

    def f(dt=0, M=300, dy=P, dys=64, x=2 * P, xs=3 * P, dw=4 * P, db=5 * P, cs=None, ws=6 * P, wb=need):
        return lib.sfm_linear8_wgrad(dt, M, 64, 128, dy, dys, x, xs, dw, db, cs, ws, wb, None)
    _rc(f(dt=2), -2, "dtype")
    _rc(f(M=0), -3, "rows=")
    _rc(f(dy=None), -1, "dy")
    _rc(f(dw=None, db=None), -1, "dy")
    _rc(f(dys=63), -5, "dy")
    _rc(f(x=None), -1, "x8")
    _rc(f(dw=4 * P + 1), -7, "dw")
    _rc(f(ws=None), -6, "workspace")
    _rc(f(ws=6 * P + 16), -6, "workspace")
    _rc(f(wb=need - 1), -6, "workspace")
    assert lib.sfm_linear8_bwd_workspace_bytes(300, 64, 128, C.byref(n)) == 0 and n.value >= 300 * 128 + need
    all_of = n.value
    _rc(lib.sfm_linear8_bwd_workspace_bytes(300, 64, 128, None), -1, "bytes")
    _rc(lib.sfm_linear8_bwd_workspace_bytes(300, 0, 128, C.byref(n)), -3, "rows=")

    def g(dt=0, dy=P, dys=64, wt=7 * P, st=8 * P, x=2 * P, xs=3 * P, dx=9 * P, dw=4 * P, db=5 * P, ws=6 * P, wb=all_of):
        return lib.sfm_linear8_bwd(dt, 300, 64, 128, dy, dys, wt, st, x, xs, dx, dw, db, ws, wb, None)
    _rc(g(dt=2), -2, "dtype")
    _rc(g(dy=None), -1, "dy")
    _rc(g(dx=None, dw=None, db=None), -1, "one of dx")
    _rc(g(wt=None), -1, "transposed")
    _rc(g(x=None), -1, "x8")
    _rc(g(dys=63), -5, "dy")
    _rc(g(dx=9 * P + 1), -7, "dx")
    _rc(g(ws=6 * P + 8), -6, "workspace")
    _rc(g(wb=all_of - 1), -6, "workspace")
    _rc(lib.sfm_gelu_bwd(0, 4, 128, None, 0, None, P, P, 128, P, 128, None), -1, "gelu_bwd")
    _rc(lib.sfm_gelu_bwd(0, 4, 128, P, 128, None, None, None, 128, P, 128, None), -1, "dy")
    _rc(lib.sfm_gelu_bwd(0, 4, 128, P, 127, None, None, P, 128, P, 128, None), -5, "x: rows")


def test_layer_norm_refusals():
    lib = L.load()
    n = C.c_size_t(0)
    assert lib.sfm_ln_bwd_workspace_bytes(60, 64, 20, C.byref(n)) == 0 and n.value >= 3 * 2 * 64 * 4
    need = n.value
    for rows, Cc, g in ((60, 12, 20), (60, 8200, 20), (0, 64, 1), (60, 64, 7), (60, 64, 0)):
        assert lib.sfm_ln_bwd_workspace_bytes(rows, Cc, g, C.byref(n)) == -3

    def f(dt=0, x=P, xs=64, data=None, sc8=None, rstd=None, dy=P, dys=64, w=None, sc=2 * P, ms=64, g=20, dx=3 * P, dxs=64, dw=4 * P, db=5 * P,
          ws=6 * P, wb=need):
        return lib.sfm_ln_bwd(dt, 60, 64, 1e-6, x, xs, data, sc8, rstd, dy, dys, w, sc, ms, g, dx, dxs, dw, db, ws, wb, None)
    _rc(f(dt=5), -2, "dtype")
    _rc(f(g=7), -3, "groups")
    _rc(f(sc=None), -1, "one of weight and scale")
    _rc(f(w=P), -1, "one of weight and scale")
    _rc(f(x=None), -1, "rstd")
    _rc(f(x=None, rstd=P), -1, "ln_bwd")
    _rc(f(ms=4), -5, "mod_stride")
    _rc(f(dys=63), -5, "strides")
    _rc(f(dx=3 * P + 2), -7, "16-byte")
    _rc(f(ws=None), -6, "workspace")
    _rc(f(wb=need - 1), -6, "workspace")
    k = lambda data=P, rstd=P, y=P, sc=P: lib.sfm_ln_keep8(0, 60, 64, 1e-6, P, 64, y, 64, sc, P, 64, 20, None, None, data, P, rstd, None)
    _rc(k(rstd=None), -1, "rstd")
    _rc(k(sc=None), -1, "scale")
    _rc(k(data=None), -1, "ln_keep8")
    _rc(k(data=P + 4), -7, "ln_keep8")


def test_python_entry_points_refuse_before_any_call():
    x, w = torch.zeros((1, 4, 128), dtype=torch.bfloat16), torch.zeros((64, 128), dtype=torch.bfloat16)
    l8, blk = sfa.linear8, sfa.block_ops
    for call in (lambda: l8.quantize(x), lambda: l8.pack(w), lambda: l8.linear8(x, w), lambda: blk.gelu_tanh(x),
                 lambda: blk.ln_affine(x, w[0], w[0], checkpoint8=True), lambda: blk.ln_affine_backward(x, x, w[0]),
                 lambda: l8.linear8(x, w, epilogue="relu"), lambda: l8.linear8(x.float(), w.float()), lambda: l8.linear8(x, w.half()),
                 lambda: l8.linear8(x, w[0])):
        with pytest.raises(ValueError):
            call()


def test_rows_of_one_buffer_overlap_only_where_they_do():
    """out may be columns of the rows that x or res are columns of; by one column too far, or with other strides, it is refused."""
    lib = L.load()
    d = dict(M=8, N=64, K=128, out_stride=256)

    def f(out, xs=256):
        return lib.sfm_linear8_fwd(C.byref(_desc(**d)), P, xs, None, None, 4 * P, 5 * P, None, None, None, out, None)
    for out in (P + 2 * 64, P + 2 * 127, P - 2 * 63, P + 2 * (256 - 63), P + 2 * (256 * 7 + 127)):
        _rc(f(out), -4, "overlaps x")
    _rc(f(P + 2 * 128, xs=257), -4, "overlaps x")                 # other strides: rows cross
    for res in (7 * P + 2, 7 * P - 2, 7 * P + 2 * 63, 7 * P + 2 * 256):
        e = _desc(**d, epilogue=L.EPI_GATE_RESIDUAL, res_stride=256)
        _rc(lib.sfm_linear8_fwd(C.byref(e), P, 128, None, None, 4 * P, 5 * P, None, res, None, 7 * P, None), -4, "overlaps res")
    e = _desc(**d, epilogue=L.EPI_GATE_RESIDUAL, res_stride=320)
    _rc(lib.sfm_linear8_fwd(C.byref(e), P, 128, None, None, 4 * P, 5 * P, None, 7 * P, None, 7 * P, None), -4, "overlaps res")


def test_a_captured_backward_refuses_leaves_of_an_eager_graph(monkeypatch):
    """The rule without a GPU: graphs recorded on the default stream are remembered while they live."""
    blk = sfa.block_ops
    stream = [0]
    monkeypatch.setattr(blk, "_raw_stream", lambda index: stream[0])
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            blk._noted(ctx, x.device)
            return x * 2 + w

        @staticmethod
        @blk._once
        def backward(ctx, dy):
            return dy * 2, dy
    w, v = (torch.randn(3, requires_grad=True) for _ in range(2))
    dy = torch.ones(3)
    eager = Twice.apply(torch.ones(3), w)

    def captured(leaf):
        stream[0], capturing[0] = 5, True
        try:
            return torch.autograd.grad(Twice.apply(torch.ones(3), leaf), leaf, dy)[0]
        finally:
            stream[0], capturing[0] = 0, False
    with pytest.raises(RuntimeError, match="same leaves"):
        captured(w)
    assert torch.equal(captured(v), dy)
    assert torch.equal(torch.autograd.grad(eager, w, dy, retain_graph=True)[0], dy)      # the eager one still runs
    with pytest.raises(RuntimeError, match="same leaves"):
        captured(w)
    del eager
    assert torch.equal(captured(w), dy)
    stream[0] = 3
    other = Twice.apply(torch.ones(3), w)                         # recorded on a stream of the user's
    assert torch.equal(captured(w), dy) and other is not None
