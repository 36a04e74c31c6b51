"""Linear layers on 8-bit blocks (`sfm_linear8`), for serving and for training; no counterpart in the reference, whose linear
layers are 16 bits (wan/modules/model.py:592-650).

    w8 = pack(weight)                    # once, where the weights stay: half their memory
    y = linear8(x, w8, bias)             # x in 8 bits per call, sums kept in fp32, one rounding
    y = linear8(x, weight, bias)         # under autograd: weight packed in the call, x kept in 8 bits for the weight's gradient

A block is 128 consecutive values of a row (128 x 128 of a weight) with the smallest power of two 2^s such that their largest
magnitude is at most 448 * 2^s; a value is kept as e4m3 of v / 2^s, ties to even (half a step: 2^-4 of it), NaN where it is not
finite, 240 * 2^120 where it would round up to 2^128.

The product runs on e4m3 matrix instructions, which add the products of 8 neighbouring channels before the fp32 sum and drop of them
what is below 2^-13 of the largest: 1.7e-5 of the result on random rows, where the values' own rounding makes 2.6e-2.

The gradients are those of the product with the rounding passed through: dx = dy8 w8 (dy in 8-bit blocks too), dw = dy^T x8 with dy
as it is, dbias = sum of dy.  (In fp16 dw takes 65504 for a value of x8 that was rounded up to 65536.)"""
import ctypes as C
import functools

import torch

from . import lib as _l
from .block_ops import _HALF, _like, _mod, _noted, _once, _row_stride, _rows, _save, _saved, _written
from .monarch_attn import _DT, _on_device, _raw_stream, _stream

_EPI = {"none": _l.EPI_NONE, "gelu_tanh": _l.EPI_GELU_TANH, "gate_residual": _l.EPI_GATE_RESIDUAL}


def _pad(n):
    return -(-n // 128) * 128


class Rows8:
    """Rows [B, L, K] in 8-bit blocks: `data` uint8 [B * L, K rounded up to 128] (e4m3), `scale` uint8 (exponents + 127; the
    order is include/sfm_attn.h's).  `dtype` is that of the rows it was made from."""

    __slots__ = ("data", "scale", "shape", "dtype")

    def __init__(self, data, scale, shape, dtype):
        self.data, self.scale, self.shape, self.dtype = data, scale, torch.Size(shape), dtype

    @property
    def device(self):
        return self.data.device

    def dequantize(self, dtype=None):
        """The values the blocks stand for, rounded to `dtype` (default: the rows' own)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DT:
            raise ValueError(f"unsupported dtype {dtype}")
        y = torch.empty(self.shape, dtype=dtype, device=self.device)
        with _on_device(self.device):
            _l.check(_l.load().sfm_dequantize8(_DT[dtype], self.shape[0] * self.shape[1], self.shape[2], self.data.data_ptr(),
                                               self.scale.data_ptr(), y.data_ptr(), self.shape[2], _stream(y)))
        return y


class Weight8:
    """A weight [N, K] in 128 x 128 blocks, and (unless packed without) transposed, for the gradient of the input: a snapshot of
    the weight at `pack`.  `dequantize()` gives its values."""

    __slots__ = ("data", "scale", "data_t", "scale_t", "shape", "dtype")

    def __init__(self, data, scale, data_t, scale_t, shape, dtype):
        self.data, self.scale, self.data_t, self.scale_t = data, scale, data_t, scale_t
        self.shape, self.dtype = torch.Size(shape), dtype

    @property
    def device(self):
        return self.data.device

    def dequantize(self, dtype=None):
        N, K = self.shape
        dtype = self.dtype if dtype is None else dtype
        s = self.scale[:, :-(-K // 128)].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
        v = torch.ldexp(self.data[:, :K].contiguous().view(torch.float8_e4m3fn).double(), s.to(torch.int32) - 127)
        return (v.clamp(-65504.0, 65504.0) if dtype == torch.float16 else v).to(dtype)


def _empty_rows(rows, K, device):
    n = -(-rows // 128) * _pad(K)
    return torch.empty((rows, _pad(K)), dtype=torch.uint8, device=device), torch.empty(n, dtype=torch.uint8, device=device)


def quantize(x):
    """[B, L, K] rows (bf16, fp16 or fp32; any K) in 8-bit blocks.  Not differentiable.  linear8 takes blocks of 16-bit rows."""
    x = x.detach()
    rows, K, xs = _rows(x)
    data, scale = _empty_rows(rows, K, x.device)
    with _on_device(x.device):
        _l.check(_l.load().sfm_quantize8(_DT[x.dtype], rows, K, x.data_ptr(), xs, data.data_ptr(), scale.data_ptr(), None, 0, None, _stream(x)))
    return Rows8(data, scale, x.shape, x.dtype)


def pack(weight, transposed=True):
    """[N, K] weight (bf16, fp16 or fp32) in 8-bit blocks: lay it out once where it stays, again when it has changed.  The
    transposed form (another N * K bytes) is needed for gradients of the input only."""
    if not weight.is_cuda:
        raise ValueError("the block operators run on the GPU")
    if weight.dtype not in _DT or weight.dim() != 2:
        raise ValueError("weight must be a [N, K] tensor of bf16, fp16 or fp32")
    weight = weight.detach()
    if weight.stride(1) != 1 or weight.stride(0) < weight.shape[1]:
        weight = weight.contiguous()
    N, K = weight.shape
    if N < 1 or K < 1:
        raise ValueError("weight is empty")
    ws = weight.stride(0) if N > 1 else K            # the stride of a dimension of one says nothing

    def blocks(n, k):
        return (torch.empty((n, _pad(k)), dtype=torch.uint8, device=weight.device),
                torch.empty((-(-n // 128), -(-k // 512) * 4), dtype=torch.uint8, device=weight.device))
    data, scale = blocks(N, K)
    data_t, scale_t = blocks(K, N) if transposed else (None, None)
    with _on_device(weight.device):
        _l.check(_l.load().sfm_pack8(_DT[weight.dtype], N, K, weight.data_ptr(), ws, data.data_ptr(), scale.data_ptr(),
                                     data_t.data_ptr() if transposed else None, scale_t.data_ptr() if transposed else None, _stream(weight)))
    return Weight8(data, scale, data_t, scale_t, (N, K), weight.dtype)


def _desc(dtype, rows, N, K, out, epi, res, gate):
    """(descriptor, gate tensor to hold on to or None)."""
    if res is None:
        return _l.Linear8Desc(_DT[dtype], epi, rows, N, K, _row_stride(out), 0, 0, 0, 0), None
    g, gs, rpf = (None, 0, 1) if gate is None else _mod(gate, res)
    return _l.Linear8Desc(_DT[dtype], epi, rows, N, K, _row_stride(out), _rows(res)[2], gs, rpf, 0), g


def _ptr(t):
    return None if t is None else t.data_ptr()


def _product(x8, w_data, w_scale, N, bias, out, epi=_l.EPI_NONE, res=None, gate=None):
    B, L, K = x8.shape
    d, g = _desc(out.dtype, B * L, N, K, out, epi, res, gate)
    with _on_device(out.device):
        _l.check(_l.load().sfm_linear8(C.byref(d), x8.data.data_ptr(), x8.scale.data_ptr(), w_data.data_ptr(), w_scale.data_ptr(),
                                       _ptr(bias), _ptr(res), _ptr(g), out.data_ptr(), _stream(out)))
    return out


def _forward(x, w8, bias, out, keep, epi=_l.EPI_NONE, res=None, gate=None):
    """Quantisation and product in one call; returns the rows' blocks where they are to be kept (few rows have none otherwise)."""
    rows, K, xs = _rows(x)
    d, g = _desc(x.dtype, rows, w8.shape[0], K, out, epi, res, gate)
    data = scale = data_at = scale_at = None
    if keep:
        data, scale = _empty_rows(rows, K, x.device)
        data_at, scale_at = data.data_ptr(), scale.data_ptr()
    elif rows > _l.LINEAR8_FEW_ROWS:                 # one piece of scratch for both
        scratch = torch.empty((rows + -(-rows // 128)) * _pad(K), dtype=torch.uint8, device=x.device)
        data_at = scratch.data_ptr()
        scale_at = data_at + rows * _pad(K)
    with _on_device(x.device):
        _l.check(_l.load().sfm_linear8_fwd(C.byref(d), x.data_ptr(), xs, data_at, scale_at, w8.data.data_ptr(), w8.scale.data_ptr(),
                                           _ptr(bias), _ptr(res), _ptr(g), out.data_ptr(), _stream(x)))
    return data, scale


@functools.lru_cache(maxsize=1024)
def _bytes(query, rows, N, K, device_index):
    """Workspace that the named query asks for on a device (its compute units are in the size)."""
    n = C.c_size_t(0)
    with torch.cuda.device(device_index):
        _l.check(getattr(_l.load(), query)(rows, N, K, C.byref(n)))
    return n.value


def weight_grad(dy, x8):
    """(dw [N, K], dbias [N]) of a layer from its output's gradient dy [B, L, N] and the rows its forward kept in 8 bits (of
    fp16 rows where dy is fp16; a row's value then counts as 65504 where its block rounded it up to 65536)."""
    dy = dy.detach()
    if dy.dtype not in _HALF:
        raise ValueError("weight_grad takes float16 / bfloat16 gradients")
    if not isinstance(x8, Rows8) or dy.dim() != 3 or dy.shape[:2] != x8.shape[:2]:
        raise ValueError("expected dy [B, L, N] and the Rows8 of a [B, L, K] input")
    if dy.device != x8.device:
        raise ValueError(f"dy on {dy.device}, the rows on {x8.device}")
    if dy.dtype == torch.float16 and x8.dtype != torch.float16:
        raise ValueError(f"dy: {dy.dtype}, whose range the rows of {x8.dtype} may pass")
    dy = _even(dy)
    rows, N, dys = _rows(dy)
    K = x8.shape[2]
    dw, db = torch.empty((N, K), dtype=dy.dtype, device=dy.device), torch.empty(N, dtype=dy.dtype, device=dy.device)
    with _on_device(dy.device):
        n = _bytes("sfm_linear8_wgrad_workspace_bytes", rows, N, K, dy.device.index)
        ws = torch.empty(n, dtype=torch.uint8, device=dy.device)
        _l.check(_l.load().sfm_linear8_wgrad(_DT[dy.dtype], rows, N, K, dy.data_ptr(), dys, x8.data.data_ptr(), x8.scale.data_ptr(),
                                             dw.data_ptr(), db.data_ptr(), None, ws.data_ptr(), n, _stream(dy)))
    return dw, db


def _even(dy):
    """Gradients come in any layout (expanded from a sum, transposed): rows of contiguous channels, evenly strided."""
    s = _row_stride(dy)
    return dy if s is not None and s >= dy.shape[2] else dy.clone(memory_format=torch.contiguous_format)


class _Linear8Fn(torch.autograd.Function):
    """Keeps the input in 8 bits (1 byte a value and the scales), and the transposed 8-bit weight for the input's gradient."""

    @staticmethod
    def forward(ctx, x, weight, bias, x8, w8):
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        if w8 is None:
            w8 = pack(weight, transposed=need_x)
        if need_x and w8.data_t is None:
            raise ValueError("the weight was packed without its transposed form, which the input's gradient needs")
        rows = x if x8 is None else x8
        N = w8.shape[0]
        out = torch.empty((*rows.shape[:2], N), dtype=rows.dtype, device=rows.device)
        if x8 is None:
            data, scale = _forward(x, w8, bias, out, need_w)
        else:
            data, scale = x8.data, x8.scale
            _product(x8, w8.data, w8.scale, N, bias, out)
        n = rows.shape[0] * rows.shape[1]
        ctx.cfg = (rows.shape, rows.dtype, w8.shape, n, _bytes("sfm_linear8_bwd_workspace_bytes", n, N, rows.shape[2], rows.device.index))
        _noted(ctx, rows.device)
        _save(ctx, *((data, scale) if need_w else (None, None)), *((w8.data_t, w8.scale_t) if need_x else (None, None)))
        return out

    @staticmethod
    @_once
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        x_shape, dtype, w_shape, rows, nbytes = ctx.cfg
        xd, xs, wd, ws = (t if t is None else t.contiguous() for t in _saved(ctx, dy))
        N, K = w_shape
        dys = N
        if not dy.is_contiguous():
            dy = _even(dy)
            dys = _row_stride(dy)
        dx = dy.new_empty(x_shape) if need_x else None
        dw = dy.new_empty(w_shape) if need_w else None
        db = dy.new_empty(N) if need_b else None
        work = dy.new_empty(nbytes, dtype=torch.uint8)
        rc = _l.load().sfm_linear8_bwd(_DT[dtype], rows, N, K, dy.data_ptr(), dys, _ptr(wd), _ptr(ws), _ptr(xd), _ptr(xs), _ptr(dx), _ptr(dw), _ptr(db),
                                       work.data_ptr(), nbytes, _raw_stream(dy.get_device()))
        if rc:
            _l.check(rc)
        return dx, dw, db, None, None


def linear8(x, weight, bias=None, epilogue="none", res=None, gate=None, out=None):
    """x [B, L, K] (bf16 or fp16; quantised in the call) or Rows8, weight Weight8 or [N, K] tensor (packed in the call), bias [N] or
    None -> [B, L, N].  epilogue "none": x w^T + bias; "gelu_tanh": GELU (tanh form) of that; "gate_residual": res + (that) * gate with gate
    a per-frame modulation tensor [B, F, 1, N] (None: res + that), written to `out` (default: in place into res).  All of it on the
    fp32 sum, rounded once.
    Differentiable (epilogue "none") in x, in a weight given as a tensor, and in bias."""
    if epilogue not in _EPI:
        raise ValueError(f"unknown epilogue {epilogue!r}")
    x8 = x if isinstance(x, Rows8) else None
    w8 = weight if isinstance(weight, Weight8) else None
    dtype = x.dtype
    if dtype not in _HALF:
        raise ValueError("linear8 takes float16 / bfloat16 tensors")
    if x8 is None:
        _rows(x)
    if w8 is None:
        if weight.dim() != 2:
            raise ValueError("weight must be [N, K]")
        if weight.dtype != dtype:
            raise ValueError(f"weight: {weight.dtype}, expected {dtype} like the activations")
    if weight.device != x.device:
        raise ValueError(f"weight on {weight.device}, expected {x.device} like the activations")
    B, L, K = x.shape
    N = weight.shape[0]
    if weight.shape[1] != K:
        raise ValueError("weight must be [N, K]")
    if bias is not None:
        _like("bias", bias, x)
        if bias.shape != (N,):
            raise ValueError("bias must be [N]")
        bias = bias.contiguous()
    if torch.is_grad_enabled() and ((x8 is None and x.requires_grad) or (w8 is None and weight.requires_grad)
                                    or any(t is not None and t.requires_grad for t in (bias, res, gate))):
        if epilogue != "none" or out is not None:
            raise NotImplementedError("linear8 is differentiable with epilogue 'none' and its own output")
        if res is not None or gate is not None:
            raise ValueError("res / gate belong to the gate_residual epilogue")
        return _Linear8Fn.apply(None if x8 is not None else x, None if w8 is not None else weight, bias, x8, w8)
    if epilogue == "gate_residual":
        if res is None:
            raise ValueError("the gated-residual epilogue needs res")
        _like("res", res, x)
        if res.shape != (B, L, N):
            raise ValueError("res must be [B, L, N]")
        out = res if out is None else out
    elif res is not None or gate is not None:
        raise ValueError("res / gate belong to the gate_residual epilogue")
    if out is None:
        out = torch.empty((B, L, N), dtype=dtype, device=x.device)
    else:
        _like("out", out, x)
        if out.shape != (B, L, N):
            raise ValueError("out must be [B, L, N]")
        _rows(out)
        _written(out)
    if w8 is None:
        w8 = pack(weight, transposed=False)
    if x8 is None:
        _forward(x, w8, bias, out, False, _EPI[epilogue], res, gate)
    else:
        _product(x8, w8.data, w8.scale, N, bias, out, _EPI[epilogue], res, gate)
    return out
