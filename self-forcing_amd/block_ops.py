"""Fused element-wise operators of the causal Wan block (LayerNorm + adaLN modulation, gated residual,
RMSNorm, GELU); counterparts of the eager chains in wan/modules/causal_model.py:1176-1205 and
wan/modules/model.py:462-478.  [B, L, C] tensors, modulation rows [B, F, 1, C] (one per latent frame)."""
import ctypes
import functools
import threading
import weakref

import torch

from . import lib as _l
from .monarch_attn import _DT, _on_device, _raw_stream, _stream

_HALF = (torch.float16, torch.bfloat16)


def _row_stride(x):
    """Elements between the rows of a [B, L, C] tensor with contiguous channels; None where they are not evenly strided.  The
    stride of a dimension of one says nothing."""
    if x.dim() != 3 or (x.stride(2) != 1 and x.shape[2] > 1):
        return None
    B, L, C = x.shape
    if B == 1 or L == 1:
        return x.stride(1) if L > 1 else x.stride(0) if B > 1 else C
    return x.stride(1) if x.stride(0) == L * x.stride(1) else None


def _rows(x):
    if not x.is_cuda:
        raise ValueError("the block operators run on the GPU")
    if x.dtype not in _DT:
        raise ValueError(f"unsupported dtype {x.dtype}")
    xs = _row_stride(x)
    if xs is None:
        raise ValueError("expected a [B, L, C] tensor with contiguous channels and evenly strided rows")
    return x.shape[0] * x.shape[1], x.shape[2], xs


def _like(name, t, x):
    """The kernels read every operand in x's dtype: another dtype (or device) would be misread, not converted."""
    if t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, expected {x.dtype} on {x.device} like the activations")
    return t


def _vec(name, t, x):
    _like(name, t, x)
    if t.dim() != 1 or t.shape[0] != x.shape[2]:
        raise ValueError(f"{name}: expected a [C] vector")
    return t.contiguous()


def _mod(e, x):
    """[B, F, 1, C] (or [B, F, C]) modulation tensor -> (tensor, frame stride, rows per frame)."""
    B, L, C = x.shape
    _like("modulation", e, x)
    if e.numel() == 0 or x.numel() == 0 or e.numel() % (B * C):
        raise ValueError("modulation: expected [B, F, 1, C] rows")
    e = e.reshape(B, -1, C)
    if e.stride(2) != 1 or (B > 1 and e.stride(0) != e.shape[1] * e.stride(1)):
        e = e.contiguous()
    if L % e.shape[1]:
        raise ValueError("token count is not a multiple of the number of modulation frames")
    return e, e.stride(1), L // e.shape[1]


def _pairs(scale, shift, x):
    """The two modulation tensors as (tensor, tensor, frame stride, rows per frame); they share their frames."""
    sc, ms, rpf = _mod(scale, x)
    sh, ms2, rpf2 = _mod(shift, x)
    if rpf2 != rpf:
        raise ValueError("scale and shift must have the same number of modulation frames")
    if ms2 != ms:
        sc, sh = sc.contiguous(), sh.contiguous()
        ms = sc.stride(1)
    return sc, sh, ms, rpf


def _needs_grad(*ts):
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


def _written(t):
    """A tensor written in place through its address: autograd is told, so that a graph that has saved it does not use it."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _even(dy):
    """Gradients come in any layout (expanded from a sum, transposed): rows of contiguous channels, evenly strided and 16-byte
    aligned."""
    s = _row_stride(dy)
    ok = s is not None and s >= dy.shape[2] and dy.data_ptr() % 16 == 0 and s * dy.element_size() % 16 == 0
    return dy if ok else dy.clone(memory_format=torch.contiguous_format)


def _ln(x, mod, eps):
    rows, C, xs = _rows(x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    with _on_device(x.device):
        _l.check(_l.load().sfm_ln_modulate(_DT[x.dtype], rows, C, eps, x.data_ptr(), xs, y.data_ptr(), C, *mod, _stream(x)))
    return y


def _ln_keep8(x, mod, eps):
    """(y, normalised rows' 8-bit data, their scales, 1 / standard deviation of each row)."""
    rows, C, xs = _rows(x)
    kp = -(-C // 128) * 128
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    data = torch.empty((rows, kp), dtype=torch.uint8, device=x.device)
    scale = torch.empty(-(-rows // 128) * kp, dtype=torch.uint8, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    with _on_device(x.device):
        _l.check(_l.load().sfm_ln_keep8(_DT[x.dtype], rows, C, eps, x.data_ptr(), xs, y.data_ptr(), C, *mod, data.data_ptr(),
                                        scale.data_ptr(), rstd.data_ptr(), _stream(x)))
    return y, data, scale, rstd


@functools.lru_cache(maxsize=1024)
def _ln_bwd_bytes(rows, C, group, device_index):
    """Workspace of sfm_ln_bwd on a device (its compute units are in the size)."""
    n = ctypes.c_size_t(0)
    with torch.cuda.device(device_index):
        _l.check(_l.load().sfm_ln_bwd_workspace_bytes(rows, C, group, ctypes.byref(n)))
    return n.value


def _ln_bwd(dy, x, xs, kept, weight, scale, ms, group, nbytes, eps, w_shape, b_shape, want_dx=True):
    """(dx, dw, db): dw, db hold [groups of rows, C] in the given shapes.  From x, rows xs apart, or from `kept` = (data, scales,
    1 / standard deviations).  On the current device."""
    B, L, C = dy.shape
    dys = C
    if not dy.is_contiguous() or dy.data_ptr() & 15:
        dy = _even(dy)
        dys = _row_stride(dy)
    dx = torch.empty_like(dy, memory_format=torch.contiguous_format) if want_dx else None
    dw, db = dy.new_empty(w_shape), dy.new_empty(b_shape)
    data = sc8 = rstd = None
    if kept is not None:
        data, sc8, rstd = kept[0].data_ptr(), kept[1].data_ptr(), kept[2].data_ptr()
    ws = dy.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = _l.load().sfm_ln_bwd(_DT[dy.dtype], B * L, C, eps, None if x is None else x.data_ptr(), xs, data, sc8, rstd, dy.data_ptr(), dys,
                              None if weight is None else weight.data_ptr(), None if scale is None else scale.data_ptr(), ms, group,
                              dx.data_ptr() if want_dx else None, C, dw.data_ptr(), db.data_ptr(), ws.data_ptr() if nbytes else None, nbytes,
                              _raw_stream(dy.get_device()))
    if rc:
        _l.check(rc)
    return dx, dw, db


_eager_graphs, _eager_lock, _eager_limit = [], threading.Lock(), 1024


def _noted(ctx, device):
    """Called by the forwards: remembers a graph recorded on the default stream while it lives."""
    global _eager_limit
    if _raw_stream(device.index) == 0:
        with _eager_lock:
            _eager_graphs.append(weakref.ref(ctx))
            if len(_eager_graphs) > _eager_limit:              # most of them are gone
                _eager_graphs[:] = [r for r in _eager_graphs if r() is not None]
                _eager_limit = max(1024, 2 * len(_eager_graphs))


def _leaves(*nodes):
    """The leaves, by identity, that the gradients of these nodes go to, directly or through other operators."""
    seen, leaves, todo = set(), {}, list(nodes)
    while todo:
        node = todo.pop()
        if type(node).__name__ == "AccumulateGrad":
            leaves[id(node.variable)] = node.variable
        elif node is not None and node not in seen:
            seen.add(node)
            todo.extend(n for n, _ in node.next_functions)
    return leaves


def _check_captured(ctx):
    """Autograd sums a leaf's gradient on the stream that its oldest living graph was recorded on.  A captured backward whose leaf
    belongs to a living graph of the default stream would make that stream part of the capture, which HIP does not allow and which
    ends the process: refused before anything reaches the leaf.  Graphs are known by the operators of this module and of linear8 in
    them."""
    if not torch.cuda.is_current_stream_capturing():
        return
    with _eager_lock:
        others = [r() for r in _eager_graphs]
    others = [o for o in others if o is not None and o is not ctx]
    if others and _leaves(ctx).keys() & _leaves(*others).keys():
        raise RuntimeError("a backward cannot be captured while a graph of the same leaves, recorded on the default stream, lives: drop "
                           "its outputs first, or record it on another stream")


def _save(ctx, *tensors):
    """`save_for_backward`, and what `_saved` holds the tensors against."""
    ctx.save_for_backward(*tensors)
    ctx.saved_as = [None if t is None else (t.shape, t.dtype) for t in tensors]


def _saved(ctx, dy):
    """The saved tensors.  Saved-tensor hooks (save_on_cpu) may give them back in another layout, which the caller sees to; the kernels
    take addresses, so that another size, type or device is refused here."""
    saved, device = ctx.saved_tensors, dy.device
    for t, was in zip(saved, ctx.saved_as):
        if was is not None and (t.shape != was[0] or t.dtype != was[1] or t.device != device):
            raise RuntimeError(f"saved-tensor hooks gave back {tuple(t.shape)} {t.dtype} on {t.device} for {tuple(was[0])} {was[1]} on {device}")
    return saved


def _once(backward):
    """A backward without a derivative of its own: `once_differentiable`, but for calls that build no graph, which it would only
    slow down.

    The backwards themselves are short on purpose: autograd's thread, whose current device is the node's, runs them on another core, and every
    Python object that they touch comes over from the caller's (LayerNorm of three rows, forward and backward: 94 us a call, 41 with
    both threads on one core, 110 and 47 with checks, sizes and device contexts in the backward)."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, dy):
        if _raw_stream(dy.get_device()):                       # the default stream is never captured
            _check_captured(ctx)
        return (guarded if torch.is_grad_enabled() else backward)(ctx, dy)
    return run


class _LnFn(torch.autograd.Function):
    """LayerNorm with `a`, `b` = weight, bias ([C]) or scale, shift (per frame).  Keeps x, or with `checkpoint8` the normalised rows
    in 8 bits and a float per row."""

    @staticmethod
    def forward(ctx, x, a, b, modulate, eps, checkpoint8):
        if modulate:
            sc, sh, ms, rpf = _pairs(a, b, x)
            mod = (sc.data_ptr(), sh.data_ptr(), ms, rpf, None, None)
        else:
            sc, sh, ms, rpf = _vec("weight", a, x), _vec("bias", b, x), 0, x.shape[0] * x.shape[1]
            mod = (None, None, 0, 1, sc.data_ptr(), sh.data_ptr())
        if checkpoint8:
            y, *kept = _ln_keep8(x, mod, eps)
            _save(ctx, sc, *kept)
        else:
            y = _ln(x, mod, eps)
            _save(ctx, sc, x)
        ctx.cfg = (modulate, eps, checkpoint8, ms, rpf, _row_stride(x), _ln_bwd_bytes(x.shape[0] * x.shape[1], x.shape[2], rpf, x.get_device()),
                   a.shape, b.shape, sc.stride(), x.stride())
        _noted(ctx, x.device)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        modulate, eps, checkpoint8, ms, rpf, xs, nbytes, a_shape, b_shape, sc_strides, x_strides = ctx.cfg
        sc, *rest = _saved(ctx, dy)
        x, kept = (None, [t.contiguous() for t in rest]) if checkpoint8 else (rest[0], None)
        if sc.stride() != sc_strides:
            sc, ms = sc.contiguous(), sc.shape[-1] if modulate else 0
        if x is not None and x.stride() != x_strides:
            x, xs = x.contiguous(), x.shape[2]
        dx, dw, db = _ln_bwd(dy, x, xs, kept, None if modulate else sc, sc if modulate else None, ms, rpf, nbytes, eps, a_shape, b_shape,
                             ctx.needs_input_grad[0])
        return dx, dw, db, None, None, None


def ln_modulate(x, scale, shift, eps=1e-6, checkpoint8=False):
    """LayerNorm(x) (no affine) * (1 + scale) + shift with per-frame scale/shift.  Differentiable in all three; with `checkpoint8`
    the normalised rows are kept for the backward in 8-bit blocks (see linear8) instead of x."""
    if _needs_grad(x, scale, shift):
        return _LnFn.apply(x, scale, shift, True, eps, checkpoint8)
    sc, sh, ms, rpf = _pairs(scale, shift, x)
    return _ln(x, (sc.data_ptr(), sh.data_ptr(), ms, rpf, None, None), eps)


def ln_affine(x, weight, bias, eps=1e-6, checkpoint8=False):
    """LayerNorm(x) * weight + bias.  Differentiable in all three; `checkpoint8` as in ln_modulate."""
    if _needs_grad(x, weight, bias):
        return _LnFn.apply(x, weight, bias, False, eps, checkpoint8)
    weight, bias = _vec("weight", weight, x), _vec("bias", bias, x)
    return _ln(x, (None, None, 0, 1, weight.data_ptr(), bias.data_ptr()), eps)


def _check_dy(dy, x):
    _like("dy", dy, x)
    if dy.shape != x.shape:
        raise ValueError("dy and x must have the same shape")


def ln_affine_backward(dy, x, weight, eps=1e-6):
    """(dx, dweight, dbias) of ln_affine from its output's gradient."""
    _check_dy(dy, x)
    rows, C, xs = _rows(x)
    with _on_device(x.device):
        n = _ln_bwd_bytes(rows, C, rows, x.get_device())
        return _ln_bwd(dy, x, xs, None, _vec("weight", weight, x), None, 0, rows, n, eps, weight.shape, weight.shape)


def ln_modulate_backward(dy, x, scale, eps=1e-6):
    """(dx, dscale, dshift) of ln_modulate from its output's gradient; dscale and dshift in scale's shape."""
    _check_dy(dy, x)
    sc, ms, rpf = _mod(scale, x)
    rows, C, xs = _rows(x)
    with _on_device(x.device):
        n = _ln_bwd_bytes(rows, C, rpf, x.get_device())
        return _ln_bwd(dy, x, xs, None, None, sc, ms, rpf, n, eps, scale.shape, scale.shape)


def _gelu(x, keep8):
    rows, C, xs = _rows(x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    data = scale = None
    if keep8:
        kp = -(-C // 128) * 128
        data = torch.empty((rows, kp), dtype=torch.uint8, device=x.device)
        scale = torch.empty(-(-rows // 128) * kp, dtype=torch.uint8, device=x.device)
    with _on_device(x.device):
        _l.check(_l.load().sfm_quantize8(_DT[x.dtype], rows, C, x.data_ptr(), xs, data.data_ptr() if keep8 else None,
                                         scale.data_ptr() if keep8 else None, y.data_ptr(), C, None, _stream(x)))
    return y, data, scale


class _GeluFn(torch.autograd.Function):
    """Keeps x, or with `checkpoint8` x in 8-bit blocks."""

    @staticmethod
    def forward(ctx, x, checkpoint8):
        y, data, scale = _gelu(x, checkpoint8)
        ctx.checkpoint8 = checkpoint8
        _noted(ctx, x.device)
        _save(ctx, *((data, scale) if checkpoint8 else (x,)))
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        B, L, C = dy.shape
        dys = C
        if not dy.is_contiguous():
            dy = _even(dy)
            dys = _row_stride(dy)
        x, xs, data, scale = None, 0, None, None
        saved = _saved(ctx, dy)                # held until the call: saved-tensor hooks give tensors that nobody else holds
        if ctx.checkpoint8:
            saved = [t.contiguous() for t in saved]
            data, scale = (t.data_ptr() for t in saved)
        else:
            x, = saved
            if _row_stride(x) is None:
                saved = x = x.contiguous()
            xs, x = _row_stride(x), x.data_ptr()
        dx = torch.empty_like(dy, memory_format=torch.contiguous_format)
        rc = _l.load().sfm_gelu_bwd(_DT[dy.dtype], B * L, C, x, xs, data, scale, dy.data_ptr(), dys, dx.data_ptr(), C, _raw_stream(dy.get_device()))
        if rc:
            _l.check(rc)
        return dx, None


def gelu_tanh(x, checkpoint8=False):
    """GELU in its tanh form (wan/modules/model.py:648-650) of [B, L, C] rows.  Differentiable; with `checkpoint8` x is kept for the
    backward in 8-bit blocks (see linear8)."""
    if _needs_grad(x):
        return _GeluFn.apply(x, checkpoint8)
    return _gelu(x, False)[0]


def gate_residual_(x, y, gate=None):
    """x += y * gate (per-frame gate) in place; gate=None: x += y."""
    rows, C, xs = _rows(x)
    _, _, ys = _rows(_like("y", y, x))
    if y.shape != x.shape:
        raise ValueError("x and y must have the same shape")
    g, ms, rpf = (None, 0, 1) if gate is None else _mod(gate, x)
    _written(x)
    with torch.cuda.device(x.device):
        _l.check(_l.load().sfm_gate_residual(_DT[x.dtype], rows, C, x.data_ptr(), xs, y.data_ptr(), ys,
                                             None if g is None else g.data_ptr(), ms, rpf, _stream(x)))
    return x


def gate_residual_ln_(x, y, gate=None, scale=None, shift=None, weight=None, bias=None, eps=1e-6):
    """x += y * gate in place (gate=None: x += y), then returns (x, LayerNorm(x) * (1 + scale) + shift), or the
    affine LayerNorm when weight / bias are given: one pass over the rows instead of two kernels."""
    rows, C, xs = _rows(x)
    _, _, ys = _rows(_like("y", y, x))
    if y.shape != x.shape:
        raise ValueError("x and y must have the same shape")
    g, gms, grpf = (None, 0, 1) if gate is None else _mod(gate, x)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if weight is None:
        sc, sh, ms, rpf = _pairs(scale, shift, x)
        mod = (sc.data_ptr(), sh.data_ptr(), ms, rpf, None, None)
    else:
        weight, bias = _vec("weight", weight, x), _vec("bias", bias, x)
        mod = (None, None, 0, 1, weight.data_ptr(), bias.data_ptr())
    _written(x)
    with torch.cuda.device(x.device):
        _l.check(_l.load().sfm_gate_residual_ln(_DT[x.dtype], rows, C, eps, x.data_ptr(), xs, y.data_ptr(), ys,
                                                None if g is None else g.data_ptr(), gms, grpf, out.data_ptr(), C, *mod,
                                                _stream(x)))
    return x, out


def rms_norm(x, weight, eps=1e-6):
    rows, C, xs = _rows(x)
    weight = _vec("weight", weight, x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    with torch.cuda.device(x.device):
        _l.check(_l.load().sfm_rms_norm(_DT[x.dtype], rows, C, eps, x.data_ptr(), xs, y.data_ptr(), C, weight.data_ptr(),
                                        _stream(x)))
    return y
