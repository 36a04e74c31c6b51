"""Serving many requests from one paged key-value cache: attention of a chunk of new tokens (or of single tokens) per request over
its pages of a shared pool, as attention.full_attention_with_kv_cache does for one contiguous cache per batch.  No counterpart
in the reference, which serves one video at a time.

    k_pages, v_pages = torch.empty(pages, page_size, kv_heads, head_dim, ...)       # the pool, twice
    plan = plan_pages(table, past, new, free, tokens, page_size)                    # once per step, for all layers
    write_pages(k, v, k_pages, v_pages, plan)                                       # per layer
    x = paged_attention(q, k_pages, v_pages, plan, causal=True)

A request r has past[r] tokens in the cache and new[r] in the step; token i of those has position past[r] + i.  Row r of the block table
names the page of each page_size consecutive positions.  Tensors over new tokens ([tokens, heads, head_dim]) hold the requests
one after the other; rows behind the last one, if the program pads its steps to a fixed size, belong to nobody.

For long caches: write_pages keeps the pages' mean keys, select_pages takes for each group of tokens the pages whose mean key
scores highest, and paged_attention reads only those (`selected=`).

Lengths, tables and lists of free pages stay on the GPU: nothing here waits for it, and a step can be recorded into a HIP graph.  What
they hold cannot be refused, then: no number in them makes a kernel leave its tensors, and each function says what comes of
numbers that make no sense.  Nothing here is differentiable,
in either mode."""
import ctypes as C
import functools
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import lib as _l
from .block_ops import _written
from .monarch_attn import _DT, _KEPT, _drop_kept, _on_device, _raw_stream


class PagePlan(NamedTuple):
    """A step of requests.  table int32 [requests, width], past and lengths int32 [requests] (tokens in the cache before and after the
    step), q_start int32 [requests + 1] (first row of each request), slots int64 [tokens] (row of the pools, page * page_size + offset,
    of each new token; -1 for none), next_free int32 [1] (how far the list of free pages is used; above its length where it did not
    suffice).  table and past are the caller's tensors: they stay as they are until the step's calls are done."""
    table: torch.Tensor
    past: torch.Tensor
    lengths: torch.Tensor
    q_start: torch.Tensor
    slots: torch.Tensor
    next_free: torch.Tensor
    page_size: int


def _ints(name, t, device, n=None, dtype=torch.int32):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 1 or t.device != device:
        raise ValueError(f"{name}: expected a one-dimensional {dtype} tensor on {device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name}: {t.shape[0]} values, expected {n}")
    return t if t.stride(0) == 1 or t.shape[0] < 2 else t.contiguous()


def _table(layout):
    """(rows, columns, row stride) of a block table's (dtype, shape, strides)."""
    dt, shape, stride = layout
    if dt != torch.int32 or len(shape) != 2:
        raise ValueError("table must be an int32 [requests, width] tensor")
    R, W = shape
    if R < 1 or W < 1:
        raise ValueError("table is empty")
    if W > 1 and stride[1] != 1:
        raise ValueError("table: a request's entries must be contiguous")
    return R, W, stride[0] if R > 1 else W


@functools.lru_cache(maxsize=1024)
def _plan_bytes(requests):
    n = C.c_size_t(0)
    _l.check(_l.load().sfm_paged_plan_workspace_bytes(requests, C.byref(n)))
    return n.value


def plan_pages(table, past, new, free, tokens, page_size, next_free=None):
    """Block table, slots and row offsets of a step, on the GPU in one launch (two for more than 8192 requests).

    table int32 [requests, width], whose entries for the tokens before the step are read and whose entries for the pages that the new tokens
    open are written in place; past, new int32 [requests]; free int32 list of free pages, taken from the front, or from
    next_free [1] on, an earlier plan's; tokens: rows of the step's tensors, at least the sum of `new`; page_size a multiple of 8.
    -> PagePlan.

    Where the list runs out, or a request outgrows its row of the table, the tokens without a page get slot -1 (and the
    table's entries -1): write_pages passes them over and paged_attention gives NaN for rows that would read them.  Requests past `tokens`
    rows have as many tokens as fit.  Negative lengths count as 0."""
    if not isinstance(table, torch.Tensor):
        raise ValueError("table must be an int32 [requests, width] tensor")
    R, W, ts = _table(_layout(table))
    dev = table.device
    _together(dev)
    past, new, free = _ints("past", past, dev, R), _ints("new", new, dev, R), _ints("free", free, dev)
    if next_free is not None:
        next_free = _ints("next_free", next_free, dev, 1)
    tokens, page_size = int(tokens), int(page_size)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    if not 8 <= page_size <= _MOST:
        raise ValueError(f"page_size: {page_size}, expected a multiple of 8")
    slots = torch.empty(tokens, dtype=torch.int64, device=dev)
    q_start, lengths, taken = torch.empty(2 * R + 2, dtype=torch.int32, device=dev).split_with_sizes((R + 1, R, 1))
    nbytes = _plan_bytes(R)
    with _on_device(dev):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = _l.load().sfm_paged_plan(R, W, page_size, tokens, table.data_ptr(), ts, past.data_ptr(), new.data_ptr(), free.data_ptr(), free.shape[0],
                                      None if next_free is None else next_free.data_ptr(), q_start.data_ptr(), lengths.data_ptr(),
                                      slots.data_ptr(), taken.data_ptr(), None if ws is None else ws.data_ptr(), nbytes, _raw_stream(dev.index))
    if rc:
        _l.check(rc)
    _written(table)
    return PagePlan(table, past, lengths, q_start, slots, taken, page_size)


# What follows from the tensors' shapes, strides and types (their checks, the descriptor, workspace sizes) is worked out once for each set of
# them: a single token's call is shorter than these steps.  A layout is (dtype, shape, strides); the stride of a dimension of one says
# nothing.

def _rows(name, layout, dtype):
    """(token stride, head stride) of [tokens, heads, head_dim] rows."""
    dt, shape, stride = layout
    if len(shape) != 3:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] tensor")
    if dt != dtype:
        raise ValueError(f"{name}: {dt}, expected {dtype} like the pools")
    T, H, D = shape
    if D > 1 and stride[2] != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    hs = stride[1] if H > 1 else D
    return stride[0] if T > 1 else H * hs, hs


def _pool(name, layout):
    """(page stride, token stride, head stride) of a [pages, page_size, kv_heads, head_dim] pool."""
    dt, shape, stride = layout
    if len(shape) != 4:
        raise ValueError(f"{name} must be a [pages, page_size, kv_heads, head_dim] tensor")
    if dt not in _DT:
        raise ValueError(f"unsupported dtype {dt}")
    N, P, H, D = shape
    if D > 1 and stride[3] != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    hs = stride[2] if H > 1 else D
    ts = stride[1] if P > 1 else H * hs
    return stride[0] if N > 1 else max(P * ts, P * D), ts, hs


def _pools(k_pages, v_pages, page_size):
    ps = _pool("k_pages", k_pages)
    if v_pages[:2] != k_pages[:2]:
        raise ValueError("k_pages and v_pages must agree in shape and dtype")
    if _pool("v_pages", v_pages) != ps:
        raise ValueError("k_pages and v_pages must share strides")
    if k_pages[1][1] != page_size:
        raise ValueError(f"the pools' pages have {k_pages[1][1]} rows, the plan's {page_size}")
    return ps


def _planned(plan, tokens):
    """(requests, width, table stride) of a plan's layout for tensors of so many rows."""
    table, past, q_start, slots = plan
    R, W, ts = _table(table)
    for name, (dt, shape, stride), n, want in (("past", past, R, torch.int32), ("q_start", q_start, R + 1, torch.int32), ("slots", slots, tokens, torch.int64)):
        if dt != want or tuple(shape) != (n,) or (n > 1 and stride[0] != 1):
            raise ValueError(f"the plan's {name} must be {n} contiguous {want}")
    return R, W, ts


def _layout(t):
    return t.dtype, t.shape, t.stride()


def _plan_layout(plan):
    if not isinstance(plan, PagePlan):
        raise ValueError("plan must be a PagePlan (plan_pages)")
    return _layout(plan.table), _layout(plan.past), _layout(plan.q_start), _layout(plan.slots)


def _together(device, *tensors):
    """All on one GPU.  (The calls of every layer compare numbers of devices first, a third of a microsecond for all, and come here where one differs.)"""
    if device.type != "cuda":
        raise ValueError("the paged cache lives on the GPU")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {t.device} and {device}")


def _gpu(plan):
    """The device number of a plan's tensors that a call reads, -1 where they differ."""
    gpu = plan.table.get_device()
    return gpu if gpu == plan.past.get_device() == plan.q_start.get_device() == plan.slots.get_device() else -1


def _tangents(*tensors):
    """Whether a tensor carries a tangent of forward-mode differentiation.  (Outside of its levels, as here all but always, none does.)"""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


_I2 = C.c_int64 * 2
_MOST = 2 ** 31 - 1            # a window, sink or group past it is one of everything: there are fewer positions and tokens


@functools.lru_cache(maxsize=4096)
def _write_call(k, v, k_pages, v_pages, page_size, plan, means):
    """(descriptor, strides of k and v or None where they need a layout in common)."""
    ps = _pools(k_pages, v_pages, page_size)
    N, P, H, D = k_pages[1]
    ks = _rows("k", k, k_pages[0])
    if tuple(k[1][1:]) != (H, D):
        raise ValueError("k must be [tokens, kv_heads, head_dim] of the pools' heads")
    if v[1] != k[1]:
        raise ValueError("k and v must have the same shape")
    same = _rows("v", v, k_pages[0]) == ks or 0 in k[1]         # nothing to write has every layout, and contiguous() leaves it as it is
    R, W, ts = _planned(plan, k[1][0])
    if means is not None and (means[0] != torch.float32 or tuple(means[1]) != (N, H, D) or tuple(means[2]) != (H * D, D, 1)):
        raise ValueError("means must be a contiguous float32 [pages, kv_heads, head_dim] tensor beside the pools")
    return _l.PagedDesc(_DT[k[0]], H, H, D, k[1][0], R, W, N, P, ts, ps), _I2(*ks) if same else None


def write_pages(k, v, k_pages, v_pages, plan, means=None):
    """k_pages / v_pages[slot] = k / v rows ([tokens, kv_heads, head_dim]), in place at the plan's slots; rows without one are passed over.  Any
    strides of whole 16 bytes with a contiguous head_dim, pools alike.  With means (fp32 [pages, kv_heads, head_dim], in place): the mean key of every page that got a
    row, over the page's rows up to the request's length.  k and v must not lie in the pools (refused); where a slot is named twice one of
    the rows stays in each 16 bytes."""
    if (torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad or (
            means is not None and means.requires_grad))) or _tangents(k, v, k_pages, v_pages, means):
        raise NotImplementedError("write_pages is not differentiable")
    dev, planned, gpu = k_pages.device, _plan_layout(plan), k_pages.get_device()
    if gpu < 0 or not (gpu == k.get_device() == v.get_device() == v_pages.get_device() == _gpu(plan)) or (means is not None and means.get_device() != gpu):
        _together(dev, k, v, v_pages, means, *plan[:5])
    desc, ks = _write_call(_layout(k), _layout(v), _layout(k_pages), _layout(v_pages), plan.page_size, planned, None if means is None else _layout(means))
    if ks is None:
        return write_pages(k.contiguous(), v.contiguous(), k_pages, v_pages, plan, means)
    if k.shape[0] == 0:
        return
    if _KEPT:
        _drop_kept(dev.index)
    with _on_device(dev):
        rc = _l.load().sfm_paged_write(desc, k.data_ptr(), v.data_ptr(), ks, k_pages.data_ptr(), v_pages.data_ptr(), plan.slots.data_ptr(),
                                       plan.table.data_ptr(), plan.past.data_ptr(), plan.q_start.data_ptr(),
                                       None if means is None else means.data_ptr(), _raw_stream(dev.index))
    if rc:
        _l.check(rc)
    increment_version([t for t in ((k_pages, v_pages) if means is None else (k_pages, v_pages, means)) if not t.is_inference()])


def selected_rows(tokens, requests, group):
    """Rows of the lists that select_pages gives."""
    return tokens // group + requests + 1


@functools.lru_cache(maxsize=4096)
def _attention_call(device, q, k_pages, v_pages, page_size, plan, out, selected, sm_scale, causal, window, sink, group):
    """(descriptor, workspace bytes on the device, whose compute units are in the size)."""
    ps = _pools(k_pages, v_pages, page_size)
    N, P, Hk, D = k_pages[1]
    qs = _rows("q", q, k_pages[0])
    T, H, qd = q[1]
    if qd != D or H < Hk or H % Hk:
        raise ValueError("q must be [tokens, heads, head_dim], heads a multiple of the pools' and head_dim theirs")
    if window is not None and window < 1:
        raise ValueError("window must be a position or more (None: all)")
    if sink < 0 or (sink and window is None):
        raise ValueError("sink: positions that stay visible outside a window")
    R, W, ts = _planned(plan, T)
    top = 0
    if selected is not None:
        if window is not None:
            raise ValueError("selected pages and a window do not go together")
        if group < 1:
            raise ValueError("group must be a token or more")
        rows, (dt, shape, stride) = selected_rows(T, R, group), selected
        top = shape[2] if len(shape) == 3 else 0
        if dt != torch.int32 or top < 1 or tuple(shape[:2]) != (rows, Hk) or tuple(stride) != (Hk * top, top, 1):
            raise ValueError(f"selected must be a contiguous int32 [{rows}, {Hk}, top] tensor")
    if out is not None and tuple(out[1]) != tuple(q[1]):
        raise ValueError("out must be like q")
    os = (H * D, D) if out is None else _rows("out", out, q[0])
    desc = _l.PagedDesc(_DT[q[0]], H, Hk, D, T, R, W, N, P, ts, ps, qs, os, D ** -0.5 if sm_scale is None else sm_scale, causal, window or 0, sink,
                        top, group, out is None)
    n = C.c_size_t(0)
    if T:
        with torch.cuda.device(device):
            _l.check(_l.load().sfm_paged_workspace_bytes(desc, C.byref(n)))
    return desc, n.value


def paged_attention(q, k_pages, v_pages, plan, sm_scale=None, causal=False, window=None, sink=0, selected=None, group=1, out=None,
                    return_lse=False):
    """softmax(sm_scale q K^T) V of every new token over the positions of its request in the cache, its own step's among them
    (write_pages comes first).

    q [tokens, heads, head_dim], heads a multiple of the pools' kv_heads: query heads h * heads / kv_heads and on read key head h.  causal: a
    token's positions end at its own; else at the request's last, as a chunk of latent frames sees all of itself.  window: of those
    positions only the last `window`, and the first `sink` of the request.  selected, group: only the pages that select_pages lists
    for each `group` tokens (int32 [selected_rows(tokens, requests, group), kv_heads, top], ascending, each page once; no window then).

    -> [tokens, heads, head_dim] in q's dtype, zeros for a token that sees nothing and for rows that nobody has (with out, rows that nobody
    has stay as they were; out in q, the pools or the plan is refused); with return_lse also the natural logarithm of the sums, fp32
    [heads, tokens], -inf for nothing.  Rows that would read a position without a page (-1 or another number outside the pool,
    positions past the table) are NaN, and others of their request may be.  What lies in positions that a row does not see has no part in it,
    NaN or infinite; an infinity in a channel of V that it does see makes that channel infinite, or NaN if its weight is too small for the type.

    Sums and softmax statistics are fp32; 16-bit tensors with head sizes 64 and 128 take the weights rounded to their type into the product
    with V, as attention.attention does (off 64 bits by 1.2 to 1.4 times as much as a result that is only rounded itself).

    Which kernel a call takes, and into how many ranges its keys are cut, follows what the host knows: rows and requests on average, and the table's
    width.  table[:, :n] of the columns in use, few rows of nobody, few waiting requests, and prompts and single tokens in calls of their own cost less
    time; results do not depend on it but for the order of sums."""
    if (torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or (
            out is not None and out.requires_grad))) or _tangents(q, k_pages, v_pages, out):
        raise NotImplementedError("paged_attention is not differentiable")
    dev, planned, gpu = k_pages.device, _plan_layout(plan), k_pages.get_device()
    if gpu < 0 or not (gpu == q.get_device() == v_pages.get_device() == _gpu(plan)) or (selected is not None and selected.get_device() != gpu) or (
            out is not None and out.get_device() != gpu):
        _together(dev, q, v_pages, selected, out, *plan[:5])
    desc, nbytes = _attention_call(dev, _layout(q), _layout(k_pages), _layout(v_pages), plan.page_size, planned, None if out is None else _layout(out),
                                   None if selected is None else _layout(selected), None if sm_scale is None else float(sm_scale), bool(causal),
                                   None if window is None else min(int(window), _MOST), min(int(sink), _MOST),
                                   min(int(group), _MOST))
    T, H, _ = q.shape
    mine = out is None
    if mine:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = None
    if return_lse:             # rows of nobody that are left as they were have none
        lse = torch.empty((H, T), dtype=torch.float32, device=dev) if mine else torch.full((H, T), -math.inf, dtype=torch.float32, device=dev)
    if T:
        with _on_device(dev):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
            rc = _l.load().sfm_paged_attention(desc, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(),
                                               plan.q_start.data_ptr(), None if selected is None else selected.data_ptr(), out.data_ptr(),
                                               None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
                                               _raw_stream(dev.index))
        if rc:
            _l.check(rc)
        if not mine:
            _written(out)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=4096)
def _select_call(device, q, means, plan, page_size, top, group, causal, first, last):
    """(descriptor, rows of the lists, workspace bytes)."""
    if q[0] not in _DT:
        raise ValueError("q must be a [tokens, heads, head_dim] tensor of bf16, fp16 or fp32")
    qs = _rows("q", q, q[0])
    T, H, D = q[1]
    if means[0] != torch.float32 or len(means[1]) != 3 or means[1][2] != D or tuple(means[2]) != (means[1][1] * D, D, 1):
        raise ValueError("means must be a contiguous float32 [pages, kv_heads, head_dim] tensor")
    N, Hk, _ = means[1]
    if Hk < 1 or H < Hk or H % Hk:
        raise ValueError("q's heads must be a multiple of the means'")
    if group < 1 or not 1 <= top <= _l.PAGED_TOP_MAX:
        raise ValueError(f"group must be a token or more, top 1 to {_l.PAGED_TOP_MAX} pages")
    if first < 0 or last < 0 or first + last > top:
        raise ValueError("first and last must not be negative, nor more than top together")
    R, W, ts = _planned(plan, T)
    desc = _l.PagedDesc(_DT[q[0]], H, Hk, D, T, R, W, N, page_size, ts, (0, 0, 0), qs, (0, 0), 1.0, causal, 0, 0, top, group, 0)
    n = C.c_size_t(0)
    if T:
        with torch.cuda.device(device):
            _l.check(_l.load().sfm_paged_select_workspace_bytes(desc, C.byref(n)))
    return desc, selected_rows(T, R, group), n.value


def select_pages(q, means, plan, top, group=1, causal=False, first=1, last=1):
    """Which pages each `group` consecutive new tokens of a request read, for paged_attention's `selected`: int32
    [selected_rows(tokens, requests, group), kv_heads, top] entries of the request's row of the table, ascending, -1 behind them.

    Candidates are the pages up to the last one that the group's last token sees (causal: its own).  The first `first` and the last `last` of
    them are taken, and then those with the largest (sum of q over the group's tokens and the key head's query heads) . mean key, up
    to `top` in all; of level ones the lower.  A group's tokens share that choice, the earlier ones with what the later ones ask for, and where a group
    crosses a page the forced last page is not every token's own: last = (group + page_size - 2) // page_size + 1 forces all of those; with
    less a token of a causal group may find none of its pages taken, and gets zeros.  means: fp32 [pages, kv_heads, head_dim], kept by write_pages.  Scores are sums in 64 bits,
    so that which page is ahead does not hang on the order of an addition; NaN counts as -inf, as does a page outside the pool.  Group i of request r
    is row q_start[r] // group + r + i; rows that nobody has are -1."""
    if (torch.is_grad_enabled() and (q.requires_grad or means.requires_grad)) or _tangents(q, means):
        raise NotImplementedError("select_pages is not differentiable")
    dev, planned, gpu = q.device, _plan_layout(plan), q.get_device()
    if gpu < 0 or not (gpu == means.get_device() == _gpu(plan)):
        _together(dev, means, *plan[:5])
    top, first, last = int(top), int(first), int(last)
    desc, rows, nbytes = _select_call(dev, _layout(q), _layout(means), planned, plan.page_size, top, min(int(group), _MOST), bool(causal), first, last)
    selected = torch.empty((rows, means.shape[1], top), dtype=torch.int32, device=dev)
    if q.shape[0] == 0:
        return selected.fill_(-1)
    with _on_device(dev):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = _l.load().sfm_paged_select(desc, q.data_ptr(), means.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(), plan.q_start.data_ptr(), first,
                                        last, selected.data_ptr(), ws.data_ptr(), nbytes, _raw_stream(dev.index))
    if rc:
        _l.check(rc)
    return selected
