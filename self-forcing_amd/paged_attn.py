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
numbers that make no sense.  Nothing here is differentiable."""
import ctypes as C
import functools
import math
from typing import NamedTuple

import torch

from . import lib as _l
from .block_ops import _needs_grad, _written
from .monarch_attn import _DT, _KEPT, _drop_kept, _on_device, _raw_stream


class PagePlan(NamedTuple):
    """A step of requests.  table int32 [requests, width], past and lengths int32 [requests] (tokens in the cache before and after the
    step), q_start int32 [requests + 1] (first row of each request), slots int64 [tokens] (row of the pools, page * page_size + offset,
    of each new token; -1 for none), next_free int32 [1] (how far the list of free pages is used; above its length where it did not
    suffice)."""
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


def _table(t):
    """(rows, columns, row stride)"""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 2:
        raise ValueError("table must be an int32 [requests, width] tensor")
    if not t.is_cuda:
        raise ValueError("the paged cache lives on the GPU")
    R, W = t.shape
    if R < 1 or W < 1:
        raise ValueError("table is empty")
    if W > 1 and t.stride(1) != 1:
        raise ValueError("table: a request's entries must be contiguous")
    return R, W, t.stride(0) if R > 1 else W


@functools.lru_cache(maxsize=1024)
def _plan_bytes(requests):
    n = C.c_size_t(0)
    _l.check(_l.load().sfm_paged_plan_workspace_bytes(requests, C.byref(n)))
    return n.value


def plan_pages(table, past, new, free, tokens, page_size, next_free=None):
    """Block table, slots and row offsets of a step, on the GPU in one launch.

    table int32 [requests, width], whose entries for the tokens before the step are read and whose entries for the pages that the new tokens
    open are written in place; past, new int32 [requests]; free int32 list of free pages, taken from the front, or from
    next_free [1] on, an earlier plan's; tokens: rows of the step's tensors, at least the sum of `new`; page_size a multiple of 8.
    -> PagePlan.

    Where the list runs out, or a request outgrows its row of the table, the tokens without a page get slot -1 (and the
    table's entries -1): write_pages passes them over and paged_attention gives NaN for rows that would read them.  Requests past `tokens`
    rows have as many tokens as fit.  Negative lengths count as 0."""
    R, W, ts = _table(table)
    dev = table.device
    past, new, free = _ints("past", past, dev, R), _ints("new", new, dev, R), _ints("free", free, dev)
    if next_free is not None:
        next_free = _ints("next_free", next_free, dev, 1)
    tokens, page_size = int(tokens), int(page_size)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
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


def _rows(name, t, dtype, device):
    """[tokens, heads, head_dim] rows -> (token stride, head stride); the stride of a dimension of one says nothing."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] tensor")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, expected {dtype} on {device}")
    T, H, D = t.shape
    if D > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    hs = t.stride(1) if H > 1 else D
    return t.stride(0) if T > 1 else H * hs, hs


def _pools(k_pages, v_pages, page_size):
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{name} must be a [pages, page_size, kv_heads, head_dim] tensor")
        if not t.is_cuda:
            raise ValueError("the paged cache lives on the GPU")
    if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != k_pages.device:
        raise ValueError("k_pages and v_pages must agree in shape, dtype and device")
    if k_pages.dtype not in _DT:
        raise ValueError(f"unsupported dtype {k_pages.dtype}")
    if k_pages.shape[1] != page_size:
        raise ValueError(f"the pools' pages have {k_pages.shape[1]} rows, the plan's {page_size}")
    s = k_pages.stride()
    if s != v_pages.stride() or s[3] != 1 or 1 in k_pages.shape:           # a dimension of one may have any stride
        s = _pool_strides(k_pages)
        if s != _pool_strides(v_pages):
            raise ValueError("k_pages and v_pages must share strides")
    return s[:3]


def _pool_strides(t):
    N, P, H, D = t.shape
    if D > 1 and t.stride(3) != 1:
        raise ValueError("the pools' head_dim must be contiguous")
    hs = t.stride(2) if H > 1 else D
    ts = t.stride(1) if P > 1 else H * hs
    return t.stride(0) if N > 1 else max(P * ts, P * D), ts, hs


def _plan(plan, tokens, device):
    """(requests, width, table stride) of a plan for tensors of so many rows."""
    if not isinstance(plan, PagePlan):
        raise ValueError("plan must be a PagePlan (plan_pages)")
    R, W, ts = _table(plan.table)
    if plan.table.device != device:
        raise ValueError(f"the plan is on {plan.table.device}, the tensors on {device}")
    for name, t, n, dt in (("past", plan.past, R, torch.int32), ("q_start", plan.q_start, R + 1, torch.int32), ("slots", plan.slots, tokens, torch.int64)):
        if t.shape != (n,) or t.dtype != dt or t.device != device or not t.is_contiguous():
            raise ValueError(f"the plan's {name} must be {n} contiguous {dt} on {device}")
    return R, W, ts


def write_pages(k, v, k_pages, v_pages, plan, means=None):
    """k_pages / v_pages[slot] = k / v rows ([tokens, kv_heads, head_dim]), in place at the plan's slots; rows without one are passed over.  Any
    strides with a contiguous head_dim, pools alike.  With means (fp32 [pages, kv_heads, head_dim], in place): the mean key of every page that got a
    row, over the page's rows up to the request's length.  k and v must not lie in the pools; where a slot is named twice one of
    the rows stays in each 16 bytes."""
    if _needs_grad(k, v):
        raise NotImplementedError("write_pages is not differentiable")
    ps = _pools(k_pages, v_pages, getattr(plan, "page_size", None))
    N, P, H, D = k_pages.shape
    dev = k_pages.device
    ks = _rows("k", k, k_pages.dtype, dev)
    if k.shape[1:] != (H, D):
        raise ValueError("k must be [tokens, kv_heads, head_dim] of the pools' heads")
    if v.shape != k.shape or _rows("v", v, k.dtype, dev) != ks:
        if v.shape != k.shape:
            raise ValueError("k and v must have the same shape")
        k, v = k.contiguous(), v.contiguous()
        ks = _rows("k", k, k.dtype, dev)
    R, W, ts = _plan(plan, k.shape[0], dev)
    if means is not None and (means.dtype != torch.float32 or means.device != dev or means.shape != (N, H, D) or not means.is_contiguous()):
        raise ValueError("means must be a contiguous float32 [pages, kv_heads, head_dim] tensor beside the pools")
    if k.shape[0] == 0:
        return
    d = _l.PagedDesc(_DT[k.dtype], H, H, D, k.shape[0], R, W, N, P, ts, ps)
    if _KEPT:
        _drop_kept(dev.index)
    with _on_device(dev):
        _l.check(_l.load().sfm_paged_write(C.byref(d), k.data_ptr(), v.data_ptr(), (C.c_int64 * 2)(*ks), k_pages.data_ptr(), v_pages.data_ptr(),
                                           plan.slots.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(), plan.q_start.data_ptr(),
                                           None if means is None else means.data_ptr(), _raw_stream(dev.index)))
    _written(k_pages)
    _written(v_pages)
    if means is not None:
        _written(means)


def _q_desc(q, qs, kv_heads, plan, pages, pool, out, sm_scale, causal, window, sink, top, group, zero_rest):
    T, H, D = q.shape
    R, W, ts = _plan(plan, T, q.device)
    return _l.PagedDesc(_DT[q.dtype], H, kv_heads, D, T, R, W, pages, plan.page_size, ts, pool, qs, out, sm_scale, causal, window, sink, top, group,
                        zero_rest)


def selected_rows(tokens, requests, group):
    """Rows of the lists that select_pages gives."""
    return tokens // group + requests + 1


def paged_attention(q, k_pages, v_pages, plan, sm_scale=None, causal=False, window=None, sink=0, selected=None, group=1, out=None,
                    return_lse=False):
    """softmax(sm_scale q K^T) V of every new token over the positions of its request in the cache, its own step's among them
    (write_pages comes first).

    q [tokens, heads, head_dim], heads a multiple of the pools' kv_heads: query heads h * heads / kv_heads and on read key head h.  causal: a
    token's positions end at its own; else at the request's last, as a chunk of latent frames sees all of itself.  window: of those
    positions only the last `window`, and the first `sink` of the request.  selected, group: only the pages that select_pages lists
    for each `group` tokens (int32 [selected_rows(tokens, requests, group), kv_heads, top], ascending, each page once; no window then).

    -> [tokens, heads, head_dim] in q's dtype, zeros for a token that sees nothing and for rows that nobody has (with out, rows that nobody
    has stay as they were; out must not overlap the other tensors); with return_lse also the natural logarithm of the sums, fp32
    [heads, tokens], -inf for nothing.  Rows that would read a position without a page (-1 or another number outside the pool,
    positions past the table) are NaN, and others of their request may be.  What lies in positions that a row does not see has no part in it,
    NaN or infinite.  table[:, :n] of the columns in use sizes the work."""
    if _needs_grad(q, k_pages, v_pages):
        raise NotImplementedError("paged_attention is not differentiable")
    ps = _pools(k_pages, v_pages, getattr(plan, "page_size", None))
    N, P, Hk, D = k_pages.shape
    dev = k_pages.device
    qs = _rows("q", q, k_pages.dtype, dev)
    T, H, qd = q.shape
    if qd != D or H < Hk or H % Hk:
        raise ValueError("q must be [tokens, heads, head_dim], heads a multiple of the pools' and head_dim theirs")
    if window is not None and window < 1:
        raise ValueError("window must be a position or more (None: all)")
    if sink < 0 or (sink and window is None):
        raise ValueError("sink: positions that stay visible outside a window")
    top = 0
    if selected is not None:
        if window is not None:
            raise ValueError("selected pages and a window do not go together")
        if group < 1:
            raise ValueError("group must be a token or more")
        rows = selected_rows(T, plan.q_start.shape[0] - 1, group)
        if (selected.dtype != torch.int32 or selected.device != dev or selected.dim() != 3 or selected.shape[:2] != (rows, Hk)
                or selected.shape[2] < 1 or not selected.is_contiguous()):
            raise ValueError(f"selected must be a contiguous int32 [{rows}, {Hk}, top] tensor on {dev}")
        top = selected.shape[2]
    zero_rest = out is None
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    elif out.shape != q.shape:
        raise ValueError("out must be like q")
    lse = None
    if return_lse:
        lse = torch.full((H, T), -math.inf, dtype=torch.float32, device=dev) if not zero_rest else torch.empty((H, T), dtype=torch.float32, device=dev)
    if T == 0:
        _plan(plan, 0, dev)
        return (out, lse) if return_lse else out
    d = _q_desc(q, qs, Hk, plan, N, ps, (H * D, D) if zero_rest else _rows("out", out, q.dtype, dev), float(D ** -0.5 if sm_scale is None else sm_scale), bool(causal),
                window or 0, sink, top, group, zero_rest)
    n = C.c_size_t(0)
    lib = _l.load()
    with _on_device(dev):
        _l.check(lib.sfm_paged_workspace_bytes(C.byref(d), C.byref(n)))
        ws = torch.empty(n.value, dtype=torch.uint8, device=dev) if n.value else None
        _l.check(lib.sfm_paged_attention(C.byref(d), q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(),
                                         plan.q_start.data_ptr(), None if selected is None else selected.data_ptr(), out.data_ptr(),
                                         None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), n.value,
                                         _raw_stream(dev.index)))
    if not zero_rest:
        _written(out)
    return (out, lse) if return_lse else out


def select_pages(q, means, plan, top, group=1, causal=False, first=1, last=1):
    """Which pages each `group` consecutive new tokens of a request read, for paged_attention's `selected`: int32
    [selected_rows(tokens, requests, group), kv_heads, top] entries of the request's row of the table, ascending, -1 behind them.

    Candidates are the pages up to the last one that the group's last token sees (causal: its own).  The first `first` and the last `last` of
    them are taken, and then those with the largest (sum of q over the group's tokens and the key head's query heads) . mean key, up
    to `top` in all; of level ones the lower.  means: fp32 [pages, kv_heads, head_dim], kept by write_pages.  Scores are sums in 64 bits,
    so that which page is ahead does not hang on the order of an addition; NaN counts as -inf, as does a page outside the pool.  Group i of request r
    is row q_start[r] // group + r + i; rows that nobody has are -1."""
    if _needs_grad(q, means):
        raise NotImplementedError("select_pages is not differentiable")
    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype not in _DT:
        raise ValueError("q must be a [tokens, heads, head_dim] GPU tensor of bf16, fp16 or fp32")
    qs = _rows("q", q, q.dtype, q.device)
    T, H, D = q.shape
    if means.dim() != 3 or means.dtype != torch.float32 or means.device != q.device or not means.is_contiguous() or means.shape[2] != D:
        raise ValueError("means must be a contiguous float32 [pages, kv_heads, head_dim] tensor on q's device")
    N, Hk = means.shape[:2]
    if H < Hk or H % Hk:
        raise ValueError("q's heads must be a multiple of the means'")
    if group < 1 or not 1 <= top <= _l.PAGED_TOP_MAX:
        raise ValueError(f"group must be a token or more, top 1 to {_l.PAGED_TOP_MAX} pages")
    if first < 0 or last < 0 or first + last > top:
        raise ValueError("first and last must not be negative, nor more than top together")
    R = _plan(plan, T, q.device)[0]
    selected = torch.empty((selected_rows(T, R, group), Hk, top), dtype=torch.int32, device=q.device)
    if T == 0:
        return selected.fill_(-1)
    d = _q_desc(q, qs, Hk, plan, N, (0, 0, 0), (0, 0), 1.0, bool(causal), 0, 0, top, group, 0)
    n = C.c_size_t(0)
    lib = _l.load()
    with _on_device(q.device):
        _l.check(lib.sfm_paged_select_workspace_bytes(C.byref(d), C.byref(n)))
        ws = torch.empty(n.value, dtype=torch.uint8, device=q.device) if n.value else None
        _l.check(lib.sfm_paged_select(C.byref(d), q.data_ptr(), means.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(), plan.q_start.data_ptr(),
                                      first, last, selected.data_ptr(), None if ws is None else ws.data_ptr(), n.value,
                                      _raw_stream(q.device.index)))
    return selected
