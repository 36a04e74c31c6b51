"""What the paged cache's entry points and functions refuse, without a GPU."""
import ctypes as C
import random

import pytest
import torch

import self_forcing_amd as sfa
from self_forcing_amd import lib as L

PA = sfa.paged_attn
P = 4096                                          # an aligned address that nothing reads: every call here is refused


def desc(**change):
    d = L.PagedDesc(L.SFM_BF16, 8, 2, 128, 10, 3, 5, 40, 16, 5, (16 * 2 * 128, 2 * 128, 128), (8 * 128, 128), (8 * 128, 128), 0.1, 1, 0, 0, 0, 1, 1, 0)
    for k, v in change.items():
        setattr(d, k, v)
    return d


def attention(d, **ptr):
    p = dict(q=P, k=P, v=P, table=P, past=P, q_start=P, selected=None, out=P, lse=None, ws=None)
    p.update(ptr)
    return L.load().sfm_paged_attention(C.byref(d), p["q"], p["k"], p["v"], p["table"], p["past"], p["q_start"], p["selected"], p["out"], p["lse"],
                                        p["ws"], 0, None)


def select(d, first=1, last=1, **ptr):
    p = dict(q=P, means=P, table=P, past=P, q_start=P, selected=P, ws=None)
    p.update(ptr)
    return L.load().sfm_paged_select(C.byref(d), p["q"], p["means"], p["table"], p["past"], p["q_start"], first, last, p["selected"], p["ws"], 0, None)


def write(d, stride=(256, 128), **ptr):
    p = dict(k=P, v=P, kp=P, vp=P, slots=P, table=P, past=P, q_start=P, means=P)
    p.update(ptr)
    return L.load().sfm_paged_write(C.byref(d), p["k"], p["v"], (C.c_int64 * 2)(*stride), p["kp"], p["vp"], p["slots"], p["table"], p["past"],
                                    p["q_start"], p["means"], None)


def plan(requests=3, width=5, page=16, tokens=10, stride=5, free_count=9, **ptr):
    # addresses far apart: outputs must not lie in inputs
    p = dict(table=1 << 20, past=2 << 20, new=3 << 20, free=4 << 20, taken=None, q_start=5 << 20, lengths=6 << 20, slots=7 << 20, next_free=8 << 20)
    p.update(ptr)
    return L.load().sfm_paged_plan(requests, width, page, tokens, p["table"], stride, p["past"], p["new"], p["free"], free_count, p["taken"], p["q_start"],
                                   p["lengths"], p["slots"], p["next_free"], None, 0, None)


NULL, DTYPE, SHAPE, RANGE, STRIDE, WORKSPACE, ALIGN = -1, -2, -3, -4, -5, -6, -7
SHARED = [(dict(dtype=7), DTYPE), (dict(kv_heads=0), SHAPE), (dict(kv_heads=65536, H=65536), SHAPE), (dict(D=12), SHAPE), (dict(D=264), SHAPE), (dict(D=0), SHAPE), (dict(pages=0), SHAPE),
          (dict(requests=0), SHAPE), (dict(requests=(1 << 24) + 1), SHAPE), (dict(width=0), SHAPE), (dict(page_size=12), SHAPE), (dict(page_size=0), SHAPE),
          (dict(width=1 << 20, page_size=2048, table_stride=1 << 20), SHAPE), (dict(width=(1 << 20) + 1, page_size=1024, table_stride=1 << 21), SHAPE), (dict(pages=1 << 20, page_size=2048), SHAPE), (dict(tokens=0), SHAPE),
          (dict(tokens=-1), SHAPE), (dict(tokens=1 << 31), SHAPE), (dict(table_stride=4), STRIDE)]
POOL = [(dict(pool_stride=(4096, 256, 120)), STRIDE), (dict(pool_stride=(4096, 256, 132)), STRIDE), (dict(pool_stride=(4096, 64, 128)), STRIDE),
        (dict(pool_stride=(-4096, 256, 128)), STRIDE), (dict(pool_stride=(4096, 1 << 24, 128)), STRIDE)]
Q = [(dict(H=7), SHAPE), (dict(H=1), SHAPE), (dict(tokens=1 << 29), SHAPE), (dict(q_stride=(1024, 129)), STRIDE), (dict(q_stride=(-1024, 128)), STRIDE),
     (dict(top=-1), SHAPE), (dict(top=2049), SHAPE), (dict(top=2, group=0), SHAPE)]


@pytest.mark.parametrize("change,code", SHARED + POOL + Q + [
    (dict(o_stride=(1024, 64)), STRIDE), (dict(o_stride=(1020, 128)), STRIDE), (dict(sm_scale=0.0), SHAPE), (dict(sm_scale=float("nan")), SHAPE),
    (dict(sm_scale=float("inf")), SHAPE), (dict(sm_scale=3.0e38), SHAPE), (dict(top=2048, page_size=1 << 20, width=1, pages=1), SHAPE), (dict(window=-1), RANGE), (dict(sink=-1), RANGE), (dict(sink=3), RANGE), (dict(top=4, window=8), RANGE)])
def test_attention_refuses(change, code):
    d, n = desc(**change), C.c_size_t(0)
    assert attention(d, selected=P) == code
    assert L.load().sfm_paged_workspace_bytes(C.byref(d), C.byref(n)) == code
    out = [C.c_int32() for _ in range(3)]
    assert L.load().sfm_paged_attention_plan(C.byref(d), *map(C.byref, out)) == code
    assert L.load().sfm_paged_attention_plan(C.byref(desc()), None, C.byref(out[0]), C.byref(out[1])) == NULL


@pytest.mark.parametrize("ptr,code", [(dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(table=None), NULL), (dict(past=None), NULL),
                                      (dict(q_start=None), NULL), (dict(out=None), NULL), (dict(q=P + 2), ALIGN), (dict(v=P + 8), ALIGN), (dict(out=P + 4), ALIGN),
                                      (dict(table=P + 2), ALIGN), (dict(lse=P + 2), ALIGN), (dict(ws=P + 8), ALIGN)])
def test_attention_refuses_pointers(ptr, code):
    assert attention(desc(), **ptr) == code
    assert attention(desc(top=4), selected=None) == NULL and attention(desc(top=4), selected=P + 1) == ALIGN


@pytest.mark.parametrize("change,code", SHARED + Q + [(dict(top=0), SHAPE)])
def test_select_refuses(change, code):
    d, n = desc(**{"top": 4, **change}), C.c_size_t(0)
    assert select(d) == code
    assert L.load().sfm_paged_select_workspace_bytes(C.byref(d), C.byref(n)) == code


def test_select_refuses_the_rest():
    d = desc(top=4)
    for name in ("q", "means", "table", "past", "q_start", "selected"):
        assert select(d, **{name: None}) == NULL
        assert select(d, **{name: P + 2}) == ALIGN
    assert select(d, first=-1) == RANGE and select(d, last=-1) == RANGE and select(d, first=3, last=2) == RANGE
    assert select(d, first=2 ** 31 - 1, last=2 ** 31 - 1) == RANGE


@pytest.mark.parametrize("change,code", SHARED + POOL)
def test_write_refuses(change, code):
    assert write(desc(**change)) == code


def test_write_refuses_the_rest():
    for name in ("k", "v", "kp", "vp", "slots", "table", "past", "q_start"):
        assert write(desc(), **{name: None}) == NULL
        assert write(desc(), **{name: P + 2}) == ALIGN
    assert write(desc(), stride=(257, 128)) == STRIDE and write(desc(), stride=(256, -128)) == STRIDE and write(desc(), means=P + 2) == ALIGN


def test_plan_refuses():
    for kw, code in [(dict(requests=0), SHAPE), (dict(width=0), SHAPE), (dict(page=4), SHAPE), (dict(page=20), SHAPE), (dict(tokens=-1), SHAPE),
                     (dict(tokens=1 << 31), SHAPE), (dict(stride=4), STRIDE), (dict(free_count=-1), RANGE), (dict(width=1 << 28, stride=1 << 28), SHAPE)]:
        assert plan(**kw) == code, kw
    for name in ("table", "past", "new", "free", "q_start", "lengths", "slots", "next_free"):
        assert plan(**{name: None}) == NULL, name
    for name in ("table", "past", "new", "free", "taken", "q_start", "lengths", "slots", "next_free"):
        assert plan(**{name: (20 << 20) + 2}) == ALIGN, name
    assert plan(slots=(7 << 20) + 4) == ALIGN
    assert plan(q_start=2 << 20) == RANGE and plan(next_free=9 << 20, taken=9 << 20) == RANGE and plan(lengths=2 << 20) == RANGE
    assert plan(slots=(1 << 20) + 8) == RANGE and plan(table=(4 << 20) + 32) == RANGE
    assert plan(requests=9000, stride=5, width=5) == WORKSPACE
    n = C.c_size_t(1)
    assert L.load().sfm_paged_plan_workspace_bytes(0, C.byref(n)) == SHAPE and L.load().sfm_paged_plan_workspace_bytes(3, None) == NULL
    assert L.load().sfm_paged_plan_workspace_bytes(3, C.byref(n)) == 0 and n.value == 0
    assert L.load().sfm_paged_workspace_bytes(C.byref(desc()), None) == NULL and L.load().sfm_paged_select_workspace_bytes(C.byref(desc()), None) == NULL
    assert L.load().sfm_paged_workspace_bytes(None, C.byref(n)) == NULL


# ---------------------------------------------------------------- the functions, with tensors that are not on the GPU
def cpu_plan(T=4, R=2):
    i = torch.zeros(R, dtype=torch.int32)
    return PA.PagePlan(torch.zeros((R, 3), dtype=torch.int32), i, i, torch.zeros(R + 1, dtype=torch.int32), torch.zeros(T, dtype=torch.int64),
                       torch.zeros(1, dtype=torch.int32), 16)


def test_functions_want_the_gpu():
    pool, q = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16), torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        PA.plan_pages(torch.zeros((2, 3), dtype=torch.int32), i, i, i, 4, 16)
    with pytest.raises(ValueError, match="GPU"):
        PA.write_pages(q, q, pool, pool, cpu_plan())
    with pytest.raises(ValueError, match="GPU"):
        PA.paged_attention(q, pool, pool, cpu_plan())
    with pytest.raises(ValueError, match="GPU"):
        PA.select_pages(q, torch.zeros((4, 2, 64)), cpu_plan(), 2)


def test_gradients_are_refused():
    pool, q = torch.zeros((4, 16, 2, 64)), torch.zeros((4, 2, 64), requires_grad=True)
    leaf = torch.zeros((4, 16, 2, 64), requires_grad=True)
    for call in (lambda: PA.write_pages(q.detach(), q.detach(), leaf, pool, cpu_plan()), lambda: PA.paged_attention(q.detach(), pool, pool, cpu_plan(), out=q),
                 lambda: PA.write_pages(q, q, pool, pool, cpu_plan()), lambda: PA.paged_attention(q, pool, pool, cpu_plan()),
                 lambda: PA.paged_attention(q.detach(), pool, pool.requires_grad_(), cpu_plan()), lambda: PA.select_pages(q, pool[:, 0], cpu_plan(), 2)):
        with pytest.raises(NotImplementedError, match="differentiable"):
            call()


def test_tangents_are_refused():
    pool, q, means, plan = torch.zeros((4, 16, 2, 64)), torch.zeros((4, 2, 64)), torch.zeros((4, 2, 64)), cpu_plan()
    calls = {"k": lambda t: PA.write_pages(t(q), q, pool, pool, plan), "v": lambda t: PA.write_pages(q, t(q), pool, pool, plan),
             "k_pages": lambda t: PA.write_pages(q, q, t(pool), pool, plan), "v_pages": lambda t: PA.write_pages(q, q, pool, t(pool), plan),
             "means": lambda t: PA.write_pages(q, q, pool, pool, plan, means=t(means)), "q": lambda t: PA.paged_attention(t(q), pool, pool, plan),
             "keys": lambda t: PA.paged_attention(q, t(pool), pool, plan), "values": lambda t: PA.paged_attention(q, pool, t(pool), plan),
             "out": lambda t: PA.paged_attention(q, pool, pool, plan, out=t(q)), "queries": lambda t: PA.select_pages(t(q), means, plan, 2),
             "scores": lambda t: PA.select_pages(q, t(means), plan, 2)}
    with torch.autograd.forward_ad.dual_level():
        for name, call in calls.items():
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="differentiable"):
                    call(lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
            with pytest.raises(ValueError, match="GPU"):          # none: only the device is wrong
                call(lambda t: t)
    with pytest.raises(NotImplementedError, match="differentiable"):
        calls["means"](lambda t: t.clone().requires_grad_())


def test_tables_and_arrays():
    for bad in (torch.zeros((2, 3), dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros((0, 3), dtype=torch.int32),
                torch.zeros((3, 2), dtype=torch.int32).T):
        with pytest.raises(ValueError, match="table"):
            PA._table(PA._layout(bad))
    with pytest.raises(ValueError, match="table"):
        PA.plan_pages(None, None, None, None, 4, 16)
    assert PA._table(PA._layout(torch.zeros((4, 9), dtype=torch.int32)[::2, 3:5])) == (2, 2, 18)
    assert PA._table(PA._layout(torch.zeros((4, 9), dtype=torch.int32)[:1, 3:5])) == (1, 2, 2)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros((2, 1), dtype=torch.int32), [1, 2], torch.zeros(3, dtype=torch.int32)):
        with pytest.raises(ValueError):
            PA._ints("past", bad, torch.device("cpu"), 2)
    assert PA._ints("past", torch.arange(6, dtype=torch.int32)[::3], torch.device("cpu"), 2).tolist() == [0, 3]


def test_strides_of_rows_and_pools():
    x = torch.zeros((5, 3, 2, 8))
    assert PA._rows("q", PA._layout(x[:, 1]), x.dtype) == (48, 8)
    assert PA._rows("q", PA._layout(x[:1, 1, 1:]), x.dtype) == (8, 8)        # dimensions of one
    with pytest.raises(ValueError):
        PA._rows("q", PA._layout(x[:, 1].transpose(1, 2)), x.dtype)
    with pytest.raises(ValueError):
        PA._rows("q", PA._layout(x[:, 1]), torch.float16)
    with pytest.raises(ValueError):
        PA._rows("q", PA._layout(x), x.dtype)
    assert PA._pool("k", PA._layout(x)) == (48, 16, 8)
    assert PA._pool("k", PA._layout(x[:1, :, :1])) == (48, 16, 8)
    assert PA._pool("k", PA._layout(x.transpose(1, 2))) == (48, 8, 16)
    with pytest.raises(ValueError):
        PA._pool("k", PA._layout(x.transpose(2, 3)))
    assert PA._pools(PA._layout(x), PA._layout(x.clone()), 3) == (48, 16, 8)
    for other, page in ((x.half(), 3), (x[:4], 3), (x.transpose(1, 2).contiguous().transpose(1, 2), 3), (x, 16)):
        with pytest.raises(ValueError):
            PA._pools(PA._layout(x), PA._layout(other), page)


def test_layouts_of_plans():
    layout = PA._plan_layout(cpu_plan())
    assert PA._planned(layout, 4) == (2, 3, 3)
    with pytest.raises(ValueError, match="slots"):
        PA._planned(layout, 5)
    with pytest.raises(ValueError, match="q_start"):
        PA._planned(PA._plan_layout(cpu_plan()._replace(q_start=torch.zeros(2, dtype=torch.int32))), 4)
    with pytest.raises(ValueError, match="past"):
        PA._planned(PA._plan_layout(cpu_plan()._replace(past=torch.zeros(4, dtype=torch.int32)[::2])), 4)
    with pytest.raises(ValueError, match="PagePlan"):
        PA._plan_layout(tuple(cpu_plan()))


GPU_ONLY = [
    ("q heads", dict(H=3), "multiple"), ("q size", dict(D=32), "head_dim"), ("q type", dict(dtype=torch.float16), "expected"),
    ("window", dict(window=0), "window"), ("sink", dict(sink=2), "sink"), ("both", dict(window=4, selected=True), "together"), ("group", dict(group=0, selected=True), "group"),
    ("lists", dict(group=3, selected=True), "selected must"), ("out", dict(out=(5, 2, 64)), "like q"), ("rows", dict(T=5), "slots"), ("page size", dict(page=8), "rows"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("name,kw,match", GPU_ONLY, ids=[n for n, *_ in GPU_ONLY])
def test_attention_refuses_tensors(name, kw, match):
    dev = "cuda:0"
    kw = dict(kw)
    plan = PA.PagePlan(*(t.to(dev) if isinstance(t, torch.Tensor) else t for t in cpu_plan()))._replace(page_size=kw.pop("page", 16))
    pool = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16, device=dev)
    q = torch.zeros((kw.pop("T", 4), kw.pop("H", 4), kw.pop("D", 64)), dtype=kw.pop("dtype", torch.bfloat16), device=dev)
    if "out" in kw:
        kw["out"] = torch.zeros(kw["out"], dtype=q.dtype, device=dev)
    if kw.pop("selected", False):
        kw["selected"] = torch.zeros((PA.selected_rows(4, 2, 1), 2, 3), dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match=match):
        PA.paged_attention(q, pool, pool, plan, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, -16, 12, 2 ** 32 + 16])
def test_plan_refuses_pages(page):
    i = torch.zeros(2, dtype=torch.int32, device="cuda:0")
    with pytest.raises(ValueError, match="page_size"):
        PA.plan_pages(torch.zeros((2, 3), dtype=torch.int32, device="cuda:0"), i, i, i, 4, page)


@pytest.mark.gpu
def test_empty_steps():
    dev = "cuda:0"
    plan = PA.plan_pages(torch.zeros((2, 3), dtype=torch.int32, device=dev), *(torch.zeros(2, dtype=torch.int32, device=dev) for _ in range(3)), 0, 16)
    pool = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16, device=dev)
    q, k = pool.new_zeros((0, 4, 64)), pool.new_zeros((0, 2, 64))
    PA.write_pages(k, k, pool, pool, plan)
    out, lse = PA.paged_attention(q, pool, pool, plan, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    assert bool((PA.select_pages(q, torch.zeros((4, 2, 64), device=dev), plan, 2) == -1).all()) and plan.q_start.tolist() == [0, 0, 0]


def empty_rows(dev="cpu"):
    """k and v of no tokens whose strides differ, both contiguous as any tensor without elements is."""
    k, v = torch.zeros((2, 3, 64), dtype=torch.bfloat16, device=dev).transpose(0, 1)[:0], torch.zeros((0, 2, 64), dtype=torch.bfloat16, device=dev)
    assert k.stride() != v.stride() and k.is_contiguous() and v.is_contiguous()
    return k, v


def test_empty_rows_need_no_layout_in_common():
    k, v = empty_rows()
    pool, plan = PA._layout(torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)), PA._plan_layout(cpu_plan(0))
    assert PA._write_call(PA._layout(k), PA._layout(v), pool, pool, 16, plan, None)[1] is not None
    k, v = k.new_zeros((3, 2, 64))[:2], v.new_zeros((2, 2, 128))[..., :64]
    assert PA._write_call(PA._layout(k), PA._layout(v), pool, pool, 16, PA._plan_layout(cpu_plan(2)), None)[1] is None


@pytest.mark.gpu
def test_empty_steps_in_layouts_of_their_own():
    plan = PA.PagePlan(*(t.to("cuda:0") if isinstance(t, torch.Tensor) else t for t in cpu_plan(0)))
    pools = torch.ones((2, 4, 16, 2, 64), dtype=torch.bfloat16, device="cuda:0")
    PA.write_pages(*empty_rows("cuda:0"), *pools, plan)
    assert bool((pools == 1).all())


M = 1 << 20
APART = dict(q=16 * M, k=17 * M, v=18 * M, table=19 * M, past=20 * M, q_start=21 * M, out=22 * M, lse=23 * M, ws=24 * M)      # every call with them is refused


@pytest.mark.parametrize("name,at", [(n, p) for n, p in APART.items() if n not in ("out", "lse", "ws")] + [("selected", 25 * M)])
def test_out_and_lse_in_inputs_are_refused(name, at):
    d = desc(top=4, group=2)
    apart = dict(APART, selected=25 * M)
    for to in ("out", "lse"):
        assert attention(d, **dict(apart, **{to: at})) == RANGE
        assert L.load().sfm_last_error().decode() == f"{to} overlaps {dict(k='k_pages', v='v_pages').get(name, name)}"
    assert attention(d, **dict(apart, lse=APART["out"])) == RANGE and attention(d, **dict(apart, lse=APART["out"] + 9 * 8 * 128 * 2)) == RANGE
    # the last row of q, a column of q's rows, rows that overlap each other
    assert attention(d, **dict(apart, out=APART["q"] + 10 * 8 * 128 * 2 - 16)) == RANGE
    assert attention(desc(q_stride=(4096, 128), o_stride=(4096, 128)), **dict(APART, out=APART["q"] + 2048 - 16)) == RANGE
    assert attention(desc(o_stride=(128, 128)), **APART) == RANGE and attention(desc(o_stride=(960, 128)), **APART) == RANGE


def test_rows_to_write_in_the_pools_are_refused():
    far = dict(k=16 * M, v=17 * M, kp=18 * M, vp=19 * M, slots=20 * M, table=21 * M, past=22 * M, q_start=23 * M, means=24 * M)
    for name in ("k", "v"):
        for pool in ("kp", "vp"):
            assert write(desc(), **dict(far, **{name: far[pool] + 256})) == RANGE
            assert write(desc(), **dict(far, **{name: far[pool] + 40 * 16 * 2 * 128 * 2 - 16})) == RANGE
            assert write(desc(), **dict(far, **{name: far[pool] - 10 * 256 * 2 + 16})) == RANGE


# ---------------------------------------------------------------- which kernel a call takes, and in how many ranges (of 256 compute units, the GPU's and the default)
def kernel(**change):
    out = [C.c_int32() for _ in range(3)]
    assert L.load().sfm_paged_attention_plan(C.byref(desc(**change)), *map(C.byref, out)) == 0
    return tuple(x.value for x in out)


def test_ranges_follow_the_window():
    """A window's keys are a few tiles of a table for 30000 positions: ranges are of those, and what lies in the caches is read from them."""
    tokens = dict(tokens=16, requests=16, H=32, kv_heads=8, width=1875, table_stride=1875, pages=40000)
    rows, ranges, once = kernel(**tokens)
    assert rows == 32 and ranges > 8 and once
    for window, sink, most in ((500, 0, 9), (1, 0, 2), (500, 100, 11), (64, 0, 3)):
        rows, ranges, once = kernel(**tokens, window=window, sink=sink)
        assert rows == 32 and ranges <= -(-most // 4) and not once, (window, sink)
    prompt = dict(tokens=512, requests=1, H=8, kv_heads=8, width=1900, table_stride=1900, pages=2000)
    assert kernel(**prompt)[1] > 4 and kernel(**prompt, window=1000)[1] <= 4
    other = dict(tokens, D=96)
    assert kernel(**other)[1] > 4 and kernel(**other, window=500)[1] <= 3
    assert kernel(**tokens, window=40000) == kernel(**tokens) == kernel(**tokens, window=30000, sink=9)


def test_pieces_of_256_rows_fill_the_chip_in_one_range():
    rng, wide = random.Random(7), 0
    for _ in range(20000):
        kv, tokens, width = rng.choice([1, 2, 3, 4, 8, 12, 16, 40]), rng.choice([rng.randint(1, 300), rng.randint(1, 40000)]), rng.choice([3, 40, 500, 3000, 60000])
        window = rng.choice([0, 0, rng.randint(1, 5000)])
        rows, ranges, _ = kernel(tokens=tokens, requests=rng.choice([1, 1, 2, 5, 40]), kv_heads=kv, H=kv * rng.choice([1, 2, 4, 8]), width=width, table_stride=width,
                                 pages=width, D=rng.choice([64, 128]), causal=rng.randint(0, 1), window=window)
        assert rows in (32, 128, 256) and 1 <= ranges <= 64 and (rows < 256 or ranges == 1)
        wide += rows == 256
    assert wide > 100


def test_ranges_of_selected_pages():
    """One range where half the compute units or more have few pages that lie in the memory-side cache, whatever the head size."""
    def ranges(tokens, D, top, kv_heads=8, page_size=32):
        return kernel(tokens=tokens, requests=tokens, D=D, H=4 * kv_heads, kv_heads=kv_heads, width=1000, table_stride=1000, page_size=page_size, top=top, group=1)[1]
    assert ranges(16, 128, 64) == 1 and ranges(32, 64, 64) == 1 and ranges(64, 128, 16) == 1 and ranges(48, 64, 32) == 1
    assert ranges(16, 128, 160) > 1 and ranges(64, 128, 64) > 1 and ranges(64, 64, 64) > 1 and ranges(64, 64, 128) > 1 and ranges(32, 128, 128) > 1
    assert ranges(8, 128, 64) > 1 and ranges(24, 128, 64, 4) > 1


def test_what_may_be_read_again_is_read_through_the_caches():
    """Past the caches only single tokens go, and few rows to a request, of which only few can be in a second piece of one."""
    def once(tokens, requests, G, **more):
        return kernel(tokens=tokens, requests=requests, kv_heads=8, H=8 * G, width=1000, table_stride=1000, pages=40000, **more)
    assert once(32, 32, 1)[2] and once(32, 32, 32)[2] and once(128, 32, 1)[2] and once(128, 32, 4)[2] and once(20, 32, 4)[2]
    for tokens, G in ((931, 1), (32 * 20, 1), (32 * 5, 4)):
        assert once(tokens, 32, G)[0] == 32 and not once(tokens, 32, G)[2]
    assert not once(32, 32, 4, window=500)[2]
