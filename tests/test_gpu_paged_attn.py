"""Attention over pages on the GPU against the oracle in 64 bits."""
import math

import pytest
import torch

import self_forcing_amd as sfa
from oracle import paged as oracle
from test_gpu_paged_cache import DEV, ints, randn, step

pytestmark = pytest.mark.gpu
PA = sfa.paged_attn
HALF = [torch.bfloat16, torch.float16]


def close(got, lse, want, dtype):
    """Off by at most: half a step of the result; of the sum of weight * |v|: half a step of the weights, which enter the product in
    the tensors' type (fp32: none), what the logits' fp32 sums may be off (twice: weight and sum of weights), and a rounding of
    2^-24 per key in the two sums; of the largest |v| per key half the type's smallest step, which a small weight beside the largest, 1, is off."""
    u = torch.finfo(dtype).eps / 2
    rel = (0 if dtype == torch.float32 else u) + (2 * want["slip"] + 2 * want["keys"] + 8) * 2.0 ** -24
    tol = u * want["out"].abs() + rel[..., None] * want["mag"] * (1 + u)
    tol += ((want["keys"] * want["top"] + 1) * torch.finfo(dtype).smallest_normal * u)[..., None]
    fine = ~want["bad"]
    assert not torch.isnan(got[fine]).any()
    off = (got.double() - want["out"]).abs()
    assert (off <= tol)[fine].all(), f"worst {(off / tol)[fine].max().item():.2f} of the bound"
    assert torch.isnan(got[want["bad"]]).all()
    assert (got[fine & (want["keys"] == 0)] == 0).all()
    if lse is not None:
        fine = fine.T
        nothing = fine & (want["keys"].T == 0)
        assert (lse[nothing] == -math.inf).all()
        some = fine & ~nothing
        bound = (want["slip"].T + want["keys"].T + 8 + 4 * want["lse"].abs().clamp(max=1e6)) * 2.0 ** -24
        assert ((lse.double() - want["lse"]).abs() <= bound)[some].all()
        assert torch.isnan(lse[want["bad"].T]).all()


def inputs(past, n, page, H, Hk, D, dtype, pad=0, seed=0, strength=1.0):
    plan, pages, (table, q_start, *_rest) = step(past, n, page, pad, seed)
    q = randn((sum(n) + pad, H, D), seed + 1, dtype) * strength
    kp, vp = (randn((pages, page, Hk, D), seed + s, dtype) for s in (2, 3))
    return plan, table, q_start, q, kp, vp


def check(past, n, page, H, Hk, D, dtype, pad=0, seed=0, strength=1.0, **more):
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, Hk, D, dtype, pad, seed, strength)
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, return_lse=True, **more)
    close(got.cpu(), lse.cpu(), oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, **more), dtype)


CASES = [  # past, new, page, heads, kv heads, rows behind the last request
    ([0], [1], 8, 1, 1, 0), ([63], [1], 64, 2, 2, 0), ([64], [1], 64, 2, 1, 0), ([0], [65], 16, 1, 1, 0), ([700], [1], 8, 8, 1, 0),
    ([5, 0, 130, 900, 0], [1, 1, 1, 1, 0], 16, 12, 3, 0), ([5, 0, 130, 260, 31], [40, 0, 1, 130, 33], 24, 4, 2, 7), ([100], [300], 40, 2, 2, 0),
    ([1560], [160], 1560, 2, 2, 0), ([300, 10], [70, 129], 8, 5, 1, 3), ([0], [513], 256, 1, 1, 0), ([40], [3], 8, 37, 1, 1),
]


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("past,n,page,H,Hk,pad", CASES)
def test_against_the_oracle(past, n, page, H, Hk, pad, causal, D, dtype):
    check(past, n, page, H, Hk, D, dtype, pad, causal=causal)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.float32, 40), (torch.bfloat16, 8), (torch.float16, 96), (torch.bfloat16, 256)], ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("past,n,page,H,Hk,pad", [CASES[1], CASES[6], CASES[9]])
def test_other_types_and_head_sizes(past, n, page, H, Hk, pad, causal, D, dtype):
    check(past, n, page, H, Hk, D, dtype, pad, causal=causal)


OTHER = [(torch.float32, 64, 4, 2), (torch.bfloat16, 256, 5, 1), (torch.float16, 96, 2, 2), (torch.bfloat16, 8, 12, 1)]


@pytest.mark.parametrize("dtype,D,H,Hk", OTHER, ids=str)
@pytest.mark.parametrize("window,sink", [(None, 0), (1000, 0), (1000, 70), (3, 1)])
@pytest.mark.parametrize("past,n,page", [([9000, 100], [1, 1], 16), ([700, 5], [9, 30], 40)])
def test_other_types_and_head_sizes_with_windows(past, n, page, window, sink, dtype, D, H, Hk):
    check(past, n, page, H, Hk, D, dtype, 3, causal=True, window=window, sink=sink)


@pytest.mark.parametrize("dtype,D,H,Hk", OTHER, ids=str)
@pytest.mark.parametrize("past,n,page,group,top", [([9000, 100], [1, 1], 16, 1, 200), ([700, 5], [9, 30], 8, 7, 9)])
def test_other_types_and_head_sizes_of_selected_pages(past, n, page, group, top, dtype, D, H, Hk):
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, Hk, D, dtype, pad=3)
    sel = lists(past, n, page, Hk, top, group, True, q.shape[0], q_start, 5, first=False)
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, selected=ints(sel.tolist()), group=group, return_lse=True)
    close(got.cpu(), lse.cpu(), oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True, selected=sel, group=group), dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 1), (64, 0), (100, 3), (100, 70), (128, 200), (5000, 9), (65, 64), (37, 500)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("past,n,page,H,Hk,pad", [CASES[6], CASES[7], CASES[5], ([900], [400], 16, 2, 1, 0)])
def test_window_and_sink(past, n, page, H, Hk, pad, causal, window, sink, D):
    check(past, n, page, H, Hk, D, torch.bfloat16, pad, causal=causal, window=window, sink=sink)


@pytest.mark.parametrize("n", [1, 3, 31, 32, 33, 127, 128, 129, 255, 256, 257, 300])
@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (8, 2)])
def test_numbers_of_rows(n, H, Hk):
    check([77, 1], [n, 1], 16, H, Hk, 64, torch.bfloat16, causal=True, seed=n)


@pytest.mark.parametrize("past", [0, 1, 6, 7, 8, 54, 55, 56, 62, 63, 64, 119, 120, 127, 128, 255, 510, 511, 512, 513, 1023, 1024, 2047, 2100])
def test_lengths_about_the_tiles_edges(past):
    check([past], [1], 8, 2, 1, 128, torch.bfloat16, causal=True, seed=past)
    check([past], [150], 8, 1, 1, 64, torch.float16, causal=False, seed=past)


@pytest.mark.parametrize("requests", [1, 63, 64, 65, 200])
def test_many_requests(requests):
    g = torch.Generator().manual_seed(requests)
    past = torch.randint(0, 90, (requests,), generator=g).tolist()
    n = torch.randint(0, 4, (requests,), generator=g).tolist()
    n[-1] = 1
    check(past, n, 16, 2, 1, 64, torch.bfloat16, pad=5, causal=True)


@pytest.mark.parametrize("strength", [0.0, 30.0])
def test_flat_and_steep_softmax(strength):
    check([300, 40], [70, 1], 16, 2, 1, 128, torch.bfloat16, causal=True, strength=strength)


@pytest.mark.parametrize("scale", [1e-3, 0.5])
def test_scale(scale):
    check([300, 40], [70, 1], 16, 2, 1, 64, torch.bfloat16, causal=True, sm_scale=scale)


# ---------------------------------------------------------------- selected pages
def lists(past, n, page, Hk, top, group, causal, tokens, q_start, seed, first=True):
    """Random ascending lists with -1 behind them; some of them empty."""
    g = torch.Generator().manual_seed(seed)
    out = torch.full((tokens // group + len(past) + 1, Hk, top), -1, dtype=torch.long)
    for r, (p, m) in enumerate(zip(past, n)):
        for i, t0 in enumerate(range(0, m, group)):
            pages = -(-(p + min(m, t0 + group) if causal else p + m) // page)
            for h in range(Hk):
                take = min(pages, int(torch.randint(0 if not first else 1, top + 1, (1,), generator=g)))
                out[int(q_start[r]) // group + r + i, h, :take] = torch.sort(torch.randperm(pages, generator=g)[:take])[0]
    return out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("past,n,page,H,Hk,group,top", [
    ([500], [1], 8, 2, 2, 1, 9), ([500, 0, 77, 1200], [1, 1, 1, 1], 16, 8, 2, 1, 30), ([90, 0, 400], [70, 65, 1], 8, 4, 2, 1, 6),
    ([90, 0, 400], [70, 65, 1], 16, 4, 2, 16, 12), ([300], [300], 64, 2, 2, 64, 4), ([300, 20], [300, 131], 24, 3, 1, 100, 10), ([700], [270], 8, 2, 2, 128, 100),
    ([700], [570], 32, 1, 1, 512, 30), ([1600, 900], [40, 300], 1560, 1, 1, 128, 1),
])
def test_selected_pages(past, n, page, H, Hk, group, top, causal, D):
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, Hk, D, torch.bfloat16, pad=3)
    sel = lists(past, n, page, Hk, top, group, causal, q.shape[0], q_start, 5, first=False)
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=causal, selected=ints(sel.tolist()), group=group, return_lse=True)
    close(got.cpu(), lse.cpu(), oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=causal, selected=sel, group=group), torch.bfloat16)


@pytest.mark.parametrize("group", [231, 1000, 2 ** 31 - 1])
def test_groups_larger_than_the_step(group):
    past, n, page = [300, 20], [100, 131], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 4, 2, 64, torch.bfloat16)
    means = kp.float().mean(1)
    sel = PA.select_pages(q.to(DEV), means.to(DEV), plan, 6, group=group, causal=True)
    assert torch.equal(sel.cpu().long(), oracle.select_pages(q, means, table, torch.tensor(past), q_start, page, 6, group, True))
    got = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, selected=sel, group=group)
    close(got.cpu(), None, oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True, selected=sel.cpu().long(), group=group), torch.bfloat16)


def test_counts_past_32_bits_are_one_of_everything():
    past, n, page, far = [300, 20], [100, 131], 16, 2 ** 32
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 4, 2, 64, torch.bfloat16)
    q, kp, vp = q.to(DEV), kp.to(DEV), vp.to(DEV)
    whole = PA.paged_attention(q, kp, vp, plan, causal=True)
    assert torch.equal(PA.paged_attention(q, kp, vp, plan, causal=True, window=far + 5), whole)
    got = PA.paged_attention(q, kp, vp, plan, causal=True, window=5, sink=far + 3)
    close(got.cpu(), None, oracle.attention(q.cpu(), kp.cpu(), vp.cpu(), table, torch.tensor(past), q_start, causal=True), torch.bfloat16)
    means = kp.float().mean(1)
    sel = PA.select_pages(q, means, plan, 6, group=far + 1, causal=True)
    assert torch.equal(sel, PA.select_pages(q, means, plan, 6, group=1000, causal=True))
    assert torch.equal(PA.paged_attention(q, kp, vp, plan, selected=sel, group=far + 1), PA.paged_attention(q, kp, vp, plan, selected=sel, group=1000))


@pytest.mark.parametrize("n", [[1, 1, 1], [40, 150, 3]])
def test_requests_that_share_pages(n):
    """A prompt's pages in the tables of several requests: read by all of them."""
    past, page = [96, 100, 200], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 4, 2, 128, torch.bfloat16)
    table = table.clone()
    table[1, :6] = table[2, :6] = table[0, :6]
    got = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan._replace(table=ints(table.tolist())), causal=True)
    close(got.cpu(), None, oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True), torch.bfloat16)


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)], ids=str)
def test_tables_wider_than_the_requests(D, dtype):
    """A table for 40000 positions: sizes follow from its width (many ranges, the cache read past the caches), results from the lengths."""
    g = torch.Generator().manual_seed(4)
    past, n, page = torch.randint(0, 300, (9,), generator=g).tolist(), [1] * 8 + [2], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 16, 8, D, dtype)
    wide = torch.full((9, 2500), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = plan.table
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan._replace(table=wide), causal=True, return_lse=True)
    close(got.cpu(), lse.cpu(), oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True), dtype)


def test_without_the_workspace_a_call_runs_whole():
    """The C entry takes a NULL or too small workspace: the same result within the bound, in one range."""
    import ctypes as C
    past, n, page = [5000, 300], [1, 1], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 4, 2, 128, torch.bfloat16)
    dq, dk, dv = q.to(DEV), kp.to(DEV), vp.to(DEV)
    out = torch.zeros_like(dq)
    d, _ = PA._attention_call(dq.device, PA._layout(dq), PA._layout(dk), PA._layout(dv), page, PA._plan_layout(plan), None, None, None, True, None, 0, 1)
    size = C.c_size_t(0)
    sfa.lib.check(sfa.lib.load().sfm_paged_workspace_bytes(C.byref(d), C.byref(size)))
    assert size.value > 0
    ws = torch.zeros(size.value - 1, dtype=torch.uint8, device=DEV)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True)
    for at, bytes_ in ((None, 0), (ws.data_ptr(), size.value - 1)):
        sfa.lib.check(sfa.lib.load().sfm_paged_attention(C.byref(d), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(),
                                                         plan.q_start.data_ptr(), None, out.data_ptr(), None, at, bytes_,
                                                         torch.cuda.current_stream().cuda_stream))
        close(out.cpu(), None, want, torch.bfloat16)
    assert not ws.any()


def test_workspaces_have_the_size_that_is_asked_for():
    import ctypes as C
    lib = sfa.lib.load()
    past, n, page = [5000, 300], [1, 1], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 4, 2, 128, torch.bfloat16)
    dq, dk, dv, means = q.to(DEV), kp.to(DEV), vp.to(DEV), kp.float().mean(1).to(DEV)
    out, sel = torch.zeros_like(dq), torch.zeros((PA.selected_rows(2, 2, 1), 2, 7), dtype=torch.int32, device=DEV)
    size, stream = C.c_size_t(0), torch.cuda.current_stream().cuda_stream

    def canary():
        return torch.full((size.value + 65536,), 0xA5, dtype=torch.uint8, device=DEV)
    d, _ = PA._attention_call(dq.device, PA._layout(dq), PA._layout(dk), PA._layout(dv), page, PA._plan_layout(plan), None, None, None, True, None, 0, 1)
    sfa.lib.check(lib.sfm_paged_workspace_bytes(C.byref(d), C.byref(size)))
    ws = canary()
    sfa.lib.check(lib.sfm_paged_attention(C.byref(d), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(),
                                          plan.q_start.data_ptr(), None, out.data_ptr(), None, ws.data_ptr(), size.value, stream))
    assert bool((ws[size.value:] == 0xA5).all()) and torch.equal(out, PA.paged_attention(dq, dk, dv, plan, causal=True))
    d, _, _ = PA._select_call(dq.device, PA._layout(dq), PA._layout(means), PA._plan_layout(plan), page, 7, 1, True, 1, 1)
    sfa.lib.check(lib.sfm_paged_select_workspace_bytes(C.byref(d), C.byref(size)))
    ws = canary()
    sfa.lib.check(lib.sfm_paged_select(C.byref(d), dq.data_ptr(), means.data_ptr(), plan.table.data_ptr(), plan.past.data_ptr(), plan.q_start.data_ptr(), 1, 1,
                                       sel.data_ptr(), ws.data_ptr(), size.value, stream))
    assert bool((ws[size.value:] == 0xA5).all()) and torch.equal(sel, PA.select_pages(dq, means, plan, 7, causal=True))


def test_all_pages_selected_is_the_whole_attention():
    past, n, page = [300, 20], [100, 131], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 4, 2, 64, torch.bfloat16)
    args = (q.to(DEV), kp.to(DEV), vp.to(DEV), plan)
    sel = torch.arange(26, device=DEV, dtype=torch.int32).expand(PA.selected_rows(231, 2, 64), 2, 26).contiguous()
    a, b = PA.paged_attention(*args, causal=True), PA.paged_attention(*args, causal=True, selected=torch.where(sel < 26, sel, -1), group=64)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True)
    # request 1 has 10 pages: entries past them belong to no position that is seen, and have no page to be read from
    close(a.cpu(), None, want, torch.bfloat16)
    close(b.cpu(), None, want, torch.bfloat16)


# ---------------------------------------------------------------- what must have no part
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 64), (torch.float32, 64)], ids=str)
@pytest.mark.parametrize("past,n,H", [([70, 3], [1, 1], 4), ([70, 3], [140, 1], 4), ([500], [300], 1), ([9000], [1], 1)])
def test_what_a_row_does_not_see_has_no_part(past, n, H, dtype, D, value):
    """Stale rows behind the requests' ends, pages of nobody, and (causal) the request's later tokens."""
    page = 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, 1, D, dtype)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True)
    used = torch.zeros(kp.shape[:2], dtype=torch.bool)
    for r, (p, m) in enumerate(zip(past, n)):
        pos = torch.arange(p + m)
        used[table[r, pos // page], pos % page] = True
    for t in (kp, vp):
        t[~used] = value
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, return_lse=True)
    close(got.cpu(), lse.cpu(), want, dtype)
    # the last new token of request 0 on top: seen by its own row alone
    last = past[0] + n[0] - 1
    for t in (kp, vp):
        t[table[0, last // page], last % page] = value
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, return_lse=True)
    row = n[0] - 1
    assert not torch.isfinite(got[row].cpu()).any()
    want["bad"][row] = False
    keep = torch.ones(q.shape[0], dtype=torch.bool)
    keep[row] = False
    close(got.cpu()[keep], lse.cpu()[:, keep], {k: (v[:, keep] if k == "lse" else v[keep]) for k, v in want.items()}, dtype)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)], ids=str)
def test_infinite_values_reach_the_rows_that_see_them(dtype, D):
    """An infinity in a channel of one V row: that channel of the rows that see it, and no other."""
    past, n, page = [40], [150], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 2, 1, D, dtype)
    for pos, channel, value in ((100, 5, math.inf), (101, 6, -math.inf), (110, 5, math.nan), (189, 0, math.inf)):
        vp[table[0, pos // page], pos % page, 0, channel] = value
    got = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True).cpu()
    end = torch.arange(150) + 41
    assert (got[end <= 100][:, :, 5].isfinite()).all() and (got[(end > 100) & (end <= 110)][:, :, 5] == math.inf).all()
    assert got[end > 110][:, :, 5].isnan().all() and (got[end > 101][:, :, 6] == -math.inf).all() and got[end <= 101][:, :, 6].isfinite().all()
    assert got[:-1, :, 0].isfinite().all() and (got[-1, :, 0] == math.inf).all()
    rest = torch.ones(D, dtype=torch.bool)
    rest[[0, 5, 6]] = False
    vp = torch.where(vp.isfinite(), vp, 0.0).to(dtype)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True)
    want["out"], want["mag"] = want["out"][..., rest], want["mag"][..., rest]
    close(got[..., rest], None, want, dtype)


@pytest.mark.parametrize("past,n,H,D,dtype", [([9000, 700], [1, 1], 2, 128, torch.bfloat16), ([9000], [1], 8, 64, torch.float16), ([9000], [40], 1, 128, torch.bfloat16),
                                              ([700], [150], 2, 64, torch.bfloat16), ([9000], [1], 2, 40, torch.bfloat16)], ids=str)
def test_logits_of_minus_infinity(past, n, H, D, dtype):
    """Keys that a row sees with a logit of -infinity weigh nothing, a whole range of them too; a row that sees no others is NaN, as 0 / 0."""
    page = 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, 1, D, dtype)
    q[..., 0] = 1.0
    far = 60000.0 if dtype == torch.float16 else 1e6              # a logit of -6e3 and less: the weight is 0 in 64 bits
    for r, p in enumerate(past):
        pos = torch.arange(p // 2)
        kp[table[r, pos // page], pos % page, 0, 0] = -far
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True)
    kp[kp == -far] = -math.inf
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, return_lse=True)
    close(got.cpu(), lse.cpu(), want, dtype)
    kp[..., 0] = -math.inf
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, return_lse=True)
    assert got.isnan().all() and (lse == -math.inf).all()


def test_a_window_hides_what_has_left_it():
    """Pages behind the window may be gone from the table, and what they held may be anything."""
    past, n, page, window, sink = [1000, 300], [90, 1], 16, 200, 20
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 2, 1, 128, torch.bfloat16)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True, window=window, sink=sink)
    gone = table.clone()
    for r, (p, m) in enumerate(zip(past, n)):
        lo = p + 1 - window                                    # of the request's first new token
        for pos in range(sink, lo):
            vp[table[r, pos // page], pos % page] = math.nan
            kp[table[r, pos // page], pos % page] = math.nan
        gone[r, -(-sink // page):lo // page] = -1
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan._replace(table=ints(gone.tolist())), causal=True, window=window, sink=sink,
                                  return_lse=True)
    close(got.cpu(), lse.cpu(), want, torch.bfloat16)


# ---------------------------------------------------------------- pages outside the pool, rows of nobody
@pytest.mark.parametrize("page_no", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
@pytest.mark.parametrize("D,H,n", [(128, 2, [150, 3]), (64, 8, [1, 1]), (40, 2, [9, 3])])
def test_rows_that_read_a_position_without_a_page_are_nan(page_no, D, H, n):
    past, page = [100, 500], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, 1, D, torch.bfloat16)
    table = table.clone()
    table[1, 9] = kp.shape[0] if page_no == "pages" else page_no
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan._replace(table=ints(table.tolist())), causal=True, return_lse=True)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True)
    assert want["bad"][n[0]:].all() and not want["bad"][:n[0]].any()
    close(got.cpu(), lse.cpu(), want, torch.bfloat16)


@pytest.mark.parametrize("D", [128, 40])
def test_a_request_longer_than_its_row_of_the_table(D):
    past, n, page = [100, 500], [20, 30], 16
    plan, table, q_start, q, kp, vp = inputs(past, n, page, 2, 1, D, torch.bfloat16)
    narrow = plan.table[:, :20]
    got = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan._replace(table=narrow), causal=True).cpu()
    close(got, None, oracle.attention(q, kp, vp, table[:, :20], torch.tensor(past), q_start, causal=True), torch.bfloat16)
    assert got[20:].isnan().all()


@pytest.mark.parametrize("D", [128, 40])
def test_rows_of_nobody_stay_as_they_were(D):
    past, n = [100, 0], [20, 2]
    plan, table, q_start, q, kp, vp = inputs(past, n, 16, 2, 1, D, torch.bfloat16, pad=70)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    got, lse = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, out=out, return_lse=True)
    assert got is out and (out[22:] == 7).all() and (lse[:, 22:] == -math.inf).all()
    free = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True)
    assert torch.equal(free[:22], out[:22]) and (free[22:] == 0).all()


def test_offsets_that_make_no_sense_stay_inside():
    """q_start and past that no plan makes: whatever comes out, rows past the tensors are neither read nor written."""
    past, n = [100, 40, 7], [20, 2, 300]
    plan, table, q_start, q, kp, vp = inputs(past, n, 16, 4, 2, 64, torch.bfloat16)
    for qs, ps in (([0, 20, 10, 322], past), ([5, 5, 5, 5], past), ([-9, 20, 2 ** 31 - 1, 3], past), ([0, 20, 22, 322], [2 ** 31 - 1, -4, 10 ** 6])):
        out = torch.full((q.shape[0] + 2, 4, 64), 7.0, dtype=q.dtype, device=DEV)
        bad = plan._replace(q_start=ints(qs), past=ints(ps))
        PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), bad, causal=True, out=out[1:-1])
        assert (out[0] == 7).all() and (out[-1] == 7).all()
        means = torch.zeros((kp.shape[0], 2, 64), device=DEV)
        sel = PA.select_pages(q.to(DEV), means, bad, 4, group=16, causal=True)
        PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), bad, causal=True, selected=sel, group=16, out=out[1:-1])
        assert (out[0] == 7).all() and (out[-1] == 7).all()
        PA.write_pages(q[:, :2].to(DEV), q[:, 2:].to(DEV), kp.to(DEV), vp.to(DEV), bad, means=means)


def test_lists_that_make_no_sense_stay_inside():
    past, n = [100, 40], [70, 1]
    plan, table, q_start, q, kp, vp = inputs(past, n, 16, 4, 2, 64, torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    for hi in (20, 10 ** 6, 2 ** 31 - 1):
        sel = torch.randint(0, hi, (PA.selected_rows(71, 2, 32), 2, 9), generator=g).to(torch.int32).to(DEV)
        out = torch.full((73, 4, 64), 7.0, dtype=q.dtype, device=DEV)
        PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True, selected=sel, group=32, out=out[1:-1])
        assert (out[0] == 7).all() and (out[-1] == 7).all()


# ---------------------------------------------------------------- layouts, streams, graphs
@pytest.mark.parametrize("D,n", [(128, [150, 3]), (64, [1, 2]), (40, [9, 3])])
def test_layouts(D, n):
    """Heads outside the rows of a page, rows of a fused projection, an output inside a larger tensor, one head of many."""
    past, page, H, Hk = [100, 300], 16, 4, 2
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, Hk, D, torch.bfloat16)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True)
    pools = [t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)]
    fused = torch.zeros((q.shape[0], 3, H, D), dtype=q.dtype, device=DEV)
    fused[:, 1] = q.to(DEV)
    out = torch.zeros((q.shape[0] + 2, H + 1, D), dtype=q.dtype, device=DEV)
    PA.paged_attention(fused[:, 1], *pools, plan, causal=True, out=out[1:-1, 1:])
    close(out[1:-1, 1:].cpu(), None, want, torch.bfloat16)
    assert not out[0].any() and not out[-1].any() and not out[:, 0].any()
    one = PA.paged_attention(fused[:, 1, 2:3], pools[0][:, :, 1:], pools[1][:, :, 1:], plan, causal=True)
    want = {k: (v[2:3] if k == "lse" else v[:, 2:3]) for k, v in want.items()}
    close(one.cpu(), None, want, torch.bfloat16)


def serve(dtype, D, H, Hk, group, top, steps, seed, page=16):
    """A few steps of two requests: plan, write with means, attention over everything and over selected pages; every step against the
    oracle, which keeps a cache of its own."""
    g = torch.Generator().manual_seed(seed)
    pages, W, R = 90, 40, 3
    order = torch.randperm(pages, generator=g)
    table, past, taken = torch.full((R, W), -1), torch.zeros(R, dtype=torch.long), 0
    kp = vp = torch.zeros((pages, page, Hk, D), dtype=dtype)
    means = torch.zeros((pages, Hk, D))
    d = dict(table=ints(table.tolist()), past=ints([0] * R), free=ints(order.tolist()), nf=None, k=kp.to(DEV), v=vp.to(DEV), m=means.to(DEV))
    for i, n in enumerate(steps):
        n = torch.tensor(n)
        T = int(n.sum()) + 2
        q, k, v = (randn((T, h, D), seed + 10 * i + s, dtype) for s, h in ((0, H), (1, Hk), (2, Hk)))
        plan = PA.plan_pages(d["table"], d["past"], ints(n.tolist()), d["free"], T, page, next_free=d["nf"])
        PA.write_pages(k.to(DEV), v.to(DEV), d["k"], d["v"], plan, means=d["m"])
        got, lse = PA.paged_attention(q.to(DEV), d["k"], d["v"], plan, causal=True, return_lse=True)
        table, q_start, lengths, slots, taken = oracle.plan(table, past, n, order, T, page, taken)
        kp, vp, means = oracle.write(k, v, kp, vp, slots, table, past, q_start, means)
        assert torch.equal(d["k"].cpu(), kp) and torch.equal(d["v"].cpu(), vp)
        close(got.cpu(), lse.cpu(), oracle.attention(q, kp, vp, table, past, q_start, causal=True), dtype)
        sel = PA.select_pages(q.to(DEV), d["m"], plan, top, group=group, causal=True)
        # from the means as the device has them: which page is ahead may hang on their last bit
        assert torch.equal(sel.cpu().long(), oracle.select_pages(q, d["m"].cpu(), table, past, q_start, page, top, group, True, 1, 1))
        got = PA.paged_attention(q.to(DEV), d["k"], d["v"], plan, causal=True, selected=sel, group=group)
        close(got.cpu(), None, oracle.attention(q, kp, vp, table, past, q_start, causal=True, selected=sel.cpu().long(), group=group), dtype)
        past, d["past"], d["nf"] = lengths, plan.lengths, plan.next_free


@pytest.mark.parametrize("dtype,D,H,Hk,group", [(torch.bfloat16, 128, 4, 2, 16), (torch.float16, 64, 2, 2, 1), (torch.float32, 40, 2, 1, 8)], ids=str)
def test_steps_of_serving(dtype, D, H, Hk, group):
    serve(dtype, D, H, Hk, group, 4, [[150, 0, 20], [1, 70, 1], [1, 1, 1], [1, 0, 1], [40, 1, 1]], 7)


@pytest.mark.parametrize("n", [[1, 1, 1], [150, 3, 40]])
def test_another_stream_and_a_graph(n):
    past, page, H, Hk, D = [400, 50, 7], 16, 4, 2, 128
    plan0, pages, (table, q_start, *_rest) = step(past, n, page)
    T = sum(n)
    k, v, q = (randn((T, h, D), s, torch.bfloat16).to(DEV) for s, h in ((1, Hk), (2, Hk), (3, H)))
    kp, vp = (randn((pages, page, Hk, D), s, torch.bfloat16).to(DEV) for s in (4, 5))
    means = randn((pages, Hk, D), 6, torch.float32).to(DEV)
    held = torch.where(torch.arange(table.shape[1])[None] < -(-torch.tensor(past)[:, None] // page), table, -1)
    used = set(held[held >= 0].tolist())
    free = ints([p for p in range(pages) if p not in used])
    d_table, d_past, d_n = ints(held.tolist()), ints(past), ints(n)

    def run():
        plan = PA.plan_pages(d_table, d_past, d_n, free, T, page)
        PA.write_pages(k, v, kp, vp, plan, means=means)
        full, lse = PA.paged_attention(q, kp, vp, plan, causal=True, return_lse=True)
        sel = PA.select_pages(q, means, plan, 3, group=4, causal=True)
        return plan.slots, full, lse, sel, PA.paged_attention(q, kp, vp, plan, causal=True, selected=sel, group=4)
    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        q.copy_(randn(q.shape, 50 + i, torch.bfloat16).to(DEV))
        k.copy_(randn(k.shape, 60 + i, torch.bfloat16).to(DEV))
        want = [t.clone() for t in run()]
        for t in out:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16), (96, torch.bfloat16)], ids=str)
def test_decoding_steps_of_one_graph(D, dtype):
    """A step that moves its own lengths and list of free pages on, replayed: every step the bits of the eager one, over pages' and tiles' ends."""
    page, H, Hk, R, W, steps = 16, 8, 2, 3, 40, 40
    g = torch.Generator().manual_seed(3)
    pages = R * W
    free = ints(torch.randperm(pages, generator=g).tolist())
    new, (q, k, v) = ints([1, 0, 1]), (torch.zeros((3, h, D), dtype=dtype, device=DEV) for h in (H, Hk, Hk))

    def state():
        prompt = PA.plan_pages(torch.full((R, W), -1, dtype=torch.int32, device=DEV), ints([0] * R), ints([250, 9, 30]), free, 289, page)
        kp, vp = (torch.full((pages, page, Hk, D), math.nan, dtype=dtype, device=DEV) for _ in range(2))
        means = torch.zeros((pages, Hk, D), device=DEV)
        PA.write_pages(*(randn((289, Hk, D), s, dtype).to(DEV) for s in (1, 2)), kp, vp, prompt, means=means)
        return prompt.table, prompt.lengths.clone(), prompt.next_free.clone(), kp, vp, means

    def run(table, past, taken, kp, vp, means):
        plan = PA.plan_pages(table, past, new, free, 3, page, next_free=taken)
        PA.write_pages(k, v, kp, vp, plan, means=means)
        out, lse = PA.paged_attention(q, kp, vp, plan, causal=True, return_lse=True)
        sel = PA.select_pages(q, means, plan, 5, causal=True)
        some = PA.paged_attention(q, kp, vp, plan, causal=True, selected=sel)
        torch.add(plan.lengths, 0, out=past)
        torch.add(plan.next_free, 0, out=taken)
        return plan.slots, out, lse, sel, some
    eager, replayed = state(), state()
    run(*state())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*replayed)
    for i in range(steps):
        for t, s in ((q, 100), (k, 200), (v, 300)):
            t.copy_(randn(t.shape, s + i, dtype).to(DEV))
        want = run(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) if a.is_floating_point() else torch.equal(a, b) for a, b in zip(got, want)), i
        assert want[1][:2].isfinite().all() and not want[1][2].any()           # two rows, and one of nobody
    assert replayed[1].tolist() == [250 + steps, 9, 30 + steps] and torch.equal(replayed[0], eager[0]) and torch.equal(replayed[2], eager[2])


def test_calls_at_once_on_two_streams():
    """Each call has a workspace of its own (ranges of keys, scores): the same bits as one after the other."""
    def make(seed):
        past, n, page = [3000, 200], [1, 1], 16
        plan, _, _, q, kp, vp = inputs(past, n, page, 8, 2, 128, torch.bfloat16, seed=seed)
        q, kp, vp = q.to(DEV), kp.to(DEV), vp.to(DEV)
        means = kp.float().mean(1)

        def run():
            sel = PA.select_pages(q, means, plan, 9, causal=True)
            return sel, PA.paged_attention(q, kp, vp, plan, causal=True, selected=sel), *PA.paged_attention(q, kp, vp, plan, causal=True, return_lse=True)
        return run, run(), kernel(plan, q, kp)
    runs = [make(1), make(2)]
    assert all(k[1] > 1 for _, _, k in runs)                   # split
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (run, _, _) in enumerate(runs):
            with torch.cuda.stream(streams[i]):
                got[i].append(run())
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(runs):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_under_inference_mode():
    past, n, page = [30, 7], [40, 1], 16
    plan0, table, q_start, q, kp, vp = inputs(past, n, page, 2, 1, 64, torch.bfloat16)
    with torch.inference_mode():
        own = [t.to(DEV) for t in (kp, vp)]
        means = torch.zeros((kp.shape[0], 1, 64), device=DEV)
        plan = PA.plan_pages(plan0.table.clone(), plan0.past, ints(n), ints([]), 41, page)
        PA.write_pages(randn((41, 1, 64), 4, torch.bfloat16).to(DEV), randn((41, 1, 64), 5, torch.bfloat16).to(DEV), *own, plan, means=means)
        out = PA.paged_attention(q.to(DEV), *own, plan, causal=True)
        again = PA.paged_attention(q.to(DEV), *own, plan, causal=True, out=torch.empty_like(out))
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))             # bits: without free pages some rows are NaN
    assert out[:40].isnan().any() and out[40].isfinite().all()


def test_repeated_calls_agree_bit_for_bit():
    plan, table, q_start, q, kp, vp = inputs([4000, 3000, 100], [1, 1, 70], 16, 8, 2, 128, torch.bfloat16)
    args = (q.to(DEV), kp.to(DEV), vp.to(DEV), plan)
    first = PA.paged_attention(*args, causal=True)
    for _ in range(5):
        assert torch.equal(PA.paged_attention(*args, causal=True), first)


@pytest.mark.parametrize("D,n", [(128, [1, 1]), (128, [200, 70]), (64, [1, 130])])
def test_pools_past_four_gib(D, n):
    """Pages near the end of pools of 5 GiB: row offsets pass 32 bits."""
    past, page, Hk = [100, 700], 64, 4
    plan, pages, (table, q_start, _, slots, _) = step(past, n, page)
    big = 5 * 2 ** 30 // (page * Hk * D * 2)
    at = big - pages
    kp, vp = (torch.zeros((big, page, Hk, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    small = [randn((pages, page, Hk, D), s, torch.bfloat16) for s in (1, 2)]
    kp[at:], vp[at:] = small[0].to(DEV), small[1].to(DEV)
    T = sum(n)
    k, v = (randn((T, Hk, D), s, torch.bfloat16) for s in (3, 4))
    far = plan._replace(table=torch.where(plan.table >= 0, plan.table + at, plan.table), slots=plan.slots + at * page)
    means = torch.zeros((big, Hk, D), device=DEV)
    PA.write_pages(k.to(DEV), v.to(DEV), kp, vp, far, means=means)
    wk, wv, wm = oracle.write(k, v, *small, slots, table, torch.tensor(past), q_start, torch.zeros((pages, Hk, D)))
    assert torch.equal(kp[at:].cpu(), wk) and torch.equal(vp[at:].cpu(), wv) and not kp[:at].any()
    assert (means[at:].cpu().double() - wm).abs().max() <= 65 * 2.0 ** -24 * wk.abs().max().double()
    q = randn((T, 2 * Hk, D), 9, torch.bfloat16)
    got, lse = PA.paged_attention(q.to(DEV), kp, vp, far, causal=True, return_lse=True)
    close(got.cpu(), lse.cpu(), oracle.attention(q, wk, wv, table, torch.tensor(past), q_start, causal=True), torch.bfloat16)


# ---------------------------------------------------------------- which kernel a call takes
def kernel(plan, q, kp, causal=True, window=None, selected=None, group=1):
    """(rows of a piece, ranges of the keys, whether the cache is read past the caches)."""
    import ctypes as C
    out = [C.c_int32() for _ in range(3)]
    d, _ = PA._attention_call(kp.device, PA._layout(q), PA._layout(kp), PA._layout(kp), kp.shape[1], PA._plan_layout(plan), None,
                              None if selected is None else PA._layout(selected), None, causal, window, 0, group)
    sfa.lib.check(sfa.lib.load().sfm_paged_attention_plan(d, *map(C.byref, out)))
    return tuple(x.value for x in out)


def test_every_kernel_is_reached_by_the_tests_above():
    def of(past, n, page, H, Hk, D=128, dtype=torch.bfloat16, width=None):
        plan, _, _, q, kp, _ = inputs(past, n, page, H, Hk, D, dtype)
        if width:
            plan = plan._replace(table=torch.full((len(past), width), -1, dtype=torch.int32, device=DEV))
        return kernel(plan, q.to(DEV), kp.to(DEV))
    assert of([63], [1], 64, 2, 2) == (32, 1, 0)                               # test_against_the_oracle
    assert of([700], [1], 8, 8, 1)[:2] == (32, 2)
    rows, ranges, once = of([0] * 9, [1] * 8 + [2], 16, 16, 8, width=2500)     # test_tables_wider_than_the_requests
    assert rows == 32 and ranges > 1 and once == 1
    assert of([100], [300], 40, 2, 2) == (128, 1, 0)
    assert of([300, 10], [70, 129], 8, 5, 1)[0] == 128
    assert of([9000, 100], [1, 1], 16, 5, 1, 256)[1] > 1                         # test_other_types_and_head_sizes_with_windows
    assert of([63], [1], 64, 2, 2, 40)[0] == 0 and of([63], [1], 64, 2, 2, 64, torch.float32)[0] == 0


def test_every_kernel_is_reached_by_long_contexts():
    def of(past, n, page, H, Hk, D):
        plan, q, kp, _ = long_inputs(past, n, page, H, Hk, D, torch.bfloat16)
        return kernel(plan, q, kp)
    rows, ranges, _ = of([40000], [1], 64, 8, 2, 128)
    assert rows == 32 and ranges > 8
    assert of([18000], [2048], 16, 16, 16, 64) == (128, 1, 0)                  # more tiles than a stretch of places holds
    assert of([34000], [3700], 1560, 16, 16, 64) == (256, 1, 0)
    rows, ranges, _ = of([20000, 19000], [40, 2], 40, 12, 2, 128)
    assert rows == 128 and ranges > 1


# ---------------------------------------------------------------- long contexts, against the definition in 64 bits on the GPU
def long_inputs(past, n, page, H, Hk, D, dtype, seed=0):
    """Pools on the GPU whose pages lie in no order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    whole = [-(-(p + m) // page) for p, m in zip(past, n)]
    pages = sum(whole) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table, at = torch.full((len(past), max(whole)), -1, dtype=torch.int32, device=DEV), 0
    for r, w in enumerate(whole):
        table[r, :w] = order[at:at + w]
        at += w
    held = table.clone()
    for r, p in enumerate(past):
        held[r, -(-p // page):] = -1
    free = torch.cat([table[r, -(-p // page):w] for r, (p, w) in enumerate(zip(past, whole))] + [order[at:]])
    plan = PA.plan_pages(held, ints(past), ints(n), free, sum(n), page)
    assert torch.equal(plan.table, table)
    kp, vp = (torch.randn((pages, page, Hk, D), generator=g, device=DEV, dtype=torch.float32).to(dtype) for _ in range(2))
    return plan, torch.randn((sum(n), H, D), generator=g, device=DEV).to(dtype), kp, vp


def check_rows(got, lse, plan, q, kp, vp, past, n, tokens, causal, window=None, sink=0, selected=None, group=1):
    """A few tokens of the output, all heads, within the bound of `close`."""
    page, Hk, D = kp.shape[1:]
    G, want, start = q.shape[1] // Hk, [], 0
    for r, (p, m) in enumerate(zip(past, n)):
        for t in [t - start for t in tokens if start <= t < start + m]:
            end = p + t + 1 if causal else p + m
            pos = torch.arange(end, device=DEV)
            if window is not None:
                pos = pos[(pos >= end - window) | (pos < sink)]
            rows = plan.table[r].long()[pos // page] * page + pos % page
            k, v = (x.view(-1, Hk, D)[rows].double() for x in (kp, vp))
            x = torch.einsum("hgd,khd->hgk", q[start + t].double().view(Hk, G, D).cpu(), k.cpu()).to(DEV) * D ** -0.5
            if selected is not None:
                e = selected[start // group + r + t // group].long()
                seen = (e[:, :, None] == (pos // page)[None, None]).any(1)
                x = x.masked_fill(~seen[:, None], -math.inf)
            l = torch.logsumexp(x, -1)
            w = torch.exp(x - l[..., None])
            y = torch.stack([w[h] @ v[:, h] for h in range(Hk)]).view(-1, D)
            mag = torch.stack([w[h] @ v[:, h].abs() for h in range(Hk)]).view(-1, D)
            mass = torch.einsum("hgd,khd->hgk", q[start + t].double().abs().view(Hk, G, D).cpu(), k.abs().cpu()).to(DEV).amax(-1) * D ** -0.5
            fin = torch.where(x.isfinite(), x, 0.0)
            slip = (mass * (D + 4) + fin.abs().amax(-1) * 4 + 16).view(-1)
            want.append((start + t, y, l.view(-1), mag, slip, len(pos), v.abs().amax()))
        start += m
    t = torch.tensor([w[0] for w in want], device=DEV)
    ref = dict(out=torch.stack([w[1] for w in want]), lse=torch.stack([w[2] for w in want]).T, mag=torch.stack([w[3] for w in want]),
               slip=torch.stack([w[4] for w in want]), keys=torch.tensor([[w[5]] * q.shape[1] for w in want], device=DEV),
               top=torch.stack([w[6].expand(q.shape[1]) for w in want]))
    ref["bad"] = torch.zeros_like(ref["slip"], dtype=torch.bool)
    close(got[t].cpu(), lse[:, t].cpu(), {k: v.cpu() for k, v in ref.items()}, q.dtype)


@pytest.mark.parametrize("past,n,page,H,Hk,D,causal,window,sink", [
    ([40000], [1], 64, 8, 2, 128, True, None, 0), ([33000, 70, 16000], [1, 1, 1], 8, 4, 4, 64, True, None, 0),
    ([18000], [2048], 16, 16, 16, 64, True, None, 0), ([16500], [2048], 64, 16, 16, 128, False, None, 0),
    ([34000], [3700], 1560, 16, 16, 64, False, None, 0), ([33000], [3700], 32, 16, 16, 128, True, None, 0),
    ([18000], [2048], 16, 16, 16, 64, True, 100, 17000), ([34000], [3700], 64, 16, 16, 64, True, 2000, 33000), ([20000, 19000], [40, 2], 40, 12, 2, 128, True, 5000, 64),
    ([0], [4680], 64, 12, 12, 64, True, None, 0), ([0, 1000, 5], [1000, 1024, 700], 40, 16, 4, 128, True, None, 0), ([0], [6000], 16, 32, 8, 64, True, None, 0),
])
@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_long_contexts(past, n, page, H, Hk, D, causal, window, sink, dtype):
    plan, q, kp, vp = long_inputs(past, n, page, H, Hk, D, dtype)
    got, lse = PA.paged_attention(q, kp, vp, plan, causal=causal, window=window, sink=sink, return_lse=True)
    T = sum(n)
    tokens = sorted({0, 1, T // 3, T // 2, T - 2, T - 1} & set(range(T)))
    check_rows(got, lse, plan, q, kp, vp, past, n, tokens, causal, window, sink)


def test_long_contexts_selected():
    past, n, page, group, top = [30000], [1024], 64, 128, 300
    plan, q, kp, vp = long_inputs(past, n, page, 16, 16, 64, torch.bfloat16)
    means = kp.float().mean(1)
    sel = PA.select_pages(q, means, plan, top, group=group, causal=True)
    got, lse = PA.paged_attention(q, kp, vp, plan, causal=True, selected=sel, group=group, return_lse=True)
    check_rows(got, lse, plan, q, kp, vp, past, n, [0, 127, 128, 700, 1023], True, selected=sel, group=group)


@pytest.mark.parametrize("past,n,H,Hk,D,window,sink,rows", [
    ([9000, 100, 0], [1, 1, 1], 4, 2, 128, 3000, 70, 32), ([9000, 2037], [30, 1], 2, 2, 64, 2000, 0, 32), ([3000, 700], [300, 2], 2, 2, 128, 1500, 1, 128),
    ([9000], [40], 4, 1, 64, 4000, 200, 128), ([9000, 100], [1, 3], 4, 2, 96, 2000, 9, 0)])
@pytest.mark.parametrize("causal", [False, True])
def test_ranges_of_a_window(past, n, H, Hk, D, window, sink, rows, causal):
    """Ranges hold the most tiles that a piece can have, in a table of any width."""
    plan, table, q_start, q, kp, vp = inputs(past, n, 8, H, Hk, D, torch.bfloat16)
    want = oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=causal, window=window, sink=sink)
    q, kp, vp = q.to(DEV), kp.to(DEV), vp.to(DEV)
    for width in (plan.table.shape[1], 5000):
        wide = torch.full((len(past), width), -1, dtype=torch.int32, device=DEV)
        wide[:, :plan.table.shape[1]] = plan.table
        p = plan._replace(table=wide)
        assert kernel(p, q, kp, causal, window)[0] == rows and kernel(p, q, kp, causal, window)[1] > 1
        got, lse = PA.paged_attention(q, kp, vp, p, causal=causal, window=window, sink=sink, return_lse=True)
        close(got.cpu(), lse.cpu(), want, torch.bfloat16)


@pytest.mark.parametrize("n", [[150, 3], [1, 1]])
def test_columns_of_one_buffer(n):
    """q, out, k and v as columns of the same rows, K's and V's pools as halves of one: nothing is shared, nothing refused."""
    past, page, H, Hk, D = [70, 30], 16, 4, 2, 64
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, Hk, D, torch.bfloat16)
    T = sum(n)
    rows = torch.zeros((T, 2 * H + 2 * Hk, D), dtype=torch.bfloat16, device=DEV)
    rows[:, :H] = q.to(DEV)
    pool = torch.stack([kp, vp], 1).to(DEV)
    k, v = (randn((T, Hk, D), s, torch.bfloat16) for s in (5, 6))
    rows[:, 2 * H:2 * H + Hk], rows[:, 2 * H + Hk:] = k.to(DEV), v.to(DEV)
    PA.write_pages(rows[:, 2 * H:2 * H + Hk], rows[:, 2 * H + Hk:], pool[:, 0], pool[:, 1], plan)
    out = rows[:, H:2 * H]
    assert PA.paged_attention(rows[:, :H], pool[:, 0], pool[:, 1], plan, causal=True, out=out) is out
    kp, vp, _ = oracle.write(k, v, kp, vp, plan.slots.cpu(), table, torch.tensor(past), q_start)
    assert torch.equal(pool[:, 0].cpu(), kp) and torch.equal(pool[:, 1].cpu(), vp)
    close(out.cpu(), None, oracle.attention(q, kp, vp, table, torch.tensor(past), q_start, causal=True), torch.bfloat16)
    assert torch.equal(rows[:, :H].cpu(), q)
    for taken in (rows[:, :H], rows[:, 1:H + 1], rows[:, H - 1:2 * H - 1]):
        with pytest.raises(sfa.lib.SfmError, match="out overlaps q"):
            PA.paged_attention(rows[:, :H], pool[:, 0], pool[:, 1], plan, causal=True, out=taken)
    inside = pool[0, 0].expand(T, page, Hk, D)[:, 0]
    with pytest.raises(sfa.lib.SfmError, match="k overlaps k_pages"):
        PA.write_pages(inside, inside, pool[:, 0], pool[:, 1], plan)
    assert torch.equal(pool[:, 0].cpu(), kp) and torch.equal(rows[:, :H].cpu(), q)


@pytest.mark.parametrize("past,n,H,Hk,D,dtype,rows", [
    ([9000], [1], 4, 1, 128, torch.bfloat16, 32), ([700], [5], 2, 2, 64, torch.float16, 32), ([700], [300], 1, 1, 128, torch.bfloat16, 128),
    ([9000], [40], 1, 1, 64, torch.float16, 128), ([700], [9], 2, 1, 96, torch.bfloat16, 0), ([3000], [2], 1, 1, 64, torch.float32, 0)], ids=str)
@pytest.mark.parametrize("weight", [0, 1])
def test_infinite_values_with_any_weight(past, n, H, Hk, D, dtype, rows, weight):
    """Infinities in whole tiles, in early ranges and in the last tile, whose weights go to 0 or do not: never a finite number in that channel of
    a row that sees them, infinite where the weight is a plain number, and nothing in the others."""
    page, total = 16, past[0] + n[0]
    plan, table, q_start, q, kp, vp = inputs(past, n, page, H, Hk, D, dtype)
    q[..., 0] = 1.0
    at = {3: 1, 70: 2, past[0] // 2: 3, past[0] - 1: 4, total - 1: 5}              # position: channel
    for pos in at:
        kp[table[0, pos // page], pos % page, :, 0] = 0.0 if weight else -8000.0        # a logit of -700 and less: exp is 0 in 32 bits
    want = oracle.attention(q, kp, torch.where(vp.isfinite(), vp, 0.0), table, torch.tensor(past), q_start, causal=True)
    for pos, channel in at.items():
        vp[table[0, pos // page], pos % page, :, channel] = math.inf
    assert kernel(plan, q.to(DEV), kp.to(DEV))[0] == rows
    got = PA.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), plan, causal=True).cpu()
    end = torch.arange(n[0]) + past[0] + 1
    for pos, channel in at.items():
        assert not got[end > pos][:, :, channel].isfinite().any() and got[end <= pos][:, :, channel].isfinite().all()
        assert not weight or (got[end > pos][:, :, channel] == math.inf).all()
    rest = torch.ones(D, dtype=torch.bool)
    rest[list(at.values())] = False
    want["out"], want["mag"] = want["out"][..., rest], want["mag"][..., rest]
    close(got[..., rest], None, want, dtype)
