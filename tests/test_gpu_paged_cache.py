"""Block tables, slots, paged writes with the pages' mean keys and the selection of pages, on the GPU against the oracle."""
import pytest
import torch

import self_forcing_amd as sfa
from oracle import paged as oracle

pytestmark = pytest.mark.gpu
PA = sfa.paged_attn
DEV = "cuda:0"


def ints(v, dev=DEV):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def draw_lens(R, past_hi, new, seed):
    g = torch.Generator().manual_seed(seed)
    past = torch.randint(0, past_hi + 1, (R,), generator=g)
    return past, torch.randint(new[0], new[1] + 1, (R,), generator=g)


def held_table(past, W, page, seed):
    """Random distinct pages for what the requests hold, -1 elsewhere; the pages left."""
    g = torch.Generator().manual_seed(seed + 1)
    held = [min(W, -(-int(p) // page)) for p in past]
    n = sum(held)
    order = torch.randperm(n + 20000 if n > 50000 else 2 * n + 4000, generator=g)
    table, at = torch.full((len(past), W), -1, dtype=torch.long), 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    return table, order[at:]


def check_plan(plan, want):
    table, q_start, lengths, slots, next_free = want
    assert torch.equal(plan.table.cpu().long(), table)
    assert torch.equal(plan.q_start.cpu().long(), q_start)
    assert torch.equal(plan.lengths.cpu().long(), lengths)
    assert torch.equal(plan.slots.cpu(), slots)
    assert plan.next_free.item() == next_free


PLANS = [  # requests, past up to, new, page size, rows behind the last request, table columns past the need
    (1, 0, (1, 1), 8, 0, 0), (1, 40, (0, 0), 8, 3, 0), (1, 5000, (4680, 4680), 1560, 0, 2), (3, 7, (0, 1), 16, 0, 0),
    (64, 300, (1, 1), 16, 0, 1), (65, 300, (0, 9), 24, 11, 0), (257, 100, (0, 40), 8, 0, 0), (1023, 60, (0, 3), 64, 1, 0),
    (4097, 30, (0, 2), 16, 0, 0), (8192, 20, (0, 1), 8, 5, 0), (8193, 20, (0, 1), 8, 0, 0), (20000, 20, (0, 2), 8, 0, 0),
]


@pytest.mark.parametrize("R,past_hi,new,page,pad,wider", PLANS)
def test_plan(R, past_hi, new, page, pad, wider):
    past, n = draw_lens(R, past_hi, new, R + page)
    W = max(1, -(-int((past + n).max()) // page)) + wider
    table, free = held_table(past, W, page, R)
    tokens = int(n.sum()) + pad
    plan = PA.plan_pages(ints(table.tolist()), ints(past.tolist()), ints(n.tolist()), ints(free.tolist()), tokens, page)
    check_plan(plan, oracle.plan(table, past, n, free, tokens, page))


def test_plan_where_the_list_ends_or_the_table_is_too_narrow():
    past, n, page = torch.tensor([30, 0, 17, 100, 5]), torch.tensor([40, 0, 60, 50, 9]), 16
    for W, pages in ((12, 3), (12, 0), (5, 100), (5, 4)):
        table, free = held_table(past, W, page, 3)
        free = free[:pages]
        plan = PA.plan_pages(ints(table.tolist()), ints(past.tolist()), ints(n.tolist()), ints(free.tolist()), int(n.sum()), page)
        check_plan(plan, oracle.plan(table, past, n, free, int(n.sum()), page))


def test_plan_fewer_rows_than_tokens():
    past, n, page = torch.tensor([30, 0, 17, 8]), torch.tensor([40, 33, 60, 50]), 8
    table, free = held_table(past, 20, page, 3)
    for tokens in (0, 1, 40, 41, 100, 182):
        plan = PA.plan_pages(ints(table.tolist()), ints(past.tolist()), ints(n.tolist()), ints(free.tolist()), tokens, page)
        check_plan(plan, oracle.plan(table, past, n, free, tokens, page))


def test_plan_numbers_that_make_no_sense():
    big = 2 ** 31 - 1
    past, n, page = torch.tensor([-5, 3, big, 16]), torch.tensor([20, -7, 2, 4]), 16
    table, free = held_table(torch.tensor([0, 3, 0, 16]), 6, page, 3)
    free[1], table[3, 0] = -9, -3
    plan = PA.plan_pages(ints(table.tolist()), ints(past.tolist()), ints(n.tolist()), ints(free.tolist()), 30, page, next_free=ints([-4]))
    t, q_start, lengths, slots, nf = oracle.plan(table, past, n, free, 30, page, next_free=-4)
    check_plan(plan, (t, q_start, lengths.clamp(max=big), slots, nf))


def test_steps_go_on_with_the_list_where_the_last_plan_left_it():
    page, R, W = 8, 5, 12
    past = torch.zeros(R, dtype=torch.long)
    table, free = torch.full((R, W), -1), torch.randperm(200, generator=torch.Generator().manual_seed(1))
    d_table, d_free, d_past, nf, taken = ints(table.tolist()), ints(free.tolist()), ints([0] * R), None, 0
    for step in range(12):
        n = torch.randint(0, 9, (R,), generator=torch.Generator().manual_seed(step))
        plan = PA.plan_pages(d_table, d_past, ints(n.tolist()), d_free, int(n.sum()) + 2, page, next_free=nf)
        want = oracle.plan(table, past, n, free, int(n.sum()) + 2, page, taken)
        check_plan(plan, want)
        table, _, past, _, taken = want
        d_past, nf = plan.lengths, plan.next_free


def test_plan_of_a_view_of_the_table_leaves_the_rest():
    past, n, page = torch.tensor([30, 0, 17]), torch.tensor([40, 9, 60]), 16
    table, free = held_table(past, 6, page, 3)
    whole = torch.full((7, 11), 77, dtype=torch.int32, device=DEV)
    view = whole[::2][1:, 2:8]
    view.copy_(table)
    plan = PA.plan_pages(view, ints(past.tolist()), ints(n.tolist()), ints(free.tolist()), int(n.sum()), page)
    want = oracle.plan(table, past, n, free, int(n.sum()), page)
    check_plan(plan, want)
    rest = torch.full((7, 11), 77, dtype=torch.long)
    rest[::2][1:, 2:8] = want[0]
    assert torch.equal(whole.cpu().long(), rest)


# ---------------------------------------------------------------- write
def step(past, n, page, pad=0, seed=0, spare=4):
    """(plan, pages of the pool, cpu copies) for the requests' lengths."""
    past, n = torch.tensor(past), torch.tensor(n)
    W = max(1, max(-(-(int(p) + int(m)) // page) for p, m in zip(past, n))) + 1
    g = torch.Generator().manual_seed(seed)
    held = [-(-int(p) // page) for p in past]
    pages = sum(-(-(int(p) + int(m)) // page) for p, m in zip(past, n)) + spare
    order = torch.randperm(pages, generator=g)
    table, at = torch.full((len(past), W), -1, dtype=torch.long), 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    plan = PA.plan_pages(ints(table.tolist()), ints(past.tolist()), ints(n.tolist()), ints(order[at:].tolist()), int(n.sum()) + pad, page)
    return plan, pages, oracle.plan(table, past, n, order[at:], int(n.sum()) + pad, page)


def randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


WRITES = [  # past, new, page, heads, head size, rows behind the last request
    ([0], [1], 8, 1, 8, 0), ([7, 8, 9], [1, 1, 1], 8, 2, 64, 0), ([0, 13, 100, 40], [30, 0, 1, 77], 16, 3, 128, 5),
    ([1560], [4680], 1560, 2, 128, 0), ([5] * 40, [1] * 40, 16, 8, 128, 3), ([0, 3], [300, 500], 40, 2, 40, 0), ([250], [20], 256, 1, 256, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("past,n,page,H,D,pad", WRITES)
def test_write(past, n, page, H, D, pad, dtype):
    plan, pages, (table, q_start, _, slots, _) = step(past, n, page, pad, seed=len(past))
    k, v = (randn((slots.shape[0], H, D), s, dtype) for s in (1, 2))
    kp, vp = (randn((pages, page, H, D), s, dtype) for s in (3, 4))
    means = randn((pages, H, D), 5, torch.float32)
    dk, dv, dm = kp.to(DEV), vp.to(DEV), means.to(DEV)
    PA.write_pages(k.to(DEV), v.to(DEV), dk, dv, plan, means=dm)
    wk, wv, wm = oracle.write(k, v, kp, vp, slots, table, torch.tensor(past), q_start, means)
    assert torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)
    # fp32 sums of up to `page` terms and one division: page + 1 roundings of at most 2^-24 of the sum of magnitudes, whose mean
    # is at most the largest key
    assert (dm.cpu().double() - wm).abs().max() <= (page + 1) * 2.0 ** -24 * wk.abs().max().double()
    touched = (wm - means.double()).abs().amax((1, 2)) > 0
    assert torch.equal(dm.cpu()[~touched], means[~touched])
    ek, ev = kp.to(DEV), vp.to(DEV)
    PA.write_pages(k.to(DEV), v.to(DEV), ek, ev, plan)
    assert torch.equal(ek, dk) and torch.equal(ev, dv)


def test_write_strided_rows_and_pools():
    plan, pages, (table, q_start, _, slots, _) = step([3, 20], [30, 9], 16, 2)
    T, H, D = slots.shape[0], 3, 64
    qkv = randn((T, 3, H, D), 1, torch.bfloat16).to(DEV)
    pools = randn((2, pages, H, 16, D), 2, torch.bfloat16).to(DEV)         # heads outside the rows of a page
    kp, vp = (p.transpose(1, 2) for p in pools)
    wk, wv, _ = oracle.write(qkv[:, 1].cpu(), qkv[:, 2].cpu(), kp.cpu(), vp.cpu(), slots, table, None, q_start)
    PA.write_pages(qkv[:, 1], qkv[:, 2], kp, vp, plan)
    assert torch.equal(kp.cpu(), wk) and torch.equal(vp.cpu(), wv)
    # rows of v in another layout than k's
    PA.write_pages(qkv[:, 2], qkv[:, 1].contiguous(), kp, vp, plan)
    wk, wv, _ = oracle.write(qkv[:, 2].cpu(), qkv[:, 1].cpu(), wk, wv, slots, table, None, q_start)
    assert torch.equal(kp.cpu(), wk) and torch.equal(vp.cpu(), wv)


def test_write_passes_over_slots_outside_the_pool():
    plan, pages, (table, q_start, _, slots, _) = step([3, 20], [30, 9], 16, 2)
    bad = slots.clone()
    bad[::3] = torch.tensor([-1, -7, pages * 16, 2 ** 40, -2 ** 40])[torch.arange(len(bad[::3])) % 5]
    k, v = (randn((slots.shape[0], 2, 64), s, torch.float16) for s in (1, 2))
    kp, vp = (randn((pages, 16, 2, 64), s, torch.float16) for s in (3, 4))
    dk, dv = kp.to(DEV), vp.to(DEV)
    PA.write_pages(k.to(DEV), v.to(DEV), dk, dv, plan._replace(slots=bad.to(DEV)))
    wk, wv, _ = oracle.write(k, v, kp, vp, bad, table, None, q_start)
    assert torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)


def test_write_means_of_pages_outside_the_pool_are_not_formed():
    plan, pages, (table, q_start, _, slots, _) = step([3, 20], [30, 9], 16, 2)
    table = table.clone()
    table[0, 1], table[1, 1] = pages, -5
    k, v = (randn((slots.shape[0], 2, 64), s, torch.float16) for s in (1, 2))
    kp, vp = (randn((pages, 16, 2, 64), s, torch.float16) for s in (3, 4))
    means = randn((pages, 2, 64), 5, torch.float32)
    dk, dv, dm = kp.to(DEV), vp.to(DEV), means.to(DEV)
    PA.write_pages(k.to(DEV), v.to(DEV), dk, dv, plan._replace(table=ints(table.tolist())), means=dm)
    _, _, wm = oracle.write(k, v, kp, vp, slots, table, torch.tensor([3, 20]), q_start, means)
    assert (dm.cpu().double() - wm).abs().max() <= 17 * 2.0 ** -24 * max(k.abs().max(), kp.abs().max()).double()


# ---------------------------------------------------------------- select
SELECTS = [  # past, new, page, heads, kv heads, head size, top, group, first, last, causal, rows behind
    ([0], [1], 8, 1, 1, 64, 1, 1, 0, 0, True, 0), ([500], [1], 8, 4, 2, 128, 5, 1, 1, 1, True, 0), ([500], [1], 8, 4, 4, 128, 64, 1, 1, 1, True, 0),
    ([500], [1], 8, 4, 4, 128, 63, 1, 0, 0, True, 2), ([100, 0, 700, 900], [1, 1, 1, 1], 16, 6, 2, 64, 9, 1, 1, 1, True, 0),
    ([100, 0, 700, 300], [37, 0, 200, 1], 16, 6, 2, 64, 9, 16, 1, 2, True, 9), ([0, 300], [300, 65], 8, 2, 2, 128, 7, 64, 0, 1, True, 0),
    ([0, 300], [300, 65], 8, 2, 1, 128, 7, 100, 1, 0, False, 0), ([2000], [20], 8, 2, 2, 40, 200, 3, 1, 1, False, 0), ([900], [5], 8, 2, 2, 256, 12, 2, 2, 2, True, 0),
]


def select_inputs(past, n, page, H, Hk, D, pad, dtype, seed=0):
    plan, pages, (table, q_start, *_rest) = step(past, n, page, pad, seed)
    q = randn((sum(n) + pad, H, D), 11, dtype)
    means = randn((pages, Hk, D), 12, torch.float32)
    return plan, pages, table, q_start, q, means


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("past,n,page,H,Hk,D,top,group,first,last,causal,pad", SELECTS)
def test_select(past, n, page, H, Hk, D, top, group, first, last, causal, pad, dtype):
    plan, pages, table, q_start, q, means = select_inputs(past, n, page, H, Hk, D, pad, dtype)
    got = PA.select_pages(q.to(DEV), means.to(DEV), plan, top, group=group, causal=causal, first=first, last=last)
    want = oracle.select_pages(q, means, table, torch.tensor(past), q_start, page, top, group, causal, first, last)
    assert torch.equal(got.cpu().long(), want)


@pytest.mark.parametrize("pages_of", [2047, 2048, 2049, 4100, 9000])
@pytest.mark.parametrize("top", [1, 64, 2048])
def test_select_from_long_tables(pages_of, top):
    plan, pages, table, q_start, q, means = select_inputs([pages_of * 8 - 1, 400], [1, 1], 8, 2, 1, 64, 0, torch.bfloat16)
    got = PA.select_pages(q.to(DEV), means.to(DEV), plan, top, causal=True, first=0, last=1)
    x = q[0].double().sum(0)
    s = means[table[0, :pages_of], 0].double() @ x
    s[-1] = float("inf")
    want = torch.sort(torch.sort(s, descending=True, stable=True)[1][:top])[0]
    assert torch.equal(got[0, 0, :len(want)].cpu().long(), want) and bool((got[0, 0, len(want):] == -1).all())


def test_select_level_and_odd_scores():
    """Level scores go to the lower page, -0 is 0, NaN and pages outside the pool come last, infinities first."""
    plan, pages, table, q_start, q, means = select_inputs([400, 400], [1, 1], 8, 2, 1, 64, 0, torch.bfloat16)
    means[:, 0] = torch.randint(-1, 2, (pages, 1), generator=torch.Generator().manual_seed(3)).float() * torch.ones(64)
    means[table[0, 5], 0, 0], means[table[0, 6], 0, 0], means[table[0, 9]] = float("nan"), float("inf"), -0.0
    table = table.clone()
    table[1, 7], table[1, 8] = -1, pages
    plan = plan._replace(table=ints(table.tolist()))
    for top in (1, 2, 5, 20, 40, 49):
        got = PA.select_pages(q.to(DEV), means.to(DEV), plan, top, causal=True, first=0, last=0)
        want = oracle.select_pages(q, means, table, torch.tensor([400, 400]), q_start, 8, top, 1, True, 0, 0)
        assert torch.equal(got.cpu().long(), want), top


def test_select_strided_queries_and_table():
    plan, pages, table, q_start, q, means = select_inputs([300, 70], [5, 9], 8, 4, 2, 64, 3, torch.bfloat16)
    wide = torch.full((2, table.shape[1] + 3), 10 ** 6, dtype=torch.int32, device=DEV)
    wide[:, :-3] = plan.table
    big = torch.zeros((q.shape[0], 2, 4, 64), dtype=q.dtype, device=DEV)
    big[:, 1] = q.to(DEV)
    got = PA.select_pages(big[:, 1], means.to(DEV), plan._replace(table=wide[:, :-3]), 6, group=2, causal=True)
    assert torch.equal(got.cpu().long(), oracle.select_pages(q, means, table, torch.tensor([300, 70]), q_start, 8, 6, 2, True, 1, 1))


def passes(rows, Hk, W, D):
    """Scores of so many rows are formed at a time in 256 MB."""
    return -(-rows // max(1, min(2 ** 28 // (8 * Hk * (W + D)), 65535)))


@pytest.mark.parametrize("H,group,width,least", [(2, 1, 60000, 4), (4, 20, 2 ** 20, 4), (2, 7, 400000, 4)])
@pytest.mark.parametrize("causal", [False, True])
def test_select_in_several_passes(H, group, width, least, causal):
    """More rows than a pass holds, by a table wide with entries of nobody: tiles of four rows and requests go on in the next pass, queries
    summed by whom they are for (group * heads to a key head up to 16) and beforehand."""
    past, n, page, Hk, D, pad = [90, 300, 4], [3, 700, 500], 8, 2, 16, 41
    plan, pages, table, q_start, q, means = select_inputs(past, n, page, H, Hk, D, pad, torch.bfloat16)
    rows = PA.selected_rows(sum(n) + pad, 3, group)
    assert passes(rows, Hk, width, D) >= least and passes(rows, Hk, table.shape[1], D) == 1
    wide = torch.full((3, width), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = plan.table
    got = PA.select_pages(q.to(DEV), means.to(DEV), plan._replace(table=wide), 9, group=group, causal=causal)
    assert torch.equal(got, PA.select_pages(q.to(DEV), means.to(DEV), plan, 9, group=group, causal=causal))
    assert torch.equal(got.cpu().long(), oracle.select_pages(q, means, table, torch.tensor(past), q_start, page, 9, group, causal, 1, 1))


def test_select_for_more_rows_than_a_pass_takes():
    """A pass ends at 65535 rows too: 50000 requests of a token, against themselves in parts of one pass."""
    R, page, D = 50000, 8, 8
    g = torch.Generator().manual_seed(5)
    past, order = torch.randint(0, 150, (R,), generator=g), torch.randint(0, 997, (R, 19), generator=g).int()
    plan = PA.plan_pages(order.to(DEV), ints(past.tolist()), ints([1] * R), ints(list(range(997)) * 30), R, page)
    q, means = randn((R, 2, D), 1, torch.bfloat16).to(DEV), randn((997, 2, D), 2, torch.float32).to(DEV)
    assert passes(PA.selected_rows(R, R, 1), 2, 19, D) == 2
    got = PA.select_pages(q, means, plan, 4, causal=True)
    assert got.shape[0] == 2 * R + 1
    for at in range(0, R, 12500):
        part = slice(at, at + 12500)
        own = PA.PagePlan(plan.table[part], plan.past[part], plan.lengths[part], torch.arange(12501, dtype=torch.int32, device=DEV), plan.slots[part],
                          plan.next_free, page)
        want = PA.select_pages(q[part], means, own, 4, causal=True)
        assert torch.equal(got[2 * at:2 * (at + 12500)], want[:-1])
    few = torch.arange(0, R, 5003)                         # and a few of them against the oracle
    for r in few.tolist():
        want = oracle.select_pages(q[r:r + 1].cpu(), means.cpu(), plan.table[r:r + 1].cpu(), past[r:r + 1], torch.tensor([0, 1]), page, 4, 1, True, 1, 1)
        assert torch.equal(got[2 * r].cpu().long(), want[0])
    assert bool((got[1::2] == -1).all())                   # rows that nobody has


@pytest.mark.parametrize("group,page", [(1, 8), (7, 8), (8, 8), (9, 8), (10, 8), (40, 16), (128, 64), (33, 1560)])
def test_last_pages_of_a_group_hold_every_tokens_own(group, page):
    past, n, Hk = [3 * page - 1, 5], [2 * group + 3, group], 2
    plan, pages, table, q_start, q, means = select_inputs(past, n, page, 2, Hk, 64, 0, torch.bfloat16)
    last = (group + page - 2) // page + 1
    for more in (0, -1):
        got = PA.select_pages(q.to(DEV), means.to(DEV), plan, last + 1, group=group, causal=True, first=0, last=last + more)
        assert torch.equal(got.cpu().long(), oracle.select_pages(q, means, table, torch.tensor(past), q_start, page, last + 1, group, True, 0, last + more))
    got, own = PA.select_pages(q.to(DEV), means.to(DEV), plan, last, group=group, causal=True, first=0, last=last).cpu(), []
    for r in range(2):
        for t in range(n[r]):
            row = got[int(q_start[r]) // group + r + t // group]
            own.append(bool((row == (past[r] + t) // page).any(1).all()))
    assert all(own)
