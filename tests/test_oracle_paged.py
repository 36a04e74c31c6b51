"""What pins the paged cache's oracle: the library's attention on a cache in order, and the rules' own words in scalar loops."""
import math

import pytest
import torch

from oracle import paged


def in_order(past, n, page, Hk, D, seed=0):
    """One request whose pages lie one after the other."""
    g = torch.Generator().manual_seed(seed)
    whole = -(-(past + n) // page)
    kp, vp = (torch.randn((whole, page, Hk, D), generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.arange(whole)[None]
    return kp, vp, table, torch.tensor([past]), torch.tensor([0, n])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("past,n,page,H,Hk", [(0, 1, 8, 1, 1), (13, 9, 8, 4, 2), (40, 17, 16, 6, 3)])
def test_attention_is_the_librarys_on_a_cache_in_order(past, n, page, H, Hk, causal):
    kp, vp, table, p, qs = in_order(past, n, page, Hk, 8)
    q = torch.randn((n, H, 8), dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    k, v = (x.view(-1, Hk, 8)[:past + n].transpose(0, 1).repeat_interleave(H // Hk, 0) for x in (kp, vp))
    mask = torch.ones(n, past + n, dtype=torch.bool)
    if causal:
        mask = mask.tril(past)
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1), k, v, attn_mask=mask).transpose(0, 1)
    got = paged.attention(q, kp, vp, table, p, qs, causal=causal)
    assert (got["out"] - want).abs().max() < 1e-12
    s = (q.transpose(0, 1) @ k.transpose(1, 2) * 8 ** -0.5).masked_fill(~mask, -math.inf)
    assert (got["lse"] - torch.logsumexp(s, -1)).abs().max() < 1e-12
    assert torch.equal(got["keys"][:, 0], mask.sum(1))


def test_attention_follows_the_table():
    kp, vp, table, p, qs = in_order(30, 5, 8, 2, 8)
    q = torch.randn((5, 2, 8), dtype=torch.float64)
    want = paged.attention(q, kp, vp, table, p, qs, causal=True)
    order = torch.tensor([3, 0, 4, 1, 2])
    moved_k, moved_v = torch.empty_like(kp), torch.empty_like(vp)
    moved_k[order], moved_v[order] = kp, vp
    got = paged.attention(q, moved_k, moved_v, order[None], p, qs, causal=True)
    assert torch.equal(got["out"], want["out"])


@pytest.mark.parametrize("window,sink", [(1, 0), (5, 2), (9, 30), (100, 0)])
def test_window_and_sink(window, sink):
    kp, vp, table, p, qs = in_order(20, 6, 8, 1, 8)
    q = torch.randn((6, 1, 8), dtype=torch.float64)
    got = paged.attention(q, kp, vp, table, p, qs, causal=True, window=window, sink=sink)
    k, v = kp.view(-1, 8), vp.view(-1, 8)
    for i in range(6):
        seen = [j for j in range(26) if j <= 20 + i and (j > 20 + i - window or j < sink)]
        w = [math.exp(float(q[i, 0] @ k[j]) * 8 ** -0.5) for j in seen]
        want = sum(x * v[j] for x, j in zip(w, seen)) / sum(w)
        assert (got["out"][i, 0] - want).abs().max() < 1e-12 and got["keys"][i, 0] == len(seen)


def test_selected_pages_are_a_mask():
    kp, vp, table, p, qs = in_order(37, 4, 8, 1, 8)
    q = torch.randn((4, 1, 8), dtype=torch.float64)
    sel = torch.tensor([[[1, 3, -1]], [[0, 5, -1]], [[-1, -1, -1]], [[-1, -1, -1]]])
    got = paged.attention(q, kp, vp, table, p, qs, causal=True, selected=sel, group=2)
    for i in range(4):
        seen = [j for j in range(38 + i) if j // 8 in sel[i // 2, 0].tolist()]
        w = torch.softmax(torch.stack([q[i, 0] @ kp.view(-1, 8)[j] for j in seen]) * 8 ** -0.5, 0)
        assert (got["out"][i, 0] - sum(x * vp.view(-1, 8)[j] for x, j in zip(w, seen))).abs().max() < 1e-12


def test_plan_and_write():
    """Every new token's row comes to lie where the table says its position is; tokens before the step keep theirs."""
    past, new, page = torch.tensor([0, 5, 16]), torch.tensor([9, 0, 3]), 8
    table = torch.tensor([[-1, -1, -1], [7, -1, -1], [2, 9, -1]])
    t, qs, lens, slots, nf = paged.plan(table, past, new, [4, 0, 8, 1], 14, page, next_free=1)
    assert t.tolist() == [[0, 8, -1], [7, -1, -1], [2, 9, 1]] and qs.tolist() == [0, 9, 9, 12] and lens.tolist() == [9, 5, 19] and nf == 4
    assert slots.tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 64, 8, 9, 10, -1, -1]
    k = torch.arange(14.)[:, None, None].expand(14, 1, 2)
    kp = torch.full((10, page, 1, 2), -1.0)
    wk, wv, m = paged.write(k, k + 100, kp, kp, slots, t, past, qs, torch.zeros(10, 1, 2))
    for r in range(3):
        for i in range(int(new[r])):
            pos = int(past[r]) + i
            assert (wk[t[r, pos // page], pos % page] == int(qs[r]) + i).all() and (wv[t[r, pos // page], pos % page] == 100 + int(qs[r]) + i).all()
    assert (wk == -1).sum() == wk.numel() - 2 * 12
    assert m[0, 0, 0] == 3.5 and m[8, 0, 0] == 8 and m[1, 0, 0] == 10 and m[9, 0, 0] == 0 and m[7, 0, 0] == 0


def test_select_takes_the_largest_scores_and_the_lower_of_level_ones():
    means = torch.tensor([[[1.0, 0]], [[3.0, 0]], [[3.0, 0]], [[2.0, 0]], [[9.0, 0]]])
    q = torch.tensor([[[1.0, 0]]])
    args = (q, means, torch.tensor([[0, 1, 2, 3, 4]]), torch.tensor([31]), torch.tensor([0, 1]), 8)
    pick = lambda top, first, last: paged.select_pages(*args, top, 1, True, first, last)[0, 0].tolist()
    assert pick(1, 0, 0) == [1] and pick(2, 0, 0) == [1, 2] and pick(3, 0, 0) == [1, 2, 3]          # page 4 is not seen
    assert pick(2, 1, 0) == [0, 1] and pick(2, 1, 1) == [0, 3] and pick(6, 0, 0) == [0, 1, 2, 3, -1, -1]
