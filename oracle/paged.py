"""The paged cache's operators restated on the CPU, request by request, in float64.

Positions of a request lie in pages: row r of the block table names the page of each page_size consecutive ones.  `past` tokens
of a request are in the cache before a step, `new` of them come with it."""
import math

import torch


def plan(table, past, new, free, tokens, page_size, next_free=0):
    """(table, q_start, lengths, slots, next_free): what plan_pages leaves, as int64 tensors."""
    table = table.clone().long()
    W, at, next_free = table.shape[1], 0, max(int(next_free), 0)
    q_start, lengths, slots = [0], [], []
    for r in range(table.shape[0]):
        p, n = max(int(past[r]), 0), min(max(int(new[r]), 0), tokens - at)
        for e in range(min(W, -(-p // page_size)), min(W, -(-(p + n) // page_size))):
            table[r, e] = int(free[next_free]) if next_free < len(free) else -1
            next_free += 1
        for pos in range(p, p + n):
            page = int(table[r, pos // page_size]) if pos // page_size < W else -1
            slots.append(page * page_size + pos % page_size if page >= 0 else -1)
        at += n
        q_start.append(at)
        lengths.append(p + n)
    slots += [-1] * (tokens - at)
    return table, torch.tensor(q_start), torch.tensor(lengths), torch.tensor(slots, dtype=torch.long), next_free


def write(k, v, k_pages, v_pages, slots, table, past, q_start, means=None):
    """In place on clones: (k_pages, v_pages, means)."""
    k_pages, v_pages = k_pages.clone(), v_pages.clone()
    N, P = k_pages.shape[:2]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < N * P:
            k_pages[s // P, s % P], v_pages[s // P, s % P] = k[t], v[t]
    if means is not None:
        means = means.double().clone()
        for r in range(table.shape[0]):
            p, n = max(int(past[r]), 0), int(q_start[r + 1] - q_start[r])
            for e in range(p // P, -(-(p + n) // P)) if n else ():
                page = int(table[r, e]) if e < table.shape[1] else -1
                if 0 <= page < N:
                    means[page] = k_pages[page, :min(P, p + n - e * P)].double().mean(0)
    return k_pages, v_pages, means


def attention(q, k_pages, v_pages, table, past, q_start, sm_scale=None, causal=False, window=None, sink=0, selected=None, group=1):
    """dict of out [T, H, D] and lse [H, T]; mag: sum of weight * |v|; slip: how far fp32 sums of the products may move a logit, as a
    bound on its error in units of 2^-24; keys: number of visible positions; top: their largest |v|; bad: the row would read a position
    without a page (all of these [T, H])."""
    T, H, D = q.shape
    N, P, Hk = k_pages.shape[:3]
    W, G, R = table.shape[1], H // Hk, table.shape[0]
    scale = D ** -0.5 if sm_scale is None else sm_scale
    out, mag = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    lse, slip = torch.full((H, T), -math.inf, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    top = torch.zeros(T, H, dtype=torch.float64)
    keys, bad = torch.zeros(T, H, dtype=torch.long), torch.zeros(T, H, dtype=torch.bool)
    for r in range(R):
        first, n, p = int(q_start[r]), int(q_start[r + 1] - q_start[r]), max(int(past[r]), 0)
        L = p + n
        for i in range(n):
            end = p + i + 1 if causal else L
            for kh in range(Hk):
                if selected is None:
                    pos = range(end)
                    if window is not None:
                        pos = sorted(set(range(max(0, end - window), end)) | set(range(min(sink, end))))
                else:
                    row = selected[first // group + r + i // group, kh].tolist()
                    pos = [e * P + j for e in row[:row.index(-1) if -1 in row else len(row)] for j in range(P) if e * P + j < end]
                pos = torch.tensor(list(pos), dtype=torch.long)
                t, hs = first + i, slice(kh * G, (kh + 1) * G)
                entry = pos // P
                page = torch.where(entry < W, table[r].long()[entry.clamp(max=W - 1)], -1)
                if ((page < 0) | (page >= N)).any():
                    bad[t, hs] = True
                    continue
                keys[t, hs] = len(pos)
                if not len(pos):
                    continue
                k, v = k_pages[page, pos % P, kh].double(), v_pages[page, pos % P, kh].double()
                x = q[t, hs].double() @ k.T * scale
                slip[t, hs] = (q[t, hs].double().abs() @ k.abs().T * scale).max(1)[0] * (D + 4) + x.abs().max(1)[0] * 4 + 16
                lse[hs, t] = torch.logsumexp(x, 1)
                w = torch.exp(x - lse[hs, t, None])
                out[t, hs], mag[t, hs], top[t, hs] = w @ v, w @ v.abs(), v.abs().max()
    return dict(out=out, lse=lse, mag=mag, slip=slip, keys=keys, top=top, bad=bad)


def select_pages(q, means, table, past, q_start, page_size, top, group=1, causal=False, first=1, last=1):
    """Entries that each group of tokens reads, [T // group + R + 1, Hk, top], -1 behind them."""
    T, H, D = q.shape
    N, Hk = means.shape[:2]
    R, W, G = table.shape[0], table.shape[1], H // Hk
    out = torch.full((T // group + R + 1, Hk, top), -1, dtype=torch.long)
    for r in range(R):
        start, n, p = int(q_start[r]), int(q_start[r + 1] - q_start[r]), max(int(past[r]), 0)
        for g, t0 in enumerate(range(0, n, group)):
            t1 = min(n, t0 + group)
            pages = -(-(p + t1 if causal else p + n) // page_size)
            x = q[start + t0:start + t1].double().sum(0).view(Hk, G, D).sum(1)
            for kh in range(Hk):
                score = []
                for e in range(min(pages, W)):
                    page = int(table[r, e])
                    s = float(x[kh] @ means[page, kh].double()) if 0 <= page < N else -math.inf
                    s = -math.inf if math.isnan(s) else s
                    score.append(math.inf if e < first or e >= pages - last else s)
                best = sorted(range(len(score)), key=lambda e: (-score[e], e))[:top]
                out[start // group + r + g, kh, :len(best)] = torch.tensor(sorted(best), dtype=torch.long)
    return out
