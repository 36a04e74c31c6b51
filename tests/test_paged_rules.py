"""Arithmetic of the paged cache's kernels (csrc/paged_rules.hpp), compiled for the host."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "paged_rules.hpp"
extern "C" unsigned quotient(unsigned n, unsigned d) { return sfm::quot(n, sfm::fast_div(d)); }
extern "C" void request(const int* q_start, const int* past, int r, int R, int T, int* out) {
    const sfm::Request q = sfm::request_of(q_start, past, r, R, T);
    out[0] = q.first; out[1] = q.n; out[2] = q.past;
}
extern "C" long long piece(long long start, long long heads, long long per, int r) { return sfm::first_piece(start, heads, per, r); }
extern "C" long long all_pieces(long long rows, long long per, int R) { return sfm::pieces(rows, per, R); }
extern "C" void tiles(int past, int n, int none, int t0, int t1, int causal, int window, int sink, int cap, int* out) {
    const sfm::Request q{0, n, past};
    const sfm::KeyTiles k = sfm::key_tiles(q, none, t0, t1, causal, window, sink, cap);
    const int v[] = {k.end_min, k.end_max, k.lo_min, k.lo_max, k.sinks, k.first, k.tiles, k.fast0, k.fast1, k.beyond};
    for (int i = 0; i < 10; ++i) out[i] = v[i];
}
extern "C" long long most(long long rows, long long heads, long long tokens, int causal, long long window, long long sink, long long cap) {
    return sfm::most_tiles(rows, heads, tokens, causal, window, sink, cap);
}
static sfm::Rows3 rows3(long long bytes, const long long* n, const long long* stride) {
    return {nullptr, bytes, {n[0], n[1], n[2]}, {stride[0], stride[1], stride[2]}};
}
extern "C" int meets(long long ab, const long long* an, const long long* as, long long bb, const long long* bn, const long long* bs, long long x) {
    return sfm::meet(rows3(ab, an, as), rows3(bb, bn, bs), x);
}
extern "C" int folded(long long bytes, const long long* n, const long long* stride) { return sfm::folds(rows3(bytes, n, stride)); }
extern "C" int paired(int i, int n, int place) { return place ? sfm::paired_place(i, n) : sfm::paired_piece(i, n); }
"""


SOURCE += """
extern "C" long long block(int past, int n, int t0, int t1, int causal, int window, int sink, int cap, const int* table, int width, int pages,
                           int page_size, const int* sel, int count, long long page_bytes, long long row_bytes, int vb, int* pos, int* entry, int* page) {
    sfm::KeyTiles k = sfm::key_tiles(sfm::Request{0, n, past}, false, t0, t1, causal, window, sink, cap);
    if (sel) { k.sinks = k.first = 0; k.tiles = (int)(((long long)count * page_size + 63) / 64); }
    sfm::BlockMap b{table, sel, k.tiles * 8, count, k.sinks * 8, (k.first - k.sinks) * 8, k.end_max, k.lo_min, sink, width, pages, sfm::fast_div(page_size / 8),
                    page_bytes, 8 * row_bytes};
    unsigned off8;
    *entry = b.entry(vb, &off8, pos);
    *page = b.page(*entry);
    return b.offset(*page, off8);
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.hip").write_text(SOURCE)
    csrc = os.path.join(ROOT, "self-forcing_amd", "csrc")
    subprocess.run([hipcc, "--offload-host-only", "-std=c++17", "-shared", "-fPIC", "-I" + csrc, "-I" + os.path.join(ROOT, "include"),
                    str(d / "rules.hip"), "-o", str(d / "rules.so")], check=True, capture_output=True)
    lib = C.CDLL(str(d / "rules.so"))
    lib.quotient.restype = C.c_uint
    lib.piece.restype = lib.all_pieces.restype = C.c_longlong
    lib.piece.argtypes = [C.c_longlong] * 3 + [C.c_int]
    lib.block.restype = C.c_longlong
    lib.block.argtypes = [C.c_int] * 8 + [C.c_void_p] + [C.c_int] * 3 + [C.c_void_p, C.c_int] + [C.c_longlong] * 2 + [C.c_int] + [C.c_void_p] * 3
    lib.all_pieces.argtypes = [C.c_longlong] * 2 + [C.c_int]
    lib.most.restype = C.c_longlong
    lib.meets.argtypes = [C.c_longlong, C.c_void_p, C.c_void_p] * 2 + [C.c_longlong]
    lib.folded.argtypes = [C.c_longlong, C.c_void_p, C.c_void_p]
    lib.most.argtypes = [C.c_longlong] * 3 + [C.c_int] + [C.c_longlong] * 3
    return lib


def test_quotients(rules):
    rng = random.Random(1)
    top = 2 ** 28 - 1
    for d in [1, 2, 3, 5, 7, 8, 195, 2 ** 14 - 1, 2 ** 20 + 1, 2 ** 27 + 1, 2 ** 28 - 1] + [rng.randint(1, top) for _ in range(300)]:
        near = [k * d + e for k in (1, 2, 3, top // d) for e in (-1, 0, 1)]
        for n in [0, 1, d, top, top - 1] + near + [rng.randint(0, top) for _ in range(60)]:
            if 0 <= n <= top:
                assert rules.quotient(n, d) == n // d, (n, d)


def test_pieces_are_every_row_once(rules):
    rng = random.Random(2)
    for _ in range(200):
        R, per, heads = rng.randint(1, 40), rng.choice([1, 2, 7, 32, 128, 256]), rng.choice([1, 3, 8])
        n = [rng.choice([0, 1, 1, rng.randint(0, 300)]) for _ in range(R + 1)]          # the last: rows of nobody
        start, at = [], 0
        for m in n:
            start.append(at)
            at += m
        taken = set()
        for r, m in enumerate(n):
            first = rules.piece(start[r], heads, per, r)
            own = range(first, first - (-m * heads // per))
            assert not taken & set(own)
            taken |= set(own)
            assert r == R or rules.piece(start[r + 1], heads, per, r + 1) >= first + len(own)
            assert first + len(own) <= rules.all_pieces(at * heads, per, R)


def test_requests_stay_inside_the_rows(rules):
    rng = random.Random(3)
    odd = [0, 1, 5, 100, -1, -2 ** 31, 2 ** 31 - 1, 101]
    for _ in range(500):
        R, T = 3, 100
        qs, ps = [rng.choice(odd) for _ in range(R + 1)], [rng.choice(odd) for _ in range(R)]
        for r in range(R + 1):
            out = (C.c_int * 3)()
            rules.request((C.c_int * (R + 1))(*qs), (C.c_int * R)(*ps), r, R, T, out)
            assert 0 <= out[0] <= T and 0 <= out[1] <= T - out[0] and out[2] >= 0


@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 55, 56, 64, 1001])
def test_paired_pieces_are_every_piece_once(rules, n):
    pieces = [rules.paired(i, n, 0) for i in range(n)]
    assert sorted(pieces) == list(range(n)) and pieces[:3] == [n - 1, 0, n - 2][:n]
    places = [rules.paired(i, n, 1) for i in range(n)]
    assert sorted(places) == list(range(n)) and places == sorted(range(n), key=lambda i: (i % 2, i))


def visible(past, n, t, causal, window, sink, cap):
    end = past + t + 1 if causal else past + n
    end = min(end, cap)
    return {p for p in range(end) if not window or p >= end - window or p < sink}


def test_tiles_hold_what_a_piece_sees_and_fast_ones_nothing_else(rules):
    rng = random.Random(4)
    for _ in range(3000):
        past, n, causal = rng.choice([0, 1, 63, 64, 65, 500, rng.randint(0, 900)]), rng.randint(1, 300), rng.randint(0, 1)
        t0 = rng.randint(0, n - 1)
        t1 = rng.randint(t0, min(n - 1, t0 + 255))
        window = rng.choice([0, 1, 64, 100, rng.randint(1, 700), 5000])
        sink = rng.choice([0, 1, 64, rng.randint(0, 400)]) if window else 0
        cap = rng.choice([10 ** 6, 8 * rng.randint(1, 100)])
        out = (C.c_int * 10)()
        rules.tiles(past, n, 0, t0, t1, causal, window, sink, cap, out)
        end_min, end_max, lo_min, lo_max, sinks, first, count, fast0, fast1, beyond = out
        assert bool(beyond) == ((past + t1 + 1 if causal else past + n) > cap)
        seen = [visible(past, n, t, causal, window, sink, cap) for t in range(t0, t1 + 1)]
        order = [v if v < sinks else v - sinks + first for v in range(count)]
        assert order == sorted(set(order))
        covered = {p for i in order for p in range(64 * i, 64 * i + 64)}
        assert set().union(*seen) <= covered
        assert 0 <= fast0 <= fast1 <= count
        for v in range(fast0, fast1):
            assert all(set(range(64 * order[v], 64 * order[v] + 64)) <= s for s in seen)
        for t, s in zip(range(t0, t1 + 1), seen):          # the mask that a kernel takes from a row's own end
            end = min(past + t + 1 if causal else past + n, cap)
            lo = max(0, end - window) if window else 0
            assert s == {p for p in covered if p < end and (p >= lo or p < sink)}
            assert end_min <= end <= end_max and lo_min <= lo <= lo_max
    rules.tiles(9, 5, 1, 0, 4, 1, 0, 0, 100, out)
    assert out[6] == 0                                     # rows of nobody


@pytest.mark.parametrize("listed", [False, True])
def test_blocks_lie_where_the_table_says_and_always_inside_the_pool(rules, listed):
    rng = random.Random(5)
    odd = [-1, -2 ** 31, 2 ** 31 - 1]
    for _ in range(800):
        page = 8 * rng.choice([1, 2, 3, 5, 8, 195])
        past, n, causal = rng.randint(0, 900), rng.randint(1, 200), rng.randint(0, 1)
        t0 = rng.randint(0, n - 1)
        t1 = rng.randint(t0, n - 1)
        window = 0 if listed else rng.choice([0, 1, 64, rng.randint(1, 700)])
        sink = rng.randint(0, 300) if window else 0
        need = -(-(past + n) // page)
        width, pages = max(1, need + rng.choice([0, 1, -1])), rng.randint(1, 2 * need + 2)
        table = [rng.choice([rng.randrange(pages), rng.randrange(pages), rng.randrange(pages), rng.choice(odd + [pages])]) for _ in range(width)]
        cap = width * page
        sel = sorted(rng.sample(range(need), rng.randint(0, need))) if listed else None
        if listed and rng.random() < 0.3:
            sel = [rng.choice([rng.randrange(need), rng.randint(0, 2 ** 31 - 1)]) for _ in range(rng.randint(1, 9))]
        row_bytes = 16 * rng.randint(1, 40)
        page_bytes = page * row_bytes + 16 * rng.randint(0, 3)
        ctable, csel = (C.c_int * width)(*table), (C.c_int * max(1, len(sel or [])))(*(sel or [])) if listed else None
        pos, entry, number = C.c_int(), C.c_int(), C.c_int()
        out = (C.c_int * 10)()
        rules.tiles(past, n, 0, t0, t1, causal, window, sink, cap, out)
        some = {p for t in range(t0, t1 + 1) for p in visible(past, n, t, causal, window, sink, cap)}
        blocks = 8 * (-(-len(sel) * page // 64) if listed else out[6])
        met = set()
        for vb in [*range(blocks + 3), 2 ** 31 - 8]:
            off = rules.block(past, n, t0, t1, causal, window, sink, cap, ctable, width, pages, page, csel, len(sel or []), page_bytes, row_bytes, vb,
                              C.byref(pos), C.byref(entry), C.byref(number))
            assert 0 <= off <= (pages - 1) * page_bytes + (page - 8) * row_bytes      # eight rows from there are a page's
            own = set(range(pos.value, pos.value + 8)) if pos.value < 2 ** 31 - 8 else set()
            if entry.value >= 0:
                assert own and pos.value % 8 == 0 and entry.value == pos.value // page
                p = table[entry.value]
                assert number.value == (p if 0 <= p < pages else -1)
                if number.value >= 0:
                    assert off == p * page_bytes + pos.value % page * row_bytes
                assert listed or not own & met
                met |= own & some
            elif own:
                assert not own & some                          # skipped: nobody sees it
        if not listed:
            assert met == some
        elif sel == sorted(set(sel)) and (not sel or sel[-1] < need):
            assert met == {p for p in some if p // page in sel}


def test_no_piece_has_more_tiles_than_the_ranges_are_made_for(rules):
    rng = random.Random(6)
    reached = 0
    for _ in range(4000):
        heads, rows = rng.choice([1, 2, 3, 5, 8, 40]), rng.choice([4, 32, 128, 256])
        past, n, causal = rng.choice([0, 1, 63, 64, 65, 500, rng.randint(0, 5000)]), rng.choice([1, 2, rng.randint(1, 700)]), rng.randint(0, 1)
        window = rng.choice([0, 1, 2, 63, 64, 65, 66, rng.randint(1, 900), 2 ** 31 - 1])
        sink = rng.choice([0, 1, 64, 65, rng.randint(0, 900), 2 ** 31 - 1]) if window else 0
        cap = rng.choice([past + n, 10 ** 6, 2 ** 30, 8 * rng.randint(1, 600)])
        most = rules.most(rows, heads, n + rng.choice([0, 0, 100]), causal, window, sink, cap)
        assert most <= -(-cap // 64) and (window or most == -(-cap // 64))
        row0 = rng.randint(0, n * heads - 1)                # a piece may begin at any row of a token
        row1 = min(n * heads, row0 + rows)
        out = (C.c_int * 10)()
        rules.tiles(past, n, 0, row0 // heads, (row1 - 1) // heads, causal, window, sink, cap, out)
        assert out[6] <= most
        reached += window > 0 and out[6] == most
    assert reached > 100                                   # and some have as many


def test_rows_that_share_bytes(rules):
    """Never missed; and rows whose strides nest, as those of tensors and of their slices do, are told apart exactly."""
    rng = random.Random(8)

    def where(n, stride, w):
        return [a * stride[0] + b * stride[1] + c * stride[2] for a in range(n[0]) for b in range(n[1]) for c in range(n[2])]

    def nested(fused):
        """A slice of a buffer: counts, strides and offset of its rows, in any order of the dimensions."""
        n, stride, at, size = [], [], 0, fused["w"]
        for most in fused["n"]:
            m = rng.randint(1, most)
            at += rng.randint(0, most - m) * size
            n.append(m)
            stride.append(size)
            size *= most
        order = rng.sample(range(3), 3)
        return [n[i] for i in order], [stride[i] for i in order], at
    ll3 = C.c_longlong * 3
    seen = [0, 0]
    for i in range(4000):
        if i % 2:
            fused = dict(w=rng.randint(1, 5), n=[rng.randint(1, 4) for _ in range(3)])
            (an, as_, a), (bn, bs, b), w = nested(fused), nested(fused), fused["w"]
            bw, x = w, b - a
        else:
            an, bn = ([rng.randint(1, 4) for _ in range(3)] for _ in range(2))
            as_, bs = ([rng.randint(0, 40) for _ in range(3)] for _ in range(2))
            w, bw, x = rng.randint(1, 5), rng.randint(1, 5), rng.randint(-200, 200)
        mine = {p + k for p in where(an, as_, w) for k in range(w)}
        share = bool(mine & {x + p + k for p in where(bn, bs, bw) for k in range(bw)})
        got = bool(rules.meets(w, ll3(*an), ll3(*as_), bw, ll3(*bn), ll3(*bs), x))
        assert got or not share
        if i % 2:
            assert got == share
            seen[share] += 1
        if all(s >= w for s in as_):
            twice = len(mine) < w * an[0] * an[1] * an[2]
            assert rules.folded(w, ll3(*an), ll3(*as_)) or not twice
            assert not i % 2 or not rules.folded(w, ll3(*an), ll3(*as_))
    assert min(seen) > 300
