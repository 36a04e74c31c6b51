// Arithmetic of the paged cache that kernels and host share: which request and which rows a work item has, which keys they see,
// and where a position's row lies.
//
// Tensors over new tokens hold the requests one after the other, request r's from q_start[r] on; n of them with G query heads
// to a key head are n * G rows of that key head, row = token * G + head.  How many there are is known on the device only.  A
// grid over pieces of `per` rows has floor(rows / per) + requests + 1 of them: request r's begin at piece floor(start / per) + r,
// which leaves it the ceil(n / per) that it needs and at most one that nobody has.
#pragma once

#include "sfm_common.hpp"

namespace sfm {

// Quotient by a divisor that the host knows: exact for n < 2^28, with magic = floor(2^k / d) + 1, k = 28 + ceil(log2 d): the
// product is above n 2^k / d by n (magic - 2^k / d) <= n < 2^28 <= 2^k / d, too little to reach the next quotient.
struct FastDiv {
    uint32_t magic, shift, d;
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t log = 0;
    while (((uint64_t)1 << log) < d) ++log;
    FastDiv f;
    f.shift = 28 + log;
    f.magic = (uint32_t)(((uint64_t)1 << f.shift) / d + 1);
    f.d = d;
    return f;
}
__host__ __device__ __forceinline__ uint32_t quot(uint32_t n, const FastDiv& f) { return (uint32_t)(((uint64_t)n * f.magic) >> f.shift); }

// A request's new tokens, whatever the tensors say: rows [first, first + n) of T; its keys are positions [0, past + n).
// Request R stands for the rows behind the last one: no keys.
struct Request {
    int first, n, past;
};
__host__ __device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__host__ __device__ __forceinline__ Request request_of(const int32_t* q_start, const int32_t* past, int r, int R, int T) {
    Request q;
    q.first = clamp_int(q_start[r], 0, T);
    const int end = r < R ? clamp_int(q_start[r + 1], 0, T) : T;
    q.n = end > q.first ? end - q.first : 0;
    q.past = r < R ? (past[r] > 0 ? past[r] : 0) : 0;
    return q;
}
// first piece of request r
__host__ __device__ __forceinline__ int64_t first_piece(int64_t start, int64_t heads, int64_t per, int r) { return start * heads / per + r; }
__host__ __device__ __forceinline__ int64_t pieces(int64_t rows, int64_t per, int R) { return rows / per + R + 1; }

// The keys that a piece's tokens [t0, t1] of a request see, in tiles of 64 positions.  A token's keys end at `end`: its own position
// + 1 (causal) or the request's length; with a window only the last `window` of them and the first `sink` count.  Positions
// from `cap` on have no entry in the table.  Virtual tiles 0 .. tiles - 1 are tiles 0 .. sinks - 1 and then first, first + 1, ...;
// of them [fast0, fast1) are seen whole by every token.
struct KeyTiles {
    int end_min, end_max, lo_min, lo_max, sinks, first, tiles, fast0, fast1;
    bool beyond;               // the request has positions that no entry of the table can hold
};
__host__ __device__ __forceinline__ KeyTiles key_tiles(const Request& q, bool none, int t0, int t1, bool causal, int window, int sink, int cap) {
    KeyTiles k;
    const int64_t len = none ? 0 : (int64_t)q.past + q.n;
    const int64_t a = causal && !none ? (int64_t)q.past + t0 + 1 : len, b = causal && !none ? (int64_t)q.past + t1 + 1 : len;
    k.beyond = b > cap;
    k.end_min = (int)(a < cap ? a : cap);
    k.end_max = (int)(b < cap ? b : cap);
    k.lo_min = window && k.end_min > window ? k.end_min - window : 0;
    k.lo_max = window && k.end_max > window ? k.end_max - window : 0;
    const int s = window ? (sink < k.end_max ? sink : k.end_max) : 0;
    k.first = k.lo_min / 64;
    k.sinks = (s + 63) / 64 < k.first ? (s + 63) / 64 : k.first;
    const int last = (k.end_max + 63) / 64;
    k.tiles = k.sinks + (last > k.first ? last - k.first : 0);
    const int f0 = k.sinks + (k.lo_max + 63) / 64 - k.first, f1 = k.sinks + k.end_min / 64 - k.first;
    k.fast0 = f0 < f1 ? f0 : 0;
    k.fast1 = f0 < f1 ? f1 : 0;
    return k;
}

// How many virtual tiles a piece of `rows` rows, `heads` query heads to a token, has at most.  With a window: those of the first positions, and
// those that [lo_min, end_max) touches, at most window + span positions, where the last positions of the piece's tokens are `span` apart.
inline int64_t most_tiles(int64_t rows, int64_t heads, int64_t tokens, bool causal, int64_t window, int64_t sink, int64_t cap) {
    const int64_t all = (cap + 63) / 64, last = (rows + heads - 2) / heads, span = !causal ? 0 : last < tokens - 1 ? last : tokens - 1;
    const int64_t seen = (sink + 63) / 64 + (window + span + 126) / 64;
    return window && seen < all ? seen : all;
}

// Rows of `bytes`, n[0] n[1] n[2] of them at strides of bytes.
struct Rows3 {
    const void* at;
    int64_t bytes;
    int64_t n[3] = {1, 1, 1}, stride[3] = {0, 0, 0};
    int64_t extent() const {
        int64_t e = bytes;
        for (int i = 0; i < 3; ++i) e += (n[i] - 1) * stride[i];
        return e;
    }
    int64_t largest_stride() const {
        int64_t s = 0;
        for (int i = 0; i < 3; ++i) s = n[i] > 1 && stride[i] > s ? stride[i] : s;
        return s;
    }
    // one repetition of the rows at stride s, and how many there are
    Rows3 without(int64_t s, int64_t* count) const {
        Rows3 r = *this;
        *count = 1;
        for (int i = 0; i < 3; ++i)
            if (n[i] > 1 && stride[i] == s) {
                *count = n[i];
                r.n[i] = 1;
                break;
            }
        return r;
    }
};
// Whether rows of b, which lies x bytes behind a, share a byte with rows of a: columns, heads or pages of one buffer may lie between each
// other.  The largest stride S of both is taken apart: repetition j of b's lies x + (j - i) S behind repetition i of a's, and few of those
// distances are short enough to meet.  Where there are many the strides do not nest, and that is taken for a yes.
inline bool meet(const Rows3& a, const Rows3& b, int64_t x) {
    if (x >= a.extent() || -x >= b.extent()) return false;
    const int64_t sa = a.largest_stride(), sb = b.largest_stride(), S = sa > sb ? sa : sb;
    if (S == 0) return true;
    int64_t na, nb;
    const Rows3 ai = a.without(S, &na), bi = b.without(S, &nb);
    auto floor_div = [](int64_t v, int64_t d) { return v >= 0 ? v / d : -((-v + d - 1) / d); };
    const int64_t lo = -floor_div(bi.extent() - 1 + x, S), hi = floor_div(ai.extent() - 1 - x, S);
    const int64_t k0 = lo > 1 - na ? lo : 1 - na, k1 = hi < nb - 1 ? hi : nb - 1;
    if (k1 - k0 >= 4) return true;
    for (int64_t k = k0; k <= k1; ++k)
        if (meet(ai, bi, x + k * S)) return true;
    return false;
}
// Whether two rows of r share a byte
inline bool folds(const Rows3& r) {
    const int64_t S = r.largest_stride();
    if (S == 0) return false;
    int64_t n;
    const Rows3 one = r.without(S, &n);
    for (int64_t k = 1; k < n && k * S < one.extent(); ++k)
        if (k == 4 || meet(one, one, k * S)) return true;
    return folds(one);
}

// Pieces of a causal prompt whose workgroups are on the chip all at once, two to a compute unit.  A head's last pieces have the most keys.  In
// its list they alternate with its first, so that every XCD's share of the list is as much work; an XCD takes the even places of its
// share (the long pieces) first, one per compute unit, and then the odd ones, which join them.
__host__ __device__ __forceinline__ int paired_piece(int at, int pieces) { return at & 1 ? at / 2 : pieces - 1 - at / 2; }
__host__ __device__ __forceinline__ int paired_place(int i, int share) { return i < (share + 1) / 2 ? 2 * i : 2 * (i - (share + 1) / 2) + 1; }

constexpr int kNoPos = 0x7ffffff8;                 // of a block that nobody sees

// Eight positions that one tile and one page hold are a block.  What a lane needs of a piece to find its blocks
struct BlockMap {
    const int32_t* table;          // the request's row
    const int32_t* sel;
    int blocks, count, sinks8, skip8, end_max, lo_min, sink, width, pages;
    FastDiv page8;
    int64_t page_bytes, block_bytes;
    // entry of the table and first position of virtual block vb; the entry is -1 where no token of the piece sees the block
    __host__ __device__ __forceinline__ int entry(int vb, uint32_t* off8, int* pos) const {
        *off8 = 0;
        *pos = kNoPos;
        if (vb >= blocks) return -1;
        const uint32_t pb = sel ? (uint32_t)vb : (uint32_t)(vb < sinks8 ? vb : vb + skip8);
        const uint32_t e = quot(pb, page8);
        *off8 = pb - e * page8.d;
        int en = (int)e;
        if (sel) {
            en = (int)e < count ? sel[e] : -1;
            if (en < 0 || en >= width) return -1;
        }
        *pos = (int)(((uint32_t)en * page8.d + *off8) * 8);
        if (*pos >= end_max || (*pos + 7 < lo_min && *pos >= sink)) return -1;
        return en;
    }
    // the page of an entry, -1 where it is outside the pool
    __host__ __device__ __forceinline__ int page(int e) const {
        const int n = e >= 0 ? table[e] : -1;
        return n >= 0 && n < pages ? n : -1;
    }
    // byte offset of the block in a head's rows of the pools; blocks that nobody sees lie in page 0
    __host__ __device__ __forceinline__ int64_t offset(int page, uint32_t off8) const { return page < 0 ? 0 : page * page_bytes + off8 * block_bytes; }
};

#if defined(__HIPCC__)
template <typename T> struct Chunk;                // 16 bytes <-> floats
template <> struct Chunk<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void get(u32x4 w, float* x) {
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    }
};
template <class E> struct Chunk16 {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void get(u32x4 w, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = E::to_float((uint16_t)(w[i] & 0xffffu));
            x[2 * i + 1] = E::to_float((uint16_t)(w[i] >> 16));
        }
    }
};
template <> struct Chunk<BF16> : Chunk16<BF16> {};
template <> struct Chunk<F16> : Chunk16<F16> {};

// The last r in [0, R] with at(r) <= v, R standing for the rows behind the last request: at ascends from at(0) <= v, and a wave looks
// at 64 of its values at a time.  The same in every lane; some r in [0, R] where the values make no sense.
template <class F>
__device__ __forceinline__ int find_last(int R, int64_t v, F at) {
    int lo = 0, n = R + 1;                         // in [lo, lo + n)
    const int lane = threadIdx.x & 63;
    while (n > 1) {
        const int step = (n + 63) / 64, off = lane * step;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(off < n && at(lo + off) <= v);
        const int k = hit ? 63 - __builtin_clzll(hit) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// The request that a piece of `per` of its rows belongs to (R: nobody's rows), and what find_last and request_of say of it.  Up to 63
// requests are read at once, a lane each: one round to memory in place of two.
__device__ __forceinline__ int find_request(const int32_t* q_start, const int32_t* past, int R, int T, int64_t piece, int64_t heads, int64_t per,
                                            Request* q) {
    if (R > 63) {
        const int r = find_last(R, piece, [&](int i) { return first_piece(clamp_int(q_start[i], 0, T), heads, per, i); });
        *q = request_of(q_start, past, r, R, T);
        return r;
    }
    const int lane = threadIdx.x & 63;
    const int mine = clamp_int(lane <= R ? q_start[lane] : T, 0, T), held = lane < R ? past[lane] : 0;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(lane <= R && first_piece(mine, heads, per, lane) <= piece);
    const int r = hit ? 63 - __builtin_clzll(hit) : 0;
    q->first = __builtin_amdgcn_readlane(mine, r);
    const int end = r < R ? __builtin_amdgcn_readlane(mine, r < 63 ? r + 1 : r) : T, had = __builtin_amdgcn_readlane(held, r);
    q->n = end > q->first ? end - q->first : 0;
    q->past = had > 0 ? had : 0;
    return r;
}
#endif

}  // namespace sfm
