// Attention of the requests' new tokens over their pages of a shared key-value cache.
#include <algorithm>

#include "attn_tiles.hpp"
#include "paged_rules.hpp"

namespace sfm {

struct PagedArgs {
    sfm_paged_desc d;
    FastDiv page8;                 // page_size / 8
    int cap;                       // positions that a row of the table holds
    const void *q, *kp, *vp;
    const int32_t *table, *past, *q_start, *selected;
    void* out;
    float* lse;
};

// One value of a tensor, four of a row
template <typename T> struct PElem;
template <> struct PElem<float> {
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return ((const float*)p)[i]; }
    static __device__ __forceinline__ void put(void* p, int64_t i, float x) { ((float*)p)[i] = x; }
    static __device__ __forceinline__ void put4(void* p, int64_t i, f32x4 x) { *(f32x4*)((float*)p + i) = x; }
};
template <class E> struct PElem16 {
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return E::to_float(((const uint16_t*)p)[i]); }
    static __device__ __forceinline__ void put(void* p, int64_t i, float x) { ((uint16_t*)p)[i] = E::from_float(x); }
    static __device__ __forceinline__ void put4(void* p, int64_t i, f32x4 x) { *(u32x2*)((uint16_t*)p + i) = u32x2{pack2<E>(x.x, x.y), pack2<E>(x.z, x.w)}; }
};
template <> struct PElem<BF16> : PElem16<BF16> {};
template <> struct PElem<F16> : PElem16<F16> {};

// ------------------------------------------------------------------------------------------------
// out = softmax(sm_scale q K^T) V in one pass over the keys: with m the running maximum of a row's logits, l = sum exp(x - m) and
// O = sum exp(x - m) v, both scaled by exp(m_old - m) where m grows; out = O / l, and m + log l beside it.  Logits are in units of log 2.
//
// A piece is up to M rows (token, query head) of one request and one key head.  Its keys come in virtual tiles of 64 positions
// (KeyTiles), or of the selected pages one after the other; eight positions, a block, never straddle a page, and a lane works out where
// one block lies (BlockMap).  The matrix kernels' products (16-bit tensors, head sizes 64 and 128) are those of the dense kernel:
// S^T[l, q] = K[l,:] . Q[q,:], O^T[d, q] += V^T[d, l] P^T[l, q], a lane holds one row's logits; the weights are rounded to the tensors' type for the
// second (half a step of theirs, with signs that average out), their sum is not.
// ------------------------------------------------------------------------------------------------
struct Piece {
    Request rq;
    KeyTiles k;
    int r, kh, row0, row1;         // rows [row0, row1) of the request's n * G
    const int32_t* sel;            // selected entries, `count` of them, or NULL
    int count;
};

// Softmax state of a wave's 32 rows, lane (m, hf) row m: O^T accumulators, running maximum (base-2 units) and this half's sum
template <int D>
struct RowState {
    f32x16 o[D / 32];
    float mrun, lrun;
    bool seen;
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[dt][v] = 0.f;
        mrun = -__FLT_MAX__;
        lrun = 0.f;
        seen = false;
    }
    __device__ __forceinline__ void raise(float mnew) {
        if (__builtin_amdgcn_ballot_w64(mnew > mrun) != 0) {
            const float alpha = fast_exp2(mrun - mnew);
            lrun *= alpha;
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[dt][v] *= alpha;
            mrun = mnew;
        }
    }
};

// What a row sees of a tile: positions below `end` that, with a window, are at or past `lo` or below `sink`
struct RowMask {
    int end, lo, sink;
    bool window;
    __device__ __forceinline__ bool sees(int pos) const { return pos < end && (!window || pos >= lo || pos < sink); }
};

// Which V rows of a tile hold values that are not finite, a bit each: of rows r0 + lane / LPR, LPR lanes to a row.
template <class E, int D, int LPR>
__device__ __forceinline__ uint64_t odd_rows(const char* lds, uint32_t vbuf, int r0) {
    using L = DnLds<D>;
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    constexpr uint16_t kInf = E::kDtype == SFM_BF16 ? 0x7f80 : 0x7c00;
    const int lane = threadIdx.x & 63, r = r0 + lane / LPR, c0 = lane % LPR;
    u16x2 top = {0, 0};                                                // largest magnitude's bits
#pragma unroll 4
    for (int c = 0; c < L::kCPR / LPR; ++c) {                          // neighbouring rows begin at different chunks: apart in the banks
        const u32x4 w = *(const u32x4*)(lds + vbuf + (uint32_t)r * L::kPitch + (uint32_t)((c0 + LPR * ((c + r) % (L::kCPR / LPR))) << 4));
#pragma unroll
        for (int x = 0; x < 4; ++x) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[x] & 0x7fff7fffu));
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(max(top.x, top.y) >= kInf);
    if (LPR == 1) return hit;
    return __builtin_amdgcn_ballot_w64(lane < 64 / LPR && ((hit >> (lane * LPR & 63)) & ((1u << LPR) - 1)) != 0);
}

// A tile of 32 NB keys in LDS against the wave's rows: logits, masks, weights and V's part.  pos: first positions of its blocks.
// The second half waits for V through `v_ready`, so that K's buffer can be refilled meanwhile (`k_done`).
//
// A masked weight is 0, and 0 times an infinity or NaN is NaN: in a masked tile V rows that hold such values (`v_ready` tells which) are left out
// of the matrix product and added for the rows that see them, one by one.  (Stale rows, and later tokens of the request.)
template <class E, int D, int NB, class KDone, class VReady>
__device__ __forceinline__ void masked_tile(const char* lds, uint32_t kbuf, uint32_t vbuf, const u32x4* qb, float sc2, RowState<D>& st,
                                            const RowMask& mask, bool masked, const int* pos, KDone k_done, VReady v_ready) {
    using L = DnLds<D>;
    const int lane = threadIdx.x & 63, m = lane & 31, hf = lane >> 5;
    f32x16 s[NB];
#pragma unroll
    for (int t = 0; t < NB; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[t][v] = 0.f;
    const uint32_t sA0 = kbuf + (uint32_t)m * L::kPitch + (uint32_t)((hf ^ L::swz(m)) << 4);
#pragma unroll
    for (int j = 0; j < NB * D / 16; ++j) {
        const u32x4 a = *(const u32x4*)(lds + (sA0 ^ (uint32_t)((j / NB) << 5)) + (j % NB) * 32 * L::kPitch);
        s[j % NB] = E::mfma32(a, qb[j / NB], s[j % NB]);
    }
    k_done();
    if (masked) {
        // key 32 t + 8 g + 4 hf + i is number 4 hf + i of block 4 t + g: the block's first position against limits per i
        int end[4], lo[4], sink[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) end[i] = mask.end - 4 * hf - i;
        if (!mask.window) {
#pragma unroll
            for (int b = 0; b < 4 * NB; ++b) {
                st.seen = st.seen | (pos[b] < end[0]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[b >> 2][4 * (b & 3) + i] = pos[b] < end[i] ? s[b >> 2][4 * (b & 3) + i] : -INFINITY;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) lo[i] = mask.lo - 4 * hf - i, sink[i] = mask.sink - 4 * hf - i;
#pragma unroll
            for (int b = 0; b < 4 * NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool see = (pos[b] < end[i]) & ((pos[b] >= lo[i]) | (pos[b] < sink[i]));
                    st.seen = st.seen | see;
                    s[b >> 2][4 * (b & 3) + i] = see ? s[b >> 2][4 * (b & 3) + i] : -INFINITY;
                }
        }
    } else {
        st.seen = true;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * NB; ++i) mx = fmaxf(mx, s[i >> 4][i & 15]);
    st.raise(fmaxf(st.mrun, xhalf_max(mx) * sc2));
    u32x4 pb[2 * NB];
    float psum = 0.f;
#pragma unroll
    for (int i = 0; i < 16 * NB; i += 2) {
        const float a = fast_exp2(fmaf(s[i >> 4][i & 15], sc2, -st.mrun)), b = fast_exp2(fmaf(s[i >> 4][(i & 15) + 1], sc2, -st.mrun));
        psum += a + b;
        s[i >> 4][i & 15] = a;
        s[i >> 4][(i & 15) + 1] = b;
        pb[i >> 3][(i >> 1) & 3] = pack2<E>(a, b);
    }
    st.lrun += psum;
    uint64_t odd = v_ready();
    if (!masked) odd = 0;
    uint32_t trA[2];
    const int s16 = lane & 15, rl = 4 * hf + (s16 >> 2), cl = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = rl + 8 * half;
        trA[half] = vbuf + (uint32_t)r * L::kPitch + (uint32_t)((cl ^ L::swz(r)) << 4) + (uint32_t)(s16 & 1) * 8;
    }
    if (odd == 0) {
#pragma unroll
        for (int j = 0; j < NB * D / 16; ++j) {
            const u32x2 lo = dn_read_tr(lds + (trA[0] ^ (uint32_t)((j / (2 * NB)) << 6)), (j % (2 * NB)) * 16 * L::kPitch);
            const u32x2 hi = dn_read_tr(lds + (trA[1] ^ (uint32_t)((j / (2 * NB)) << 6)), (j % (2 * NB)) * 16 * L::kPitch);
            st.o[j / (2 * NB)] = E::mfma32(u32x4{lo.x, lo.y, hi.x, hi.y}, pb[j % (2 * NB)], st.o[j / (2 * NB)]);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < NB * D / 16; ++j) {
        const u32x2 lo = dn_read_tr(lds + (trA[0] ^ (uint32_t)((j / (2 * NB)) << 6)), (j % (2 * NB)) * 16 * L::kPitch);
        const u32x2 hi = dn_read_tr(lds + (trA[1] ^ (uint32_t)((j / (2 * NB)) << 6)), (j % (2 * NB)) * 16 * L::kPitch);
        const uint32_t bits = (uint32_t)(odd >> (16 * (j % (2 * NB)))) >> (4 * hf);   // keys 16 (j % (2 NB)) + 4 hf + {0..3, 8..11}
        const u32x4 keep = {(bits & 1 ? 0u : 0xffffu) | (bits & 2 ? 0u : 0xffff0000u), (bits & 4 ? 0u : 0xffffu) | (bits & 8 ? 0u : 0xffff0000u),
                            (bits & 0x100 ? 0u : 0xffffu) | (bits & 0x200 ? 0u : 0xffff0000u), (bits & 0x400 ? 0u : 0xffffu) | (bits & 0x800 ? 0u : 0xffff0000u)};
        st.o[j / (2 * NB)] = E::mfma32(u32x4{lo.x, lo.y, hi.x, hi.y} & keep, pb[j % (2 * NB)], st.o[j / (2 * NB)]);
    }
    while (odd) {
        const int l = __builtin_ctzll(odd);
        odd &= odd - 1;
        // the weight, rounded as the matrix product takes it, lies in half (l / 4) % 2, number 16 (l / 32) + 4 (l / 8 % 4) + l % 4
        uint32_t both = 0;
        const int at = 16 * (l >> 5) + 4 * ((l >> 3) & 3) + (l & 3);
#pragma unroll
        for (int i = 0; i < 8 * NB; ++i) both = i == at >> 1 ? pb[i >> 2][i & 3] : both;
        const float w = __shfl(E::to_float((uint16_t)(both >> (16 * (at & 1)))), m + 32 * ((l >> 2) & 1));
        int p = kNoPos;
#pragma unroll
        for (int i = 0; i < 4 * NB; ++i) p = i == (l >> 3) ? pos[i] : p;
        const bool see = !masked || mask.sees(p + (l & 7));
#pragma unroll
        for (int c = 0; c < L::kCPR; ++c) {        // channels 8 c + 4 hf + {0..3}
            const u32x2 x = *(const u32x2*)(lds + vbuf + (uint32_t)l * L::kPitch + (uint32_t)((c ^ L::swz(l)) << 4) + 8 * hf);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = E::to_float((uint16_t)(x[i >> 1] >> (16 * (i & 1))));
                // an infinity with a weight that went to 0 stays one here; rescaled or joined by a factor of 0 it becomes NaN, as it does in a
                // tile without masks: which of the two a row gets hangs on where its tiles and ranges end
                const float part = w == w && !(fabsf(v) < INFINITY) ? v : w * v;
                const float o = st.o[c >> 2][4 * (c & 3) + i];
                st.o[c >> 2][4 * (c & 3) + i] = see ? o + part : o;
            }
        }
    }
}

// Partials of split calls: [chunk][row = token * H + head] of D floats, and behind all of them (maximum, sum).  Of a range whose keys a row
// sees, but all with a logit of -infinity, the sum is 0 as of one where it sees none, for which nothing is joined.  The row is NaN then only
// if that holds of all of its ranges: such a range's maximum is -infinity and its sum 1, so that it counts, with a factor of 0.
__device__ __forceinline__ void store_partial(float* ml, float mrun, float sum, bool seen, bool bad) {
    const bool none = seen && sum == 0.f;
    ml[0] = none ? -INFINITY : mrun;
    ml[1] = bad ? NAN : !seen ? 0.f : none ? 1.f : sum;
}

template <class E, int D>
__device__ __forceinline__ void store_rows(const PagedArgs& a, const Piece& pc, RowState<D>& st, bool bad, int row0, int chunk, int chunks,
                                           float* part, char* stage) {
    const sfm_paged_desc& d = a.d;
    const int lane = threadIdx.x & 63, m = lane & 31, hf = lane >> 5, G = d.H / d.kv_heads;
    const int row = row0 + m, t = pc.rq.first + row / G, h = pc.kh * G + row % G;
    const bool mine = row < pc.row1;
    const float l = xhalf_sum(st.lrun);
    const bool seen = __shfl_xor((int)st.seen, 32) || st.seen;
    if (part != nullptr) {
        const int64_t rows = d.tokens * d.H, at = chunk * rows + (int64_t)t * d.H + h;
        if (!mine) return;
        float* const po = part + at * D + 4 * hf;
        if (seen)
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(f32x4*)(po + 32 * dt + 8 * g) = f32x4{st.o[dt][4 * g], st.o[dt][4 * g + 1], st.o[dt][4 * g + 2], st.o[dt][4 * g + 3]};
        if (hf == 0) store_partial(part + chunks * rows * D + at * 2, st.mrun, l, seen, bad);
        return;
    }
    const float inv = bad ? NAN : seen ? 1.f / l : 0.f;
    if (a.lse != nullptr && hf == 0 && mine) a.lse[(int64_t)h * d.tokens + t] = bad ? NAN : seen ? (st.mrun + log2f(l)) * kLn2 : -INFINITY;
    // through LDS, so that the rows leave in whole lines
    constexpr int kSP = D + 8;
    uint16_t* const so = (uint16_t*)stage;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(u32x2*)(so + m * kSP + 32 * dt + 8 * g + 4 * hf) = u32x2{pack2<E>(st.o[dt][4 * g] * inv, st.o[dt][4 * g + 1] * inv),
                                                                      pack2<E>(st.o[dt][4 * g + 2] * inv, st.o[dt][4 * g + 3] * inv)};
    lds_wave_sync();
    uint16_t* const out = (uint16_t*)a.out;
    for (int c = lane; c < 32 * (D / 8); c += 64) {
        const int r = row0 + c / (D / 8), ch = c % (D / 8);
        if (r < pc.row1)
            *(u32x4*)(out + (int64_t)(pc.rq.first + r / G) * d.o_stride[0] + (int64_t)(pc.kh * G + r % G) * d.o_stride[1] + ch * 8) =
                *(const u32x4*)(so + (c / (D / 8)) * kSP + ch * 8);
    }
}

// The piece of a work item; false where it has no rows.
template <int M>
__device__ __forceinline__ bool find_piece(const PagedArgs& a, int64_t piece, int kh, Piece* p) {
    const sfm_paged_desc& d = a.d;
    const int R = d.requests, T = (int)d.tokens, G = d.H / d.kv_heads;
    int64_t per = M, heads = G, j = 0, unit = piece;
    if (d.top) {                   // groups, each in pieces of M rows
        const int64_t each = ((int64_t)min(d.group, T) * G + M - 1) / M;
        unit = piece / each;
        j = piece - unit * each;
        per = d.group;
        heads = 1;
    }
    const int r = find_request(a.q_start, a.past, R, T, unit, heads, per, &p->rq);
    if (r >= R && !d.zero_rest) return false;
    p->r = r;
    p->kh = kh;
    const int64_t nth = unit - first_piece(p->rq.first, heads, per, r), rows = (int64_t)p->rq.n * G;
    int64_t row0 = nth * M, last = rows;
    if (d.top) {
        row0 = nth * d.group * G + j * M;
        last = min(rows, (nth + 1) * d.group * G);
    }
    if (nth < 0 || row0 >= last) return false;
    p->row0 = (int)row0;
    p->row1 = (int)min(last, row0 + M);
    p->k = key_tiles(p->rq, r >= R, p->row0 / G, (p->row1 - 1) / G, d.causal, d.window, d.sink, a.cap);
    p->sel = nullptr;
    p->count = 0;
    if (d.top) {
        KeyTiles& k = p->k;
        p->sel = a.selected + (unit * d.kv_heads + kh) * d.top;
        // entries up to the first that is none, and of those the ones that every token of the piece sees whole
        const int lane = threadIdx.x & 63, whole = k.end_min / d.page_size;
        int count = d.top, full = d.top;
        for (int e0 = 0; e0 < d.top; e0 += 64) {
            const int e = e0 + lane < d.top ? p->sel[e0 + lane] : -1;
            const uint64_t none = __builtin_amdgcn_ballot_w64(e < 0), part = __builtin_amdgcn_ballot_w64(e < 0 || e >= whole);
            if (part && full == d.top) full = min(full, e0 + __builtin_ctzll(part));
            if (none) {
                count = min(count, e0 + __builtin_ctzll(none));
                break;
            }
        }
        if (r >= R) count = full = 0;
        const int64_t keys = (int64_t)count * d.page_size;
        p->count = count;
        k.beyond = false;
        k.sinks = k.first = 0;
        k.tiles = (int)((keys + 63) / 64);
        k.fast0 = 0;
        k.fast1 = (int)((int64_t)full * d.page_size / 64);
    }
    return true;
}

__device__ __forceinline__ BlockMap block_map(const PagedArgs& a, const Piece& p, int esz) {
    const sfm_paged_desc& d = a.d;
    BlockMap b;
    b.table = a.table + (int64_t)(p.r < d.requests ? p.r : 0) * d.table_stride;
    b.sel = p.sel;
    b.blocks = p.k.tiles * 8;
    b.count = p.count;
    b.sinks8 = p.k.sinks * 8;
    b.skip8 = (p.k.first - p.k.sinks) * 8;
    b.end_max = p.k.end_max;
    b.lo_min = p.k.lo_min;
    b.sink = d.sink;
    b.width = d.width;
    b.pages = d.pages;
    b.page8 = a.page8;
    b.page_bytes = d.pool_stride[0] * esz;
    b.block_bytes = d.pool_stride[1] * 8 * esz;
    return b;
}

// Operands of the rows row0 .. + 31 (those past the piece repeat its last): asked for here, in front of the table's entries, and waited for
// behind those (wait_queries), before any tile is
template <class E, int D>
__device__ __forceinline__ void load_queries(const PagedArgs& a, const Piece& p, int row0, u32x4* qb) {
    const sfm_paged_desc& d = a.d;
    const int lane = threadIdx.x & 63, m = lane & 31, hf = lane >> 5, G = d.H / d.kv_heads;
    const int row = min(row0 + m, p.row1 - 1), t = row / G;
    const uint16_t* const q = (const uint16_t*)a.q + (int64_t)(p.rq.first + t) * d.q_stride[0] + (int64_t)(p.kh * G + row - t * G) * d.q_stride[1] + 8 * hf;
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds) qb[ds] = *(const u32x4*)(q + 16 * ds);
    asm volatile("" ::: "memory");
}
template <int D>
__device__ __forceinline__ void wait_queries(u32x4* qb) {
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds) asm volatile("" : "+v"(qb[ds]));
}

// What a row sees; of a wave's rows row0 .. + 31, the lane's
__device__ __forceinline__ RowMask row_mask(const PagedArgs& a, const Piece& p, int row) {
    const sfm_paged_desc& d = a.d;
    RowMask k;
    k.end = d.causal ? (int)min((int64_t)p.rq.past + row / (d.H / d.kv_heads) + 1, (int64_t)a.cap) : p.k.end_max;
    k.lo = d.window && k.end > d.window ? k.end - d.window : 0;
    k.sink = d.sink;
    k.window = d.window != 0;
    return k;
}
__device__ __forceinline__ RowMask lane_mask(const PagedArgs& a, const Piece& p, int row0) {
    return row_mask(a, p, min(row0 + (int)(threadIdx.x & 31), p.row1 - 1));
}

// ---- few rows: a wave takes tiles of its own --------------------------------------------------------------------------------
//
// Pieces of up to 32 rows, single tokens above all.  The four waves of a workgroup take its tiles in turn, in halves of 32 keys, each
// with a K and a V buffer that no other wave sees and no barrier: while a wave works on K the V rows are on their way, and the next
// K's as soon as its last is read.  Two workgroups share a compute unit, so that the one's start (its piece, table entries, first
// rows) is behind the other's loads.  Bound by reading the cache: of the matrix instructions' 32 columns a single token uses the
// query heads of its key head, and they take a tenth of the time that the rows do.  32 tokens on 100 to 16000 positions, 32 heads on 8 of 128, pages
// of 16: 848 MB in 167 us, 5.1 TB/s (a bare read 5.8).  One token on 1560 positions, 12 heads: 11 us, of which its bytes take 2: launch, the request, its
// table, first rows and the last tile are waited for one after the other.
template <int D>
struct FewLds {
    static constexpr int kMat = DnLds<D>::kMat / 2, kWave = 2 * kMat, kTotal = 4 * kWave;
};

template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <class E, int D, bool ONCE>
__global__ __launch_bounds__(256, 2) void paged_few_kernel(PagedArgs a, int64_t npieces, int chunks, int chunk_tiles, float* part, bool) {
    using L = DnLds<D>;
    constexpr int kRows = 64 / L::kCPR, kLoads = 32 / kRows, kVar = D == 128 ? 4 : 2;  // rows of a load, loads of half a tile, column orders
    extern __shared__ __attribute__((aligned(256))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds, buf = (uint32_t)wave * FewLds<D>::kWave;
    const sfm_paged_desc& d = a.d;
    // the heads of a token's row side by side
    const int item = blockIdx.x, kh = item % d.kv_heads, rest = item / d.kv_heads;
    if (rest >= npieces * chunks) return;
    const int chunk = rest % chunks;
    Piece p;
    if (!find_piece<32>(a, rest / chunks, kh, &p)) return;
    const int v0 = min(chunk * chunk_tiles, p.k.tiles), v1 = min(v0 + chunk_tiles, p.k.tiles);
    const BlockMap map = block_map(a, p, 2);
    u32x4 qb[D / 16];
    load_queries<E, D>(a, p, p.row0, qb);
    const RowMask mask = lane_mask(a, p, p.row0);
    RowState<D> st;
    st.init();
    bool bad = p.k.beyond;
    const float sc2 = d.sm_scale * kLog2e;

    const int n = v0 + wave < v1 ? 2 * ((v1 - v0 - wave + 3) / 4) : 0; // this wave's halves: of tiles v0 + wave + 4 (i / 2)
    uint32_t off_lo = 0, off_hi = 0;                                    // lane: block lane % 8 of the tile i / 2 with i / 2 % 8 = lane / 8
    int pos_of = kNoPos;
    auto blocks = [&](int t0) {
        const int t = t0 + (lane >> 3);
        uint32_t off8;
        const int e = map.entry(2 * t < n ? 8 * (v0 + wave + 4 * t) + (lane & 7) : kNoPos, &off8, &pos_of);
        const int page = map.page(e);
        bad = bad || __builtin_amdgcn_ballot_w64(e >= 0 && page < 0) != 0;
        const int64_t off = map.offset(page, off8);
        off_lo = (uint32_t)off;
        off_hi = (uint32_t)(off >> 32);
    };
    const char* const kg = (const char*)a.kp + (int64_t)kh * d.pool_stride[2] * 2;
    const char* const vg = (const char*)a.vp + (int64_t)kh * d.pool_stride[2] * 2;
    const uint32_t row_bytes = (uint32_t)d.pool_stride[1] * 2;
    uint32_t voff[kVar];
#pragma unroll
    for (int x = 0; x < kVar; ++x) {
        const int r = x * kRows + lane / L::kCPR;                      // swz repeats after 16 rows
        voff[x] = (uint32_t)(lane / L::kCPR) * row_bytes + (uint32_t)(((lane % L::kCPR) ^ L::swz(r)) * 16);
    }
    auto stage = [&](const char* g, int i, uint32_t dst) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int from = 4 * (i & 15) + j * kRows / 8;
            const uint64_t off = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(off_hi, from) << 32 | (uint32_t)__builtin_amdgcn_readlane(off_lo, from);
            const char* const from_block = g + off + (uint32_t)(j * kRows % 8) * row_bytes;
            if (ONCE) dn_load_lds16_nt(from_block, voff[j % kVar], lds0 + dst + (uint32_t)j * 1024);
            else dn_load_lds16(from_block, voff[j % kVar], lds0 + dst + (uint32_t)j * 1024);
        }
    };
    if (n > 0) {
        blocks(0);
        wait_queries<D>(qb);
        stage(kg, 0, buf);
        stage(vg, 0, buf + FewLds<D>::kMat);
    }
    for (int i = 0; i < n; ++i) {
        int pos[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) pos[b] = __builtin_amdgcn_readlane(pos_of, 4 * (i & 15) + b);
        const bool next = i + 1 < n;
        const int v = v0 + wave + 4 * (i >> 1);
        const bool masked = v < p.k.fast0 || v >= p.k.fast1;
        wait_loads<kLoads>();                                          // K of this tile; V's are behind it
        masked_tile<E, D, 1>(lds, buf, buf + FewLds<D>::kMat, qb, sc2, st, mask, masked, pos,
            [&]() {
                lds_wave_sync();                                       // K is read
                if (next) {
                    if (((i + 1) & 15) == 0) blocks((i + 1) / 2);
                    stage(kg, i + 1, buf);
                }
            },
            [&]() {
                if (next) wait_loads<kLoads>();
                else wait_loads<0>();
                return masked ? odd_rows<E, D, 2>(lds, buf + FewLds<D>::kMat, 0) : (uint64_t)0;
            });
        lds_wave_sync();
        if (next) stage(vg, i + 1, buf + FewLds<D>::kMat);
    }
    // the waves' rows joined: O, maximum and sum through LDS, 32 x D floats each
    float* const wo = (float*)(lds + buf);                             // [D][32] by (channel, row): lanes of a row group apart
    float* const ml = (float*)(lds + FewLds<D>::kTotal);               // [4 waves][3][32]
    const int m = lane & 31, hf = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) wo[(32 * dt + 8 * (v >> 2) + 4 * hf + (v & 3)) * 32 + m] = st.o[dt][v];
    const float lsum = xhalf_sum(st.lrun);
    const bool sees = __shfl_xor((int)st.seen, 32) || st.seen;
    if (hf == 0) {
        ml[wave * 96 + m] = st.mrun;
        ml[wave * 96 + 32 + m] = lsum;
        ml[wave * 96 + 64 + m] = bad ? 2.f : sees ? 1.f : 0.f;
    }
    __syncthreads();
    // wave w takes rows in turn; a lane D / 64 channels
    const int G = d.H / d.kv_heads;
    for (int row = wave; row < p.row1 - p.row0; row += 4) {
        float M = -__FLT_MAX__, sum = 0.f, o[D / 64];
        bool rbad = false, rseen = false;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            M = fmaxf(M, ml[w * 96 + row]);
            rbad = rbad || ml[w * 96 + 64 + row] == 2.f;
            rseen = rseen || ml[w * 96 + 64 + row] == 1.f;
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c) o[c] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (ml[w * 96 + 64 + row] == 0.f) continue;
            const float f = fast_exp2(ml[w * 96 + row] - M);
            sum += f * ml[w * 96 + 32 + row];
            const float* const x = (const float*)(lds + (uint32_t)w * FewLds<D>::kWave);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) o[c] += f * x[(lane * (D / 64) + c) * 32 + row];
        }
        const int rr = p.row0 + row, t = p.rq.first + rr / G, h = kh * G + rr % G;
        if (part != nullptr) {
            const int64_t rows = d.tokens * d.H, at = chunk * rows + (int64_t)t * d.H + h;
            if (rseen)
#pragma unroll
                for (int c = 0; c < D / 64; ++c) part[at * D + lane * (D / 64) + c] = o[c];
            if (lane == 0) store_partial(part + chunks * rows * D + at * 2, M, sum, rseen, rbad);
        } else {
            const float inv = rbad ? NAN : rseen ? 1.f / sum : 0.f;
            uint16_t* const out = (uint16_t*)a.out + (int64_t)t * d.o_stride[0] + (int64_t)h * d.o_stride[1] + lane * (D / 64);
            if constexpr (D == 128) *(uint32_t*)out = pack2<E>(o[0] * inv, o[1] * inv);
            else *out = E::from_float(o[0] * inv);
            if (a.lse != nullptr && lane == 0) a.lse[(int64_t)h * d.tokens + t] = rbad ? NAN : rseen ? (M + log2f(sum)) * kLn2 : -INFINITY;
        }
    }
}

// ---- many rows: the waves of a workgroup share tiles -------------------------------------------------------------------------
//
// Pieces of 32 NW rows.  The tiles that all of them see whole run through the dense kernel's loop (two K and two V buffers, tiles
// straight from memory into LDS, the logits of tile n + 1 beside the exponentials of tile n, its maximum beside P V of tile n); those that
// some row sees in part (the request's own new tokens under a causal mask, a window's edge, the last tile) follow in a plain loop.
// (The loop is written out here again, since its loads differ: what is changed in the one is to be measured in the other.)
// Where the whole tiles' blocks lie is worked out by all threads together and kept in LDS, 8 bytes a block, for a stretch of tiles at a
// time (a request's page table row is read once per workgroup, not once per wave); a step reads one tile's eight offsets, a
// step before it asks for that tile, and V's rows take the offsets that K's were read with.  (Looked up by each wave as it went, eight tiles at a
// time, they took scalar registers and a branch from the loop: 4680 x 32760 of 12 heads 1185 us, with places in LDS and better chosen ranges 918.)
// Masking inside that loop would save the plain one, and spills.
//
// Bound at D = 128 by the matrix pipes and the clock that they leave (58 % of the cycles busy; 4680 x 32760 of 12 heads 902 us, 1.04 PFLOP/s,
// the dense kernel on a contiguous cache 887), at D = 64 by the vector pipes: 32 exponentials of 16 cycles and some 100 instructions of 4
// per tile and wave.  A tile of the plain loop takes two to three times as long as one of the other.
template <int D, int NW>
struct RowsLds {
    static constexpr int kPlaces = 4 * DnLds<D, NW>::kMat;                     // behind the tiles
    static constexpr int kStretch = NW == 8 ? 512 : 240;                       // tiles; two workgroups of four waves share a compute unit's 160 KB
    static constexpr int kLoop = kPlaces + (kStretch + 1) * 64, kStage = DnLds<D, NW>::kStage;
    static constexpr int kTotal = kLoop > kStage ? kLoop : kStage;
};

template <class E, int D, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_rows_kernel(PagedArgs a, int64_t npieces, int chunks, int chunk_tiles,
                                                                                                          float* part, bool paired) {
    using L = DnLds<D, NW>;
    constexpr int DS = D / 16, DT = D / 32, NTH = 64 * NW;
    extern __shared__ __attribute__((aligned(256))) char lds[];
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds;
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const sfm_paged_desc& d = a.d;
    const int total = (int)(npieces * d.kv_heads * chunks), per = (total + 7) / 8;
    // the pieces of a head go to one XCD, under a causal mask those with the most keys first, or a long and a short one in turn
    const int item = (int)(blockIdx.x % 8) * per + (paired ? paired_place(blockIdx.x / 8, per) : (int)blockIdx.x / 8);
    if (item >= total) return;
    const int unit = item / (int)npieces, kh = unit / chunks, chunk = unit - kh * chunks;
    const int at = item - unit * (int)npieces;
    Piece p;
    if (!find_piece<32 * NW>(a, !d.causal ? at : paired ? paired_piece(at, (int)npieces) : npieces - 1 - at, kh, &p)) return;
    const int v0 = min(chunk * chunk_tiles, p.k.tiles), v1 = min(v0 + chunk_tiles, p.k.tiles);
    const int f0 = max(v0, p.k.fast0), nf = max(min(v1, p.k.fast1) - f0, 0) & ~1;      // the loop over whole tiles takes two at a time
    const BlockMap map = block_map(a, p, 2);
    bool bad = p.k.beyond;

    const uint32_t row_bytes = (uint32_t)d.pool_stride[1] * 2;
    // a load moves 64 / kCPR rows of one block; a wave's loads of a tile are kRPC rows apart, a multiple of 16
    constexpr int kCh = 64 * L::kCPR / NTH, kRPC = NTH / L::kCPR;
    const int wrow = wave * 64 / L::kCPR, srow = wrow + lane / L::kCPR;
    const uint32_t voff = (uint32_t)(lane / L::kCPR) * row_bytes + (uint32_t)(((lane % L::kCPR) ^ L::swz(srow)) * 16);
    const int64_t head = (int64_t)kh * d.pool_stride[2] * 2 + (uint32_t)(wrow % 8) * row_bytes;
    const char* const kg = (const char*)a.kp + head;
    const char* const vg = (const char*)a.vp + head;
    // offsets of this wave's loads of a tile, from the lanes that hold its blocks from `from` on
    struct Places {
        uint64_t at[kCh];
    };
    auto places = [&](uint32_t lo, uint32_t hi, int from) {
        Places x;
#pragma unroll
        for (int j = 0; j < kCh; ++j) {
            const int l = from + j * (kRPC / 8) + wrow / 8;
            x.at[j] = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, l) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, l);
        }
        return x;
    };
    auto stage = [&](const char* g, const Places& x, uint32_t dst) {
#pragma unroll
        for (int j = 0; j < kCh; ++j) dn_load_lds16(g + x.at[j], voff, lds0 + dst + (uint32_t)(j * NTH + wave * 64) * 16);
    };

    u32x4 qb[DS];
    load_queries<E, D>(a, p, p.row0 + wave * 32, qb);
    RowState<D> st;
    st.init();
    const float sc2 = d.sm_scale * kLog2e;

    // the virtual tiles that are not whole come behind them: `before` of them from v0 on, the others behind the last whole one
    const int before = nf > 0 ? f0 - v0 : v1 - v0, rest = v1 - v0 - nf;
    auto tile_at = [&](int i) { return i < nf ? f0 + i : i - nf < before ? v0 + i - nf : v0 + i; };
    u32x2* const where = (u32x2*)(lds + RowsLds<D, NW>::kPlaces);
    // places of tiles [i0, i0 + n) in that order
    auto fill = [&](int i0, int n) {
        for (int b = tid; b < 8 * n; b += NTH) {
            uint32_t off8;
            int pos;
            const int e = map.entry(8 * tile_at(i0 + b / 8) + b % 8, &off8, &pos), page = map.page(e);
            bad = bad || (e >= 0 && page < 0);
            const uint64_t off = (uint64_t)map.offset(page, off8);
            where[b] = u32x2{(uint32_t)off, (uint32_t)(off >> 32)};
        }
        bad = __syncthreads_or(bad);
        wait_queries<D>(qb);
    };
    bool ready = false;                            // the first of the rest is on its way
    for (int done = 0; done < nf; done += RowsLds<D, NW>::kStretch) {
        constexpr int NA = 2 * DS, NP = 4 * DT, kVA = 32 / NA, kVP = 32 / NP, kAhead = 3, kRing = kAhead + 1;
        const int here = min(nf - done, RowsLds<D, NW>::kStretch);             // an even number of tiles
        // the last stretch takes as many of the rest with it as there is room for
        const int filled = min(v1 - v0 - done, RowsLds<D, NW>::kStretch);
        fill(done, filled);
        ready = filled > here;
        auto look = [&](int n) { return where[8 * n + (lane & 7)]; };
        const uint32_t sA0 = (uint32_t)m * L::kPitch + (uint32_t)((hf ^ L::swz(m)) << 4);
        uint32_t trA[2];
        {
            const int s16 = lane & 15, rl = 4 * hf + (s16 >> 2), cl = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = rl + 8 * half;
                trA[half] = (uint32_t)r * L::kPitch + (uint32_t)((cl ^ L::swz(r)) << 4) + (uint32_t)(s16 & 1) * 8;
            }
        }
        auto read_k = [&](uint32_t kbuf, int j) -> u32x4 {
            return *(const u32x4*)(lds + (sA0 ^ (uint32_t)((j >> 1) << 5)) + kbuf + (j & 1) * 32 * L::kPitch);
        };
        auto read_v = [&](uint32_t vbuf, int j) -> u32x4 {
            const u32x2 lo = dn_read_tr(lds + (trA[0] ^ (uint32_t)((j >> 2) << 6)), vbuf + (j & 3) * 16 * L::kPitch);
            const u32x2 hi = dn_read_tr(lds + (trA[1] ^ (uint32_t)((j >> 2) << 6)), vbuf + (j & 3) * 16 * L::kPitch);
            return u32x4{lo.x, lo.y, hi.x, hi.y};
        };
#define PG_SVAL(s, i) s[(i) >> 4][(i) & 15]
        f32x16 sbuf[2][2];
        u32x4 ring[kRing], pb[4];
        float lrun = st.lrun;

        u32x2 next = look(0);
        Places x = places(next.x, next.y, 0);
        stage(kg, x, L::kK);
        stage(vg, x, L::kV);
        next = look(1);
        x = places(next.x, next.y, 0);                     // of tile n + 1 when tile n begins
        stage(kg, x, L::kK + L::kMat);
        next = look(min(2, filled - 1));                   // of tile n + 2
        dn_wait_tiles();
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) sbuf[0][t][v] = 0.f;
#pragma unroll
        for (int j = 0; j < NA; ++j) sbuf[0][j & 1] = E::mfma32(read_k(L::kK, j), qb[j >> 1], sbuf[0][j & 1]);
        {
            float mx = sbuf[0][0][0];
#pragma unroll
            for (int i = 1; i < 32; ++i) mx = fmaxf(mx, PG_SVAL(sbuf[0], i));
            st.lrun = lrun;
            st.raise(fmaxf(st.mrun, xhalf_max(mx) * sc2));
            lrun = st.lrun;
        }
        float mrun = st.mrun;

        // tile n of the stretch; kind 2: two more follow it at least, 1: one, 0: it is the last
        auto iteration = [&](int n, auto par_c, auto kind_c) {
            constexpr int PAR = decltype(par_c)::value, kind = decltype(kind_c)::value;
            constexpr bool has_next = kind != 0;
            constexpr uint32_t kbuf = L::kK + (uint32_t)(PAR ^ 1) * L::kMat;
            constexpr uint32_t vbuf = L::kV + (uint32_t)PAR * L::kMat;
            f32x16* scur = sbuf[PAR];
            f32x16* snext = sbuf[PAR ^ 1];
            dn_wait_tiles();
            if (has_next || ready) stage(vg, x, L::kV + (uint32_t)(PAR ^ 1) * L::kMat);
            if (kind == 2 || (kind == 1 && ready)) {
                x = places(next.x, next.y, 0);
                stage(kg, x, L::kK + (uint32_t)PAR * L::kMat);
                if (kind == 2) next = look(n + 3);         // of the last step: a place behind the stretch's, not used
            }
            float psum = 0.f;
            if (has_next) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int v = 0; v < 16; ++v) snext[t][v] = 0.f;
#pragma unroll
                for (int j = 0; j < kAhead; ++j) ring[j % kRing] = read_k(kbuf, j);
            } else {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) ring[(NA + j) % kRing] = read_v(vbuf, j);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NA; ++j) {
                if (has_next) {
                    const int ja = j + kAhead;
                    if (ja < NA) ring[ja % kRing] = read_k(kbuf, ja);
                    else ring[ja % kRing] = read_v(vbuf, ja - NA);
                    snext[j & 1] = E::mfma32(ring[j % kRing], qb[j >> 1], snext[j & 1]);
                }
#pragma unroll
                for (int i = kVA * j; i < kVA * (j + 1); ++i) {
                    const float e = fast_exp2(fmaf(PG_SVAL(scur, i), sc2, -mrun));
                    psum += e;
                    PG_SVAL(scur, i) = e;
                }
#pragma unroll
                for (int i = kVA * j; i < kVA * (j + 1); i += 2) pb[i >> 3][(i >> 1) & 3] = pack2<E>(PG_SVAL(scur, i), PG_SVAL(scur, i + 1));
                __builtin_amdgcn_sched_barrier(0);
            }
            lrun += psum;
            float mx = has_next ? snext[0][0] : 0.f;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (j + kAhead < NP) ring[(NA + j + kAhead) % kRing] = read_v(vbuf, j + kAhead);
                st.o[j >> 2] = E::mfma32(ring[(NA + j) % kRing], pb[j & 3], st.o[j >> 2]);
                if (has_next) {
#pragma unroll
                    for (int i = kVP * j; i < kVP * (j + 1); ++i) mx = fmaxf(mx, PG_SVAL(snext, i));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (has_next) {
                const float mnew = fmaxf(mrun, xhalf_max(mx) * sc2);
                if (__builtin_amdgcn_ballot_w64(mnew > mrun) != 0) {
                    const float alpha = fast_exp2(mrun - mnew);
                    lrun *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int v = 0; v < 16; ++v) st.o[dt][v] *= alpha;
                    mrun = mnew;
                }
            }
        };
        using c0 = std::integral_constant<int, 0>;
        using c1 = std::integral_constant<int, 1>;
        using c2 = std::integral_constant<int, 2>;
        int n = 0;
        for (; n + 2 < here; n += 2) {
            iteration(n, c0{}, c2{});
            iteration(n + 1, c1{}, c2{});
        }
        iteration(n, c0{}, c1{});
        iteration(n + 1, c1{}, c0{});
#undef PG_SVAL
        st.mrun = mrun;
        st.lrun = lrun;
        st.seen = true;
    }

    // ---- tiles seen in part
    if (rest > 0) {
        const int G = d.H / d.kv_heads, w0 = p.row0 + wave * 32, w1 = min(w0 + 31, p.row1 - 1);
        const bool idle = w0 >= p.row1;
        // what the wave's rows see at most and at least
        const int e0 = idle || !d.causal ? p.k.end_max : (int)min((int64_t)p.rq.past + w0 / G + 1, (int64_t)a.cap);
        const int e1 = idle || !d.causal ? p.k.end_max : (int)min((int64_t)p.rq.past + w1 / G + 1, (int64_t)a.cap);
        const int lo = d.window && e1 > d.window ? e1 - d.window : 0;
        const RowMask mask = lane_mask(a, p, w0);
        // places: behind those of the last stretch's whole tiles, as far as they went with it
        int base = ready ? (nf - 1) % RowsLds<D, NW>::kStretch + 1 : 0, held = ready ? min(rest, RowsLds<D, NW>::kStretch - base) : 0, first = 0;
        for (int u = 0; u < rest; ++u) {
            if (u == first + held) {               // the next stretch of them; nothing is on its way, and everybody is done with the last
                first = u;
                base = 0;
                held = min(rest - u, RowsLds<D, NW>::kStretch);
                fill(nf + u, held);
                const u32x2 w = where[lane & 7];
                const Places x = places(w.x, w.y, 0);
                stage(kg, x, L::kK + (uint32_t)(u & 1) * L::kMat);
                stage(vg, x, L::kV + (uint32_t)(u & 1) * L::kMat);
            }
            int pos[8];
            {
                uint32_t off8;
                int mine;
                map.entry(8 * tile_at(nf + u) + (lane & 7), &off8, &mine);
#pragma unroll
                for (int b = 0; b < 8; ++b) pos[b] = __builtin_amdgcn_readlane(mine, b);
            }
            const uint32_t buf = (uint32_t)(u & 1) * L::kMat, other = (uint32_t)(~u & 1) * L::kMat;
            dn_wait_tiles();
            if (u + 1 < first + held) {
                const u32x2 w = where[8 * (base + u + 1 - first) + (lane & 7)];
                const Places x = places(w.x, w.y, 0);
                stage(kg, x, L::kK + other);
                stage(vg, x, L::kV + other);
            }
            bool some = false, all = true;
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                some = some || pos[b] < e1;
                all = all && pos[b] < e0 - 7 && (pos[b] >= lo || pos[b] + 7 < d.sink);
            }
            if (!idle && some)
                masked_tile<E, D, 2>(lds, L::kK + buf, L::kV + buf, qb, sc2, st, mask, !all, pos, [] {}, [&]() { return all ? (uint64_t)0 : odd_rows<E, D, 1>(lds, L::kV + buf, 0); });
        }
    }
    __syncthreads();                               // the tiles are dead: rows leave through LDS
    store_rows<E, D>(a, p, st, bad, p.row0 + wave * 32, chunk, chunks, part, lds + wave * 32 * (2 * D + 16));
}

// ---- other types and head sizes --------------------------------------------------------------------------------------------------
//
// fp32 tensors, head sizes other than 64 and 128, without matrix instructions.  A workgroup takes a piece of 4 rows and 256 positions at a
// time: a thread one position's logits of the four rows, then 16 bytes of every so many V rows, so that each K and V row is read once
// per piece.  32 tokens on 4000 positions, 16 heads of 256 on 4, bf16: 193 us, 2.7 TB/s, the threads' loads of whole K rows (lines that 16
// loads of a thread share) ahead of the arithmetic; 1000 tokens on 4000 before them, 12 heads of 96: 790 us, fp32 multiplications.
constexpr int kAnyRows = 4;

template <typename T>
__global__ __launch_bounds__(256) void paged_generic_kernel(PagedArgs a, int64_t npieces, int chunks, int chunk_tiles, float* part) {
    constexpr int N = Chunk<T>::kN, M = kAnyRows, kEsz = 16 / N;
    __shared__ float qs[M][256];
    __shared__ f32x4 ws[256];                      // a position's weights, -1 in rows that do not see it
    __shared__ int64_t at[256];                    // a position's row in a head's rows of the pools, in bytes; -1 where nobody sees it
    __shared__ float red[4][M], sums[4][M];
    __shared__ float sum[256 * N];
    const sfm_paged_desc& d = a.d;
    const int tid = threadIdx.x, wave = tid >> 6, D = d.D, G = d.H / d.kv_heads;
    const int kh = blockIdx.x % d.kv_heads, rest = blockIdx.x / d.kv_heads, chunk = rest % chunks;
    Piece p;
    if (!find_piece<M>(a, rest / chunks, kh, &p)) return;
    const int v0 = min(chunk * chunk_tiles, p.k.tiles) * 64, v1 = min(chunk * chunk_tiles + chunk_tiles, p.k.tiles) * 64;
    const BlockMap map = block_map(a, p, kEsz);
    RowMask mask[M];
#pragma unroll
    for (int r = 0; r < M; ++r) mask[r] = row_mask(a, p, min(p.row0 + r, p.row1 - 1));
    for (int i = tid; i < M * D; i += 256) {
        const int r = i / D, x = i - r * D, row = min(p.row0 + r, p.row1 - 1), t = row / G;
        qs[r][x] = PElem<T>::get(a.q, (int64_t)(p.rq.first + t) * d.q_stride[0] + (int64_t)(kh * G + row - t * G) * d.q_stride[1] + x);
    }
    const char* const kg = (const char*)a.kp + (int64_t)kh * d.pool_stride[2] * kEsz;
    const char* const vg = (const char*)a.vp + (int64_t)kh * d.pool_stride[2] * kEsz;
    const int nc = D / N, groups = 256 / nc, g = tid / nc, c = tid - g * nc;           // of V: 16 bytes c of positions g, g + groups, ...
    const float sc2 = d.sm_scale * kLog2e;
    float mrun[M], lrun[M], acc[M][N];
    bool seen[M], bad = p.k.beyond;
#pragma unroll
    for (int r = 0; r < M; ++r) {
        mrun[r] = -__FLT_MAX__;
        lrun[r] = 0.f;
        seen[r] = false;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[r][i] = 0.f;
    }
    for (int p0 = v0; p0 < v1; p0 += 256) {
        const int v = p0 + tid;
        int64_t row = -1;
        int pos = kNoPos;
        if (v < v1) {
            uint32_t off8;
            const int e = map.entry(v >> 3, &off8, &pos), page = map.page(e);
            bad = bad || (e >= 0 && page < 0);
            if (page >= 0) row = map.offset(page, off8) + (v & 7) * (d.pool_stride[1] * kEsz);
            pos += v & 7;
        }
        __syncthreads();                           // the last step's weights are used; the queries are there
        float z[M] = {0.f, 0.f, 0.f, 0.f};
        if (row >= 0) {
#pragma unroll 4
            for (int x = 0; x < nc; ++x) {
                float k[N];
                Chunk<T>::get(*(const u32x4*)(kg + row + 16 * x), k);
#pragma unroll
                for (int r = 0; r < M; ++r)
#pragma unroll
                    for (int i = 0; i < N; ++i) z[r] = fmaf(qs[r][x * N + i], k[i], z[r]);
            }
        }
        bool see[M];
#pragma unroll
        for (int r = 0; r < M; ++r) {
            see[r] = row >= 0 && mask[r].sees(pos);
            seen[r] = seen[r] || see[r];
            z[r] = see[r] ? z[r] * sc2 : -INFINITY;
            float m = z[r];
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            if ((tid & 63) == 0) red[wave][r] = m;
        }
        at[tid] = row;
        __syncthreads();
        f32x4 w;
#pragma unroll
        for (int r = 0; r < M; ++r) {
            const float mnew = fmaxf(fmaxf(mrun[r], fmaxf(red[0][r], red[1][r])), fmaxf(red[2][r], red[3][r]));
            const float e = see[r] ? exp2f(z[r] - mnew) : 0.f, alpha = exp2f(mrun[r] - mnew);
            w[r] = see[r] ? e : -1.f;
            lrun[r] = lrun[r] * alpha + e;
            mrun[r] = mnew;
#pragma unroll
            for (int i = 0; i < N; ++i) acc[r][i] *= alpha;
        }
        ws[tid] = w;
        __syncthreads();
        const int count = min(256, v1 - p0);
        if (g < groups)
#pragma unroll 4
            for (int x = g; x < count; x += groups) {
                if (at[x] < 0) continue;
                const f32x4 wx = ws[x];
                float val[N];
                Chunk<T>::get(*(const u32x4*)(vg + at[x] + 16 * c), val);
#pragma unroll
                for (int r = 0; r < M; ++r)
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[r][i] = wx[r] < 0.f ? acc[r][i] : fmaf(wx[r], val[i], acc[r][i]);
            }
    }
    bad = __syncthreads_or(bad);
#pragma unroll
    for (int r = 0; r < M; ++r) {
        float l = lrun[r];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
        if ((tid & 63) == 0) sums[wave][r] = l;
    }
#pragma unroll
    for (int r = 0; r < M; ++r) {
        if (g < groups)
#pragma unroll
            for (int i = 0; i < N; ++i) sum[(g * nc + c) * N + i] = acc[r][i];
        const bool any = __syncthreads_or(seen[r]);
        const int row = p.row0 + r, t = p.rq.first + row / G, h = kh * G + row % G;
        if (row < p.row1) {
            const float l = sums[0][r] + sums[1][r] + sums[2][r] + sums[3][r];
            const int64_t rows = d.tokens * d.H, to = chunk * rows + (int64_t)t * d.H + h;
            float o = 0.f;
            if (tid < D)
                for (int j = 0; j < groups; ++j) o += sum[j * D + tid];
            if (part != nullptr) {
                if (any && tid < D) part[to * D + tid] = o;
                if (tid == 0) store_partial(part + chunks * rows * D + to * 2, mrun[r], l, any, bad);
            } else {
                if (tid < D) PElem<T>::put(a.out, (int64_t)t * d.o_stride[0] + (int64_t)h * d.o_stride[1] + tid, bad ? NAN : any ? o / l : 0.f);
                if (a.lse != nullptr && tid == 0) a.lse[(int64_t)h * d.tokens + t] = bad ? NAN : any ? (mrun[r] + log2f(l)) * kLn2 : -INFINITY;
            }
        }
        __syncthreads();
    }
}

// Combines the partials of a row: D / 4 lanes hold four channels each.  Bound by reading the partials once.  SIZE 0: any head size
template <class T, int SIZE>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a, const float* __restrict__ part, int chunks) {
    const sfm_paged_desc& d = a.d;
    const int D = SIZE ? SIZE : d.D, CH = D / 4, per = 256 / CH, mine = threadIdx.x / CH, ch = threadIdx.x - mine * CH;
    const int64_t rows = d.tokens * d.H, row = (int64_t)blockIdx.x * per + mine;
    if (mine >= per || row >= rows) return;
    const int64_t t = row / d.H;
    const int h = (int)(row - t * d.H);
    if (!d.zero_rest && t >= clamp_int(a.q_start[d.requests], 0, (int)d.tokens)) return;       // rows of nobody
    const float* const ml = part + chunks * rows * D + row * 2;
    float M = -__FLT_MAX__, sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) M = ml[c * rows * 2 + 1] == 0.f ? M : fmaxf(M, ml[c * rows * 2]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    bool seen = false;
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) {
        const float l = ml[c * rows * 2 + 1];
        if (l == 0.f) continue;                    // nothing was seen, nor written
        seen = true;
        const float f = fast_exp2(ml[c * rows * 2] - M);
        sum += f * l;
        o += *(const f32x4*)(part + (c * rows + row) * D + 4 * ch) * f;
    }
    const float inv = seen ? 1.f / sum : 0.f;                          // NaN sums make the row NaN
    PElem<T>::put4(a.out, t * d.o_stride[0] + h * d.o_stride[1] + 4 * ch, o * inv);
    if (a.lse != nullptr && ch == 0) a.lse[(int64_t)h * d.tokens + t] = seen ? (M + log2f(sum)) * kLn2 : -INFINITY;
}

// Which kernel a call takes, and in how many ranges of tiles.
struct PagedPlan {
    int rows;                      // of a piece; 0: the shape-generic kernel
    int64_t pieces;
    int chunks, chunk_tiles;
    bool once;                     // few rows: the cache is read past the caches
    bool paired;                   // many rows, causal: long and short pieces share a compute unit
};
static PagedPlan paged_plan(const sfm_paged_desc& d) {
    PagedPlan p{0, 0, 1, 0, false, false};
    const int64_t G = d.H / d.kv_heads, cu = cu_count();
    // rows of a request (of a group of tokens) and key head, on average, and pieces that have rows
    const int64_t mean = std::max<int64_t>(1, d.top ? std::min<int64_t>(d.group, d.tokens) * G : d.tokens * G / d.requests);
    const int64_t units = d.top ? (d.tokens + d.group - 1) / d.group : std::min<int64_t>(d.requests, d.tokens);
    // 256 rows a workgroup read every tile once per compute unit, 128 twice, with two of them on it: 4 to 7 % slower where both fill
    // the chip (4680 x 32760 of 12 heads 937 us and 988), but workgroups of 128 rows fill it better: taken where those of 256 would
    // leave an eighth of it idle in their last round (four requests of 1024 tokens on 15000, 16 heads on 4: 856 us and 712)
    auto wide = [&](int64_t n) {
        const double rounds = n * 1.03 / cu;
        return mean > 128 && (int64_t)rounds + 1 < 1.15 * rounds;
    };
    auto items = [&](int64_t rows) { return units * ((mean + rows - 1) / rows) * d.kv_heads; };
    // Causal prompts without much before them: a head's last piece has twice the mean's keys, and where all pieces are on the chip at once it
    // alone sets the time.  Two pieces of 128 rows to a compute unit can be a long and a short one (4680 tokens, 12 heads, 142 us -> 127; four
    // requests of 1024 on 1024, 92 -> 79); with more pieces than that the order of their lengths balances them better (8192 tokens, 32 heads
    // on 8, 556 us and 586), and behind a long cache they are much alike.
    const int64_t cap = (int64_t)d.width * d.page_size;
    const bool prompts = d.causal && !d.top && mean > 128 && items(128) <= 2 * cu, mfma = d.dtype != SFM_F32 && (d.D == 64 || d.D == 128);
    p.rows = !mfma ? 0 : mean <= 32 ? 32 : wide(items(256)) && !(prompts && cap <= 4 * d.tokens / d.requests) ? 256 : 128;
    p.paired = prompts && p.rows == 128;
    const int64_t per = mfma ? p.rows : kAnyRows;
    p.pieces = d.top ? pieces(d.tokens, d.group, d.requests) * ((std::min<int64_t>(d.group, d.tokens) * G + per - 1) / per) : pieces(d.tokens * G, per, d.requests);
    const int64_t tiles = d.top ? ((int64_t)d.top * d.page_size + 63) / 64 : most_tiles(per, G, d.tokens, d.causal, d.window, d.sink, cap), n = items(per);
    int64_t chunks = 1;
    if (!mfma) {               // a step is 256 positions; one token on 1560, 12 heads of 128 fp32: in 7 ranges 33 us, in 2 76
        chunks = std::min<int64_t>((4 * cu + n - 1) / n, (tiles + 3) / 4);
    } else if (p.rows == 32) {
        chunks = std::min<int64_t>((8 * cu + n - 1) / n, (tiles + 7) / 8);
        // More rows than twice the memory-side cache (256 MB) holds, most of them read once: past it, 848 MB (up to 2 GB by the table's width)
        // 193 -> 175 us; 134 MB that lie in it 38 -> 44.  A request's second piece reads its rows again.  Lengths are not known here, but the
        // further apart they are the more of the rows are in such pieces: 32 requests on 15000 positions, 8 key heads, with 4 rows each 340 us
        // in place of 376, with the same number but 97 in one request 356 (382); with 16 rows 376 (402), with 481 in one 493 (458);
        // with 31 rows 406 (435), with 961 in one 656 (542).
        p.once = (mean <= 16 || d.tokens <= d.requests) && n * tiles * 64.0 * d.D * 4 > 512e6;
        // Selected pages make rows equally long.  Where those of half the chip's compute units or more are few and fit the memory-side cache, one
        // range of all of them is as fast as ranges that are joined, or faster: 32 tokens, 8 key heads of 64, 1024 positions each, pages from
        // memory, 26.5 us and 33.2 (pages from the caches 18.4 and 26.4); 16 tokens, 128, 2048 each 42.9 and 42.5 (29.5 and 34.1).  Beyond, the longest
        // chain of loads sets the time: 64 tokens, 4096 positions each, 128: 249 and 209 (238 and 191), 64: 170 and 128 (157 and 115).
        if (d.top && n >= cu / 2 && tiles <= 40 && n * tiles * 64.0 * d.D * 4 <= 256e6) chunks = 1;
    } else if (p.rows == 128 && tiles >= 16) {                        // 256 rows are taken only where their pieces fill the chip
        const double scale = d.D == 64 ? 0.6 : 1.0, partial_ns = (double)d.H * d.tokens * (d.D + 2) * 8 / 3500;
        double t1 = 0, best = 0;
        for (int64_t s = 1; s <= 64 && s <= tiles / 4 && (s == 1 || n * s <= 2 * cu); ++s) {
            const double tile_ns = n * s <= cu ? 1100 : 1900;
            double t = 5000 + (double)((tiles + s - 1) / s) * tile_ns * scale;
            if (s == 1) t1 = best = t;
            else t += 6000 + s * partial_ns;
            if (t < best && t < 0.9 * t1) {
                chunks = s;
                best = t;
            }
        }
    }
    chunks = std::max<int64_t>(1, std::min<int64_t>(chunks, 64));
    p.chunk_tiles = (int)((tiles + chunks - 1) / chunks);
    if (!mfma) p.chunk_tiles = (p.chunk_tiles + 3) / 4 * 4;            // whole steps
    p.chunks = (int)((tiles + p.chunk_tiles - 1) / p.chunk_tiles);
    return p;
}

size_t paged_workspace_bytes(const sfm_paged_desc& d) {
    const PagedPlan p = paged_plan(d);
    return p.chunks < 2 ? 0 : (size_t)p.chunks * d.tokens * d.H * (d.D + 2) * sizeof(float);
}

void paged_attention_plan(const sfm_paged_desc& d, int32_t* rows, int32_t* ranges, int32_t* past_caches) {
    const PagedPlan p = paged_plan(d);
    *rows = p.rows;
    *ranges = p.chunks;
    *past_caches = p.once;
}

static int launch_status() {
    const hipError_t err = hipGetLastError();
    if (err == hipSuccess) return SFM_OK;
    set_error("hip launch failed: %s", hipGetErrorString(err));
    return SFM_ERR_HIP;
}

template <class T, int SIZE>
static int launch_merge(const PagedArgs& a, const PagedPlan& p, const float* part, hipStream_t stream) {
    const int64_t rows = a.d.tokens * a.d.H, per = 1024 / a.d.D;
    if (part != nullptr) hipLaunchKernelGGL((paged_merge_kernel<T, SIZE>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, stream, a, part, p.chunks);
    return launch_status();
}

template <class T>
static int launch_generic(const PagedArgs& a, const PagedPlan& p, float* part, hipStream_t stream) {
    hipLaunchKernelGGL(paged_generic_kernel<T>, dim3((unsigned)(p.pieces * a.d.kv_heads * p.chunks)), dim3(256), 0, stream, a, p.pieces, p.chunks, p.chunk_tiles, part);
    return launch_merge<T, 0>(a, p, part, stream);
}

template <class E, int D>
static int launch_mfma(const PagedArgs& a, const PagedPlan& p, float* part, hipStream_t stream) {
    const sfm_paged_desc& d = a.d;
    const int64_t total = p.pieces * d.kv_heads * p.chunks;
    auto go = [&](auto kern, int nw, size_t lds) -> int {
        const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) {
            set_error("hipFuncSetAttribute failed: %s", hipGetErrorString(e));
            return SFM_ERR_HIP;
        }
        hipLaunchKernelGGL(kern, dim3(xcd_grid((int)total)), dim3(64 * nw), lds, stream, a, p.pieces, p.chunks, p.chunk_tiles, part, p.paired);
        return SFM_OK;
    };
    const int rc = p.rows == 32 ? go(p.once ? paged_few_kernel<E, D, true> : paged_few_kernel<E, D, false>, 4, FewLds<D>::kTotal + 4 * 96 * sizeof(float))
                   : p.rows == 128 ? go(paged_rows_kernel<E, D, 4>, 4, RowsLds<D, 4>::kTotal) : go(paged_rows_kernel<E, D, 8>, 8, RowsLds<D, 8>::kTotal);
    return rc ? rc : launch_merge<E, D>(a, p, part, stream);
}

int launch_paged_attention(const sfm_paged_desc& d, const void* q, const void* kp, const void* vp, const int32_t* table,
                           const int32_t* past, const int32_t* q_start, const int32_t* selected, void* out, float* lse, void* workspace,
                           size_t workspace_bytes, hipStream_t stream) {
    PagedArgs a{d, fast_div(d.page_size / 8), d.width * d.page_size, q, kp, vp, table, past, q_start, selected, out, lse};
    PagedPlan p = paged_plan(d);
    if (p.chunks > 1 && (!workspace || workspace_bytes < paged_workspace_bytes(d))) {          // whole, then
        p.chunk_tiles *= p.chunks;
        p.chunks = 1;
    }
    const int64_t total = p.pieces * d.kv_heads * p.chunks;
    if (total >= (1 << 23)) {
        set_error("%lld pieces of rows, heads and ranges are more than a launch takes", (long long)total);
        return SFM_ERR_UNSUPPORTED;
    }
    float* const part = p.chunks > 1 ? (float*)workspace : nullptr;
    if (!p.rows) return d.dtype == SFM_BF16 ? launch_generic<BF16>(a, p, part, stream) : d.dtype == SFM_F16 ? launch_generic<F16>(a, p, part, stream) : launch_generic<float>(a, p, part, stream);
    if (d.dtype == SFM_BF16) return d.D == 128 ? launch_mfma<BF16, 128>(a, p, part, stream) : launch_mfma<BF16, 64>(a, p, part, stream);
    return d.D == 128 ? launch_mfma<F16, 128>(a, p, part, stream) : launch_mfma<F16, 64>(a, p, part, stream);
}

}  // namespace sfm
