// The paged cache's bookkeeping: block tables and slots from request lengths, new rows into their pages with the pages' mean
// keys, and the selection of pages by those.  (The attention over pages is paged_attn.hip's.)
#include <algorithm>

#include "paged_rules.hpp"
#include "rows8.hpp"

namespace sfm {

// ------------------------------------------------------------------------------------------------
// plan
// ------------------------------------------------------------------------------------------------
struct PlanArgs {
    int R, W;
    FastDiv page8;             // page_size / 8
    int64_t T, table_stride, free_count;
    int32_t* table;
    const int32_t *past, *fresh, *free_pages, *taken;
    int32_t *q_start, *lengths, *next_free;
    int64_t* slots;
    int32_t *ws_tokens, *ws_pages;     // [R + 1] prefix sums, more requests than a workgroup keeps in LDS
};

// Two prefix sums over the requests (tokens, pages that they open), then a search per new token and per opened page.  Bound by launch and by the
// sums' latency: 4.3 us for 16 requests, 6.7 for 333 of 33866 tokens, 12.7 for 6000 of 179251.
//
// A workgroup keeps this many requests' sums in LDS (8 bytes each): up to here every workgroup forms all the sums for itself,
// which is one launch and no wait between workgroups.
constexpr int kPlanLds = 8192;

// Exclusive sum over the workgroup's threads; *total gets the sum of all.
template <int NT>
__device__ __forceinline__ int64_t plan_scan(int64_t v, int64_t* red, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) red[wave] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w < wave) before += red[w];
        all += red[w];
    }
    *total = all;
    return before + x - v;
}

__device__ __forceinline__ int64_t plan_entries(int64_t pos, const PlanArgs& a) {      // ceil(pos / page), at most W
    const int64_t cap = (int64_t)a.W * a.page8.d * 8;
    const uint32_t b = (uint32_t)((pos < cap ? pos : cap) + 7) / 8, e = quot(b, a.page8);
    return e + (e * a.page8.d < b);
}

// at[0 .. n) becomes its exclusive sum, at most `most`, and at[n] the whole of it
template <int NT>
__device__ __forceinline__ void plan_prefix(int32_t* at, int n, int64_t most, int64_t* red) {
    const int per = (n + NT - 1) / NT, i0 = min((int)threadIdx.x * per, n), i1 = min(i0 + per, n);
    int64_t sum = 0, total;
    for (int i = i0; i < i1; ++i) sum += at[i];
    int64_t before = plan_scan<NT>(sum, red, &total);
    for (int i = i0; i < i1; ++i) {
        const int v = at[i];
        at[i] = (int32_t)min(before, most);
        before += v;
    }
    if (threadIdx.x == 0) at[n] = (int32_t)min(total, most);
    __syncthreads();
}

// tokens[r] = first row of request r (at most T), pages[r] = pages that the requests before r open; r = 0 .. R.  The lengths are
// read in whole lines and independently of each other; a thread sums a run of them.
template <int NT>
__device__ void plan_sums(const PlanArgs& a, int32_t* tokens, int32_t* pages) {
    __shared__ int64_t red[NT / 64];
#pragma unroll 8
    for (int r = threadIdx.x; r < a.R; r += NT) tokens[r] = max(a.fresh[r], 0);
    __syncthreads();
    plan_prefix<NT>(tokens, a.R, a.T, red);
#pragma unroll 8
    for (int r = threadIdx.x; r < a.R; r += NT) {
        const int64_t past = max(a.past[r], 0), len = past + tokens[r + 1] - tokens[r];
        pages[r] = (int32_t)(plan_entries(len, a) - plan_entries(past, a));
    }
    __syncthreads();
    plan_prefix<NT>(pages, a.R, 0x7fffffff, red);        // fewer pages are wanted than tokens planned, T < 2^31
}

// the last r in [0, n) with at[r] <= v (at[0] = 0 <= v, ascending)
__device__ __forceinline__ int plan_find(const int32_t* at, int n, int v) {
    int lo = 0;
    while (n - lo > 1) {
        const int mid = (lo + n) >> 1;
        if (at[mid] <= v) lo = mid;
        else n = mid;
    }
    return lo;
}

__device__ __forceinline__ int32_t plan_page(const PlanArgs& a, int64_t i) {      // the i-th page that this call opens
    const int64_t j = i + (a.taken ? max(a.taken[0], 0) : 0);
    return j < a.free_count ? a.free_pages[j] : -1;
}

__device__ void plan_fill(const PlanArgs& a, const int32_t* tokens, const int32_t* pages) {
    const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
    const int wanted = pages[a.R], planned = tokens[a.R];
    for (int64_t r = tid; r <= a.R; r += step) {
        a.q_start[r] = tokens[r];
        if (r < a.R) a.lengths[r] = (int32_t)min((int64_t)max(a.past[r], 0) + tokens[r + 1] - tokens[r], (int64_t)0x7fffffff);
        else a.next_free[0] = (int32_t)min((int64_t)wanted + (a.taken ? max(a.taken[0], 0) : 0), (int64_t)0x7fffffff);
    }
    for (int64_t i = tid; i < wanted; i += step) {
        const int r = plan_find(pages, a.R + 1, (int)i);
        a.table[r * a.table_stride + plan_entries(max(a.past[r], 0), a) + (i - pages[r])] = plan_page(a, i);
    }
    const int64_t cap = (int64_t)a.W * a.page8.d * 8;
    for (int64_t t = tid; t < a.T; t += step) {
        int64_t slot = -1;
        if (t < planned) {
            const int r = plan_find(tokens, a.R + 1, (int)t);
            const int64_t past = max(a.past[r], 0), pos = past + t - tokens[r];
            if (pos < cap) {
                const uint32_t e = quot((uint32_t)pos / 8, a.page8);
                const int64_t opened = (int64_t)e - plan_entries(past, a);
                // an entry of this call's is taken from the list, where another workgroup takes it from too
                const int32_t page = opened >= 0 ? plan_page(a, pages[r] + opened) : a.table[r * a.table_stride + e];
                if (page >= 0) slot = (int64_t)page * a.page8.d * 8 + (pos - (int64_t)e * a.page8.d * 8);
            }
        }
        a.slots[t] = slot;
    }
}

template <int NT>
__global__ __launch_bounds__(NT) void paged_plan_kernel(PlanArgs a) {
    extern __shared__ int32_t plan_lds[];
    plan_sums<NT>(a, plan_lds, plan_lds + a.R + 1);
    plan_fill(a, plan_lds, plan_lds + a.R + 1);
}
__global__ __launch_bounds__(1024) void paged_plan_sums_kernel(PlanArgs a) { plan_sums<1024>(a, a.ws_tokens, a.ws_pages); }
__global__ __launch_bounds__(256) void paged_plan_fill_kernel(PlanArgs a) { plan_fill(a, a.ws_tokens, a.ws_pages); }

static int launched() {
    const hipError_t err = hipGetLastError();
    if (err == hipSuccess) return SFM_OK;
    set_error("hip launch failed: %s", hipGetErrorString(err));
    return SFM_ERR_HIP;
}

size_t paged_plan_workspace_bytes(int R) { return R <= kPlanLds ? 0 : 2 * ((size_t)R + 1) * sizeof(int32_t); }

int launch_paged_plan(int R, int W, int page_size, int64_t T, int32_t* table, int64_t table_stride, const int32_t* past,
                      const int32_t* fresh, const int32_t* free_pages, int64_t free_count, const int32_t* taken, int32_t* q_start,
                      int32_t* lengths, int64_t* slots, int32_t* next_free, void* workspace, hipStream_t stream) {
    PlanArgs a{R, W, fast_div(page_size / 8), T, table_stride, free_count, table, past, fresh, free_pages, taken, q_start, lengths, next_free, slots,
               (int32_t*)workspace, (int32_t*)workspace + R + 1};
    const int64_t items = T > R + 1 ? T : R + 1;
    auto wgs = [&](int threads) { return dim3((unsigned)std::min<int64_t>(std::max<int64_t>((items + threads - 1) / threads, 1), 1024)); };
    const size_t lds = 2 * ((size_t)R + 1) * sizeof(int32_t);
    if (R <= 1024) {
        hipLaunchKernelGGL(paged_plan_kernel<256>, wgs(256), dim3(256), lds, stream, a);
    } else if (R <= kPlanLds) {
        hipLaunchKernelGGL(paged_plan_kernel<1024>, wgs(1024), dim3(1024), lds, stream, a);
    } else {
        hipLaunchKernelGGL(paged_plan_sums_kernel, dim3(1), dim3(1024), 0, stream, a);
        hipLaunchKernelGGL(paged_plan_fill_kernel, wgs(256), dim3(256), 0, stream, a);
    }
    return launched();
}

// ------------------------------------------------------------------------------------------------
// write
// ------------------------------------------------------------------------------------------------
struct WriteArgs {
    int T, R, W, H, chunks, page, pages;           // chunks: 16 bytes each, of a row of a head
    FastDiv row, head;             // by the chunks of a token's row, and of a head's
    int copy;                      // tokens of a workgroup that copies
    int64_t table_stride, ps, ts, hs, ks, kh;      // in chunks (the table: in entries)
    const u32x4 *k, *v;
    u32x4 *kp, *vp;
    const int64_t* slots;
    const int32_t *table, *past, *q_start;
    float* means;
    int mean_wgs;
};

// The mean key of one page, of one head: the page'th that a step's requests write to.  A request of n tokens writes to at most
// (n - 1) / page_size + 2 pages; its first has number q_start / page_size + 2 r, which leaves it as many.  New rows are taken from
// k, whatever the copying workgroups have done by then.  The rows are summed by groups of lanes, a row each, joined in LDS in
// a fixed order.
template <typename E, int NT>
__device__ void write_mean(const WriteArgs& a, int number, int h) {
    constexpr int N = Chunk<E>::kN;
    __shared__ float part[NT * N];
    const int tid = threadIdx.x, groups = NT / a.chunks, g = tid / a.chunks, c = tid - g * a.chunks, D = a.chunks * N;
    auto first = [&](int i) { return (int64_t)clamp_int(a.q_start[i], 0, a.T) / a.page + 2 * (int64_t)i; };
    const int r = find_last(a.R, number, first);
    if (r >= a.R) return;
    const Request q = request_of(a.q_start, a.past, r, a.R, a.T);
    const int64_t e = q.past / a.page + (number - first(r));
    if (q.n == 0 || number < first(r) || e * a.page >= (int64_t)q.past + q.n || e >= a.W) return;
    const int page = a.table[r * a.table_stride + e];
    if (page < 0 || page >= a.pages) return;
    const int64_t base = e * a.page;
    const int rows = (int)min((int64_t)q.past + q.n - base, (int64_t)a.page), old = (int)max((int64_t)0, min((int64_t)rows, q.past - base));
    float sum[N], x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.f;
    if (g < groups) {
        // eight rows on their way at a time
        auto add = [&](const u32x4* from, int64_t stride, int j, int end) {
            for (; j < end; j += 8 * groups) {
                u32x4 w[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) w[u] = j + u * groups < end ? from[(j + u * groups) * stride] : u32x4{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    Chunk<E>::get(w[u], x);
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] += x[i];
                }
            }
        };
        add(a.kp + page * a.ps + h * a.hs + c, a.ts, g, old);
        add(a.k + (q.first + (base - q.past)) * a.ks + h * a.kh + c, a.ks, old + (groups - old % groups + g) % groups, rows);
    }
    __syncthreads();
    if (g < groups)
#pragma unroll
        for (int i = 0; i < N; ++i) part[(g * a.chunks + c) * N + i] = sum[i];
    __syncthreads();
    if (tid < D) {
        float s = 0.f;
        for (int j = 0; j < groups; ++j) s += part[j * D + tid];
        a.means[((int64_t)page * a.H + h) * D + tid] = s / (float)rows;
    }
}

// The first mean_wgs workgroups form means, the others copy 16 bytes per lane and tensor at a time.  Bound by the rows' bytes: two chunks of 4680
// rows of 12 heads of 128, 115 MB, 23.4 us with the means of their pages and 19 without (4.9 and 6 TB/s, some of them in the caches); 32 rows 4.5 us.
template <typename E, int NT>
__global__ __launch_bounds__(NT) void paged_write_kernel(WriteArgs a) {
    if ((int)blockIdx.x < a.mean_wgs) {
        const int piece = blockIdx.x / a.H, h = blockIdx.x - piece * a.H;
        write_mean<E, NT>(a, piece, h);
        return;
    }
    const int t0 = ((int)blockIdx.x - a.mean_wgs) * a.copy, n = min(a.T - t0, a.copy) * (int)a.row.d;
    const int64_t all = (int64_t)a.pages * a.page;
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint32_t tt = quot(i, a.row), x = i - tt * a.row.d, h = quot(x, a.head), c = x - h * a.head.d;
        const int64_t t = t0 + (int)tt, slot = a.slots[t];
        if (slot < 0 || slot >= all) continue;
        const uint32_t page = (uint32_t)slot / a.page;                 // slots are below 2^31
        const int64_t to = page * a.ps + (slot - (int64_t)page * a.page) * a.ts + h * a.hs + c, from = t * a.ks + h * a.kh + c;
        a.kp[to] = a.k[from];
        a.vp[to] = a.v[from];
    }
}

int launch_paged_write(const sfm_paged_desc& d, const void* k, const void* v, const int64_t* ks, void* kp, void* vp, const int64_t* slots,
                       const int32_t* table, const int32_t* past, const int32_t* q_start, float* means, hipStream_t stream) {
    const int n16 = d.dtype == SFM_F32 ? 4 : 8;
    WriteArgs a{(int)d.tokens, d.requests, d.width, d.kv_heads, d.D / n16, d.page_size, d.pages, fast_div(d.kv_heads * d.D / n16), fast_div(d.D / n16), 1, d.table_stride,
                d.pool_stride[0] / n16, d.pool_stride[1] / n16, d.pool_stride[2] / n16, ks[0] / n16, ks[1] / n16, (const u32x4*)k, (const u32x4*)v,
                (u32x4*)kp, (u32x4*)vp, slots, table, past, q_start, means, 0};
    const int64_t numbers = means ? d.tokens / d.page_size + 2 * (int64_t)d.requests : 0;
    // a page's mean is one workgroup's: sixteen waves for long pages, whose rows take it 4 rounds of loads instead of 13 (1560 rows)
    const int nt = means && d.page_size >= 256 ? 1024 : 256;
    a.copy = std::max(1, 4 * nt / (int)a.row.d);
    const int64_t wgs = numbers * a.H + ((int64_t)a.T + a.copy - 1) / a.copy;
    if (wgs * nt >= ((int64_t)1 << 32) || a.row.d >= (1 << 24)) {
        set_error("%lld rows of %d heads are more than a launch takes", (long long)d.tokens, d.kv_heads);
        return SFM_ERR_UNSUPPORTED;
    }
    a.mean_wgs = (int)(numbers * a.H);
    auto pick = [&](auto nt_c) {
        constexpr int NT = decltype(nt_c)::value;
        return d.dtype == SFM_BF16 ? paged_write_kernel<BF16, NT> : d.dtype == SFM_F16 ? paged_write_kernel<F16, NT> : paged_write_kernel<float, NT>;
    };
    auto kern = nt == 256 ? pick(std::integral_constant<int, 256>{}) : pick(std::integral_constant<int, 1024>{});
    hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(nt), 0, stream, a);
    return launched();
}

// ------------------------------------------------------------------------------------------------
// select
// ------------------------------------------------------------------------------------------------
// Two steps: scores of every candidate page into a workspace, then the best of a row.  Few rows (single tokens) are spread over the chip by
// their pages in the first, where the means' bytes are, and the second works from LDS.  Scores are sums of 64 bits: two programs that
// add in another order still agree on which page is ahead, as long as no two scores are level to 15 digits.
struct SelectArgs {
    sfm_paged_desc d;
    const void* q;
    const float* means;
    const int32_t *table, *past, *q_start;
    int32_t* selected;
    uint64_t* keys;                // [row - row0][kv head][width]: scores as integers in their order
    int first, last;
    int row0, rows;                // of this pass
    int chunk;                     // pages that a workgroup scores
    double* sums;                  // [row - row0][kv head][D]: the queries' sums, NULL: formed by whom they are for
};

// A score's bits in the order of the scores: NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint64_t select_key(double s) {
    if (!(s == s)) s = -INFINITY;
    const uint64_t b = (uint64_t)__double_as_longlong(s + 0.0);
    return b >> 63 ? ~b : b | ((uint64_t)1 << 63);
}

// The tokens of row `row` of the lists and the pages that they choose from; n = 0: nobody's.
struct SelectRow {
    int r, n, candidates;          // entries of the table's row that the last token sees
    int64_t t0, pages;             // first token; candidates, had the table room for them
    int left;                      // tokens of the request from t0 on
    int64_t end;                   // positions up to the first of them
};
__device__ __forceinline__ void select_pages_of(const SelectArgs& s, SelectRow& x) {
    x.n = min(x.left, s.d.group);
    x.pages = (x.end + (s.d.causal ? x.n : x.left) + s.d.page_size - 1) / s.d.page_size;
    x.candidates = x.n ? (int)min(x.pages, (int64_t)s.d.width) : 0;
}
__device__ __forceinline__ SelectRow select_row(const SelectArgs& s, int row) {
    const sfm_paged_desc& d = s.d;
    SelectRow x;
    Request rq;
    x.r = find_request(s.q_start, s.past, d.requests, (int)d.tokens, row, 1, d.group, &rq);
    const int64_t t0 = (row - first_piece(rq.first, 1, d.group, x.r)) * d.group;
    x.left = x.r < d.requests && t0 >= 0 && t0 < rq.n ? (int)(rq.n - t0) : 0;
    x.t0 = rq.first + t0;
    x.end = (int64_t)rq.past + t0;
    select_pages_of(s, x);
    return x;
}
// the i-th group after it, of the same request
__device__ __forceinline__ SelectRow select_row_behind(const SelectArgs& s, SelectRow x, int i) {
    const int64_t by = (int64_t)i * s.d.group;
    x.left = by < x.left ? (int)(x.left - by) : 0;
    x.t0 += by;
    x.end += by;
    select_pages_of(s, x);
    return x;
}

// Sum of the queries of `n` tokens from t0 on and of a key head's G query heads, in sum[0 .. D).  Chunk c of the rows g, g + groups, ...
// to a thread, U of them on their way at a time; `part` holds their sums.
template <typename E, int U>
__device__ __forceinline__ void sum_queries(const SelectArgs& s, int kh, int64_t t0, int n, double* part, double* sum) {
    constexpr int N = Chunk<E>::kN;
    const sfm_paged_desc& d = s.d;
    const int tid = threadIdx.x, G = d.H / d.kv_heads, chunks = d.D / N, groups = 256 / chunks, g = tid / chunks, c = tid - g * chunks;
    const uint32_t rows = (uint32_t)n * G;         // at most tokens * H, below 2^31
    double mine[N];
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) mine[k] = 0.0;
    if (g < groups)
        for (uint32_t j0 = g; j0 < rows; j0 += U * groups) {
            u32x4 w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t j = min(j0 + u * groups, rows - 1), t = j / (uint32_t)G, h = j - t * G;
                w[u] = ((const u32x4*)s.q)[((t0 + t) * d.q_stride[0] + (kh * G + (int64_t)h) * d.q_stride[1]) / N + c];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                Chunk<E>::get(w[u], v);
#pragma unroll
                for (int k = 0; k < N; ++k) mine[k] += j0 + u * groups < rows ? (double)v[k] : 0.0;
            }
        }
    __syncthreads();
    if (g < groups)
#pragma unroll
        for (int k = 0; k < N; ++k) part[g * d.D + c * N + k] = mine[k];
    __syncthreads();
    if (tid < d.D) {
        double t = 0.0;
        for (int j = 0; j < (int)min((uint32_t)groups, rows); ++j) t += part[j * d.D + tid];
        sum[tid] = t;
    }
}

// The sums of all rows, where many queries make one: the scores' workgroups would each add them up again.
template <typename E>
__global__ __launch_bounds__(256) void paged_sums_kernel(SelectArgs s) {
    __shared__ double part[256 * Chunk<E>::kN];
    const SelectRow x = select_row(s, s.row0 + blockIdx.x);
    if (x.candidates > s.d.top)
        sum_queries<E, 8>(s, blockIdx.y, x.t0, x.n, part, s.sums + ((int64_t)blockIdx.x * s.d.kv_heads + blockIdx.y) * s.d.D);
}

// The other lane's value, of the 16 of a DPP row
template <int CTRL>
__device__ __forceinline__ double row_lane(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
    return __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo));
}
// Sums over the 16 lanes of a DPP row, lane `sub` of them, of N = 4 or 16 values: lane l gets the sum of value l N / 16.  As long as there
// are values left to share out, two lanes exchange the half that the other keeps: 15 exchanges for 16 values in place of 64.  The lanes
// meet at distances 8, 7, 2 and 1 (by exclusive or), which every pair of lanes is a sum of once.
template <int N>
__device__ __forceinline__ double row_sums(double* x, int sub) {
    auto step = [&](auto ctrl_c, auto left_c, int bit) {
        constexpr int CTRL = decltype(ctrl_c)::value, LEFT = decltype(left_c)::value;
        if constexpr (LEFT > 1) {
#pragma unroll
            for (int j = 0; j < LEFT / 2; ++j) {
                const double a = x[j], b = x[j + LEFT / 2];
                x[j] = (sub & bit ? b : a) + row_lane<CTRL>(sub & bit ? a : b);
            }
        } else {
            x[0] += row_lane<CTRL>(x[0]);
        }
    };
    using std::integral_constant;
    step(integral_constant<int, 0x128>{}, integral_constant<int, N>{}, 8);                         // rotated by 8
    step(integral_constant<int, 0x141>{}, integral_constant<int, N / 2>{}, 4);                     // mirrored in each 8
    step(integral_constant<int, 0x4e>{}, integral_constant<int, (N > 4 ? N / 4 : 1)>{}, 2);        // two on, of four
    step(integral_constant<int, 0xb1>{}, integral_constant<int, (N > 8 ? N / 8 : 1)>{}, 1);
    return x[0];
}

// Scores of `chunk` pages for RT rows of one key head.  Sixteen lanes share a page, 4 of each 64 channels a lane; their queries' sums
// stay in registers, so that rows of one request (many groups of a prompt) read a mean once.  Eight tokens on caches of up to 50826 positions in pages
// of 32, 32 heads on 8 of 128: 36 MB in 10.4 us, a chain of trips to memory (request, table, means) behind the launch; 37 groups of a prompt on
// 512 pages, 12 heads, 13.
template <typename E, int NI, int RT>
__global__ __launch_bounds__(256) void paged_score_kernel(SelectArgs s) {
    constexpr int N = Chunk<E>::kN;
    __shared__ double part[256 * N];
    __shared__ double qsum[RT][256];
    const sfm_paged_desc& d = s.d;
    const int tid = threadIdx.x, sub = tid & 15;
    const int kh = blockIdx.y, tile = s.row0 + blockIdx.x * RT, end = min(tile + RT, s.row0 + s.rows), c0 = blockIdx.z * s.chunk;
    for (int row = tile; row < end;) {
        const SelectRow x = select_row(s, row);
        int count = 1;             // rows of the same request from here on
        SelectRow last = x;
        int most = x.candidates > d.top ? x.candidates : 0;
        while (RT > 1 && row + count < end) {
            const SelectRow y = select_row_behind(s, x, count);
            if (!y.n) break;
            last = y;
            most = max(most, y.candidates > d.top ? y.candidates : 0);
            ++count;
        }
        if (c0 < most) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (s.sums != nullptr) {
                    if (tid < d.D) qsum[i][tid] = i < count ? s.sums[((int64_t)(row + i - s.row0) * d.kv_heads + kh) * d.D + tid] : 0.0;
                } else {
                    sum_queries<E, 1>(s, kh, x.t0 + (int64_t)i * d.group, i < count ? (i == count - 1 ? last.n : d.group) : 0, part, qsum[i]);
                }
            }
            __syncthreads();
            double q[RT][NI * 4];
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int k = 0; k < NI * 4; ++k) {
                    const int ch = 64 * (k >> 2) + 4 * sub + (k & 3);
                    q[i][k] = ch < d.D ? qsum[i][ch] : 0.0;
                }
            uint64_t* const keys = s.keys + ((int64_t)(row - s.row0) * d.kv_heads + kh) * d.width;
            const int32_t* const table = s.table + x.r * d.table_stride;
            const int c1 = min(c0 + s.chunk, most);
            constexpr int U = 4;                                       // pages on their way at a time
            for (int e0 = c0 + (tid >> 4); e0 < c1; e0 += 16 * U) {
                int page[U];
                f32x4 w[U][NI];
#pragma unroll
                for (int u = 0; u < U; ++u) page[u] = e0 + 16 * u < c1 ? table[e0 + 16 * u] : -1;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool fine = page[u] >= 0 && page[u] < d.pages;
                    const float* const m = s.means + ((int64_t)(fine ? page[u] : 0) * d.kv_heads + kh) * d.D;
#pragma unroll
                    for (int i = 0; i < NI; ++i) w[u][i] = 64 * i + 4 * sub < d.D ? *(const f32x4*)(m + 64 * i + 4 * sub) : f32x4{0.f, 0.f, 0.f, 0.f};
                    if (!fine) page[u] = -1;
                }
                double dot[U * RT];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        double t = 0.0;
#pragma unroll
                        for (int k = 0; k < NI * 4; ++k) t = fma(q[i][k], (double)w[u][k >> 2][k & 3], t);
                        dot[u * RT + i] = t;
                    }
                const double score = row_sums<U * RT>(dot, sub);       // of this lane's page and row
                const int at = sub / (16 / (U * RT)), u = at / RT, i = at % RT, e = e0 + 16 * u;
                bool fine = false;
#pragma unroll
                for (int x = 0; x < U; ++x) fine = x == u ? page[x] >= 0 : fine;
                if (sub % (16 / (U * RT)) == 0 && i < count && e < c1) keys[(int64_t)i * d.kv_heads * d.width + e] = select_key(fine ? score : -INFINITY);
            }
            __syncthreads();
        }
        row += count;
    }
}

constexpr int kSelPages = 4096;                    // scores that are compared at a time, beside the best so far

// The best of a row.  Scores are taken kSelPages at a time; the best of them and of the `top` before are found by the keys' bits, eight at
// a time from the highest: a histogram says in which digit the top-th largest lies.  Level ones are taken in the order of their
// pages, which is kept throughout.  8.5 us for 64 of 512 pages, 10 for 64 of 1600: launch, request and scores one after the other, then three to
// eight digits of five barriers each.  Bits that all keys share are not skipped: finding them took as long.
__global__ __launch_bounds__(256) void paged_select_kernel(SelectArgs s) {
    extern __shared__ __attribute__((aligned(16))) char sel_lds[];
    const sfm_paged_desc& d = s.d;
    const int cap = d.top + kSelPages;
    uint64_t* const key = (uint64_t*)sel_lds;                      // [cap]
    int32_t* const entry = (int32_t*)(key + cap);                  // [cap]
    __shared__ int hist[256];
    __shared__ int wsum[4][2];
    __shared__ int pick[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = s.row0 + blockIdx.x / d.kv_heads, kh = blockIdx.x % d.kv_heads;
    int32_t* const out = s.selected + ((int64_t)row * d.kv_heads + kh) * d.top;
    const SelectRow x = select_row(s, row);
    const int P = x.candidates;
    if (P <= d.top) {
        for (int i = tid; i < d.top; i += 256) out[i] = i < P ? i : -1;
        return;
    }
    const uint64_t* const keys = s.keys + ((int64_t)(row - s.row0) * d.kv_heads + kh) * d.width;
    int kept = 0;                                                  // key[0 .. kept): the best so far, in the order of their entries
    for (int p0 = 0; p0 < P; p0 += kSelPages) {
        const int count = min(kSelPages, P - p0);
        for (int i = tid; i < count; i += 256) {
            const int e = p0 + i;
            key[kept + i] = e < s.first || e >= x.pages - s.last ? ~(uint64_t)0 : keys[e];      // above infinity's
            entry[kept + i] = e;
        }
        __syncthreads();
        const int have = kept + count;
        if (have <= d.top) {
            kept = have;
            continue;
        }
        // the top-th largest key: digits from the highest, `need` of those that agree so far
        int need = d.top;
        bool whole = false;                                        // all that agree are taken: no level ones to tell apart
        uint64_t prefix = 0;
        int shift = 56;
        for (; shift >= 0; shift -= 8) {
            hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < have; i += 256)
                if (shift == 56 || (key[i] >> (shift + 8)) == prefix) atomicAdd(&hist[(key[i] >> shift) & 255], 1);
            __syncthreads();
            // number of keys in digits above this thread's
            int c = hist[tid], above = c;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_down(above, o);
                if (lane + o < 64) above += y;
            }
            if (lane == 0) wsum[wave][0] = above;
            __syncthreads();
            for (int w = wave + 1; w < 4; ++w) above += wsum[w][0];
            above -= c;
            if (above < need && above + c >= need) {
                pick[0] = tid;
                pick[1] = above;
            }
            __syncthreads();
            prefix = prefix << 8 | (uint32_t)pick[0];
            need -= pick[1];
            whole = hist[pick[0]] == need;
            __syncthreads();
            if (whole) break;
        }
        const int low = whole ? shift : 0;                         // key >> low against prefix
        // keep them in order: every thread moves a run of the list; the moves go to lower places, after all have been read
        const int per = (have + 255) / 256, i0 = min(tid * per, have), i1 = min(i0 + per, have);
        int over = 0, level = 0;
        for (int i = i0; i < i1; ++i) {
            const uint64_t k = key[i] >> low;
            over += k > prefix;
            level += k == prefix;
        }
        int ao = over, al = level;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(ao, o), z = __shfl_up(al, o);
            if (lane >= o) ao += y, al += z;
        }
        if (lane == 63) wsum[wave][0] = ao, wsum[wave][1] = al;
        __syncthreads();
        for (int w = 0; w < wave; ++w) ao += wsum[w][0], al += wsum[w][1];
        ao -= over;
        al -= level;
        constexpr int kRun = (SFM_PAGED_TOP_MAX + kSelPages) / 256;
        uint64_t mk[kRun];
        int32_t me[kRun];
#pragma unroll
        for (int j = 0; j < kRun; ++j)
            if (i0 + j < i1) mk[j] = key[i0 + j], me[j] = entry[i0 + j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
            if (i0 + j >= i1) continue;
            const uint64_t k = mk[j] >> low;
            if (k < prefix) continue;
            const bool take = k > prefix || al < need;
            if (take) {
                const int at = ao + min(al, need);
                key[at] = mk[j];
                entry[at] = me[j];
            }
            ao += k > prefix;
            al += k == prefix;
        }
        kept = d.top;
        __syncthreads();
    }
    for (int i = tid; i < d.top; i += 256) out[i] = entry[i];
}

// Rows of a pass: their scores take this many bytes at most (a row's always).
constexpr size_t kSelWorkspace = 256u << 20;
static size_t select_row_bytes(const sfm_paged_desc& d) { return (size_t)d.kv_heads * (d.width + d.D) * sizeof(uint64_t); }
static int select_pass(const sfm_paged_desc& d) {
    const size_t row = select_row_bytes(d);
    const int64_t rows = pieces(d.tokens, d.group, d.requests);
    return (int)std::max<int64_t>(1, std::min<int64_t>({rows, (int64_t)(kSelWorkspace / row), 65535}));
}
size_t paged_select_workspace_bytes(const sfm_paged_desc& d) { return select_pass(d) * select_row_bytes(d); }

template <typename E, int RT>
static auto score_kernel(int ni) {
    return ni == 1 ? paged_score_kernel<E, 1, RT> : ni == 2 ? paged_score_kernel<E, 2, RT> : ni == 3 ? paged_score_kernel<E, 3, RT> : paged_score_kernel<E, 4, RT>;
}

int launch_paged_select(const sfm_paged_desc& d, const void* q, const float* means, const int32_t* table, const int32_t* past,
                        const int32_t* q_start, int first, int last, int32_t* selected, void* workspace, hipStream_t stream) {
    const int64_t rows = pieces(d.tokens, d.group, d.requests);
    if ((int64_t)select_pass(d) * d.kv_heads >= (1 << 24) || rows / select_pass(d) > 4096) {
        set_error("%lld groups of tokens with %d key heads are more than a call takes", (long long)rows, d.kv_heads);
        return SFM_ERR_UNSUPPORTED;
    }
    const size_t lds = (size_t)(d.top + kSelPages) * 12;
    const hipError_t e = hipFuncSetAttribute((const void*)paged_select_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) {
        set_error("hipFuncSetAttribute failed: %s", hipGetErrorString(e));
        return SFM_ERR_HIP;
    }
    // four rows share a mean where most requests have that many groups
    // and the sums are formed once where a row's are of more queries than a workgroup reads at once
    const bool sums = (int64_t)d.group * (d.H / d.kv_heads) > 16;
    const int rt = d.tokens / d.group >= 4 * (int64_t)d.requests ? 4 : 1, ni = (d.D + 63) / 64;
    for (int64_t row0 = 0; row0 < rows; row0 += select_pass(d)) {
        SelectArgs s{d, q, means, table, past, q_start, selected, (uint64_t*)workspace, first, last, (int)row0, (int)std::min<int64_t>(select_pass(d), rows - row0), 0, nullptr};
        if (sums) s.sums = (double*)(s.keys + (size_t)s.rows * d.kv_heads * d.width);
        const int64_t tiles = (s.rows + rt - 1) / rt;
        // 64 pages are a round of a workgroup's loads; as few rounds as keep the chip busy
        const int64_t wanted = std::max<int64_t>(1, 8 * cu_count() / (tiles * d.kv_heads));
        s.chunk = (int)std::max<int64_t>(64, ((d.width + wanted - 1) / wanted + 63) / 64 * 64);
        s.chunk = (int)std::max<int64_t>(s.chunk, (d.width / 65535 + 64) / 64 * 64);
        const dim3 grid((unsigned)tiles, d.kv_heads, (d.width + s.chunk - 1) / s.chunk);
        auto kern = d.dtype == SFM_BF16 ? (rt == 4 ? score_kernel<BF16, 4>(ni) : score_kernel<BF16, 1>(ni))
                    : d.dtype == SFM_F16 ? (rt == 4 ? score_kernel<F16, 4>(ni) : score_kernel<F16, 1>(ni))
                                         : (rt == 4 ? score_kernel<float, 4>(ni) : score_kernel<float, 1>(ni));
        if (sums) {
            auto add = d.dtype == SFM_BF16 ? paged_sums_kernel<BF16> : d.dtype == SFM_F16 ? paged_sums_kernel<F16> : paged_sums_kernel<float>;
            hipLaunchKernelGGL(add, dim3(s.rows, d.kv_heads), dim3(256), 0, stream, s);
        }
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, s);
        hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)(s.rows * d.kv_heads)), dim3(256), lds, stream, s);
    }
    return launched();
}

}  // namespace sfm
