// Attention of the requests' new tokens over their pages of a shared key-value cache.
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

// ------------------------------------------------------------------------------------------------
// shape-generic kernel (fp32 tensors, head sizes other than 64 and 128): a workgroup takes one query row, 256 positions at a time
// ------------------------------------------------------------------------------------------------
template <typename T> struct PElem;
template <> struct PElem<float> {
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return ((const float*)p)[i]; }
    static __device__ __forceinline__ void put(void* p, int64_t i, float x) { ((float*)p)[i] = x; }
};
template <class E> struct PElem16 {
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return E::to_float(((const uint16_t*)p)[i]); }
    static __device__ __forceinline__ void put(void* p, int64_t i, float x) { ((uint16_t*)p)[i] = E::from_float(x); }
};
template <> struct PElem<BF16> : PElem16<BF16> {};
template <> struct PElem<F16> : PElem16<F16> {};

template <typename T>
__global__ __launch_bounds__(256) void paged_generic_kernel(PagedArgs a) {
    __shared__ float qs[256];
    __shared__ float ws[256];
    __shared__ float red[256];
    __shared__ int64_t at[256];                    // a position's row in the pools, -1 where the query does not see it
    const sfm_paged_desc& d = a.d;
    const int tid = threadIdx.x, t = blockIdx.x, h = blockIdx.y, D = d.D, P = d.page_size;
    const int r = find_last(d.requests, t, [&](int i) { return (int64_t)clamp_int(a.q_start[i], 0, (int)d.tokens); });
    if (r >= d.requests && !d.zero_rest) return;
    const Request rq = request_of(a.q_start, a.past, r, d.requests, (int)d.tokens);
    const int i = t - rq.first;
    if (i < 0 || i >= rq.n) return;
    const KeyTiles k = key_tiles(rq, r >= d.requests, i, i, d.causal, d.window, d.sink, a.cap);
    const int kh = h / (d.H / d.kv_heads);
    const int32_t* sel = nullptr;
    int positions = k.end_max;                     // of the request, or of the selected pages one after the other
    bool bad = k.beyond && !d.top;
    if (d.top && r < d.requests) {
        sel = a.selected + ((first_piece(rq.first, 1, d.group, r) + i / d.group) * d.kv_heads + kh) * d.top;
        int n = 0;
        while (n < d.top && sel[n] >= 0) ++n;
        positions = (int)min((int64_t)n * P, (int64_t)0x7fffffff - 512);
    }
    if (tid < D) qs[tid] = PElem<T>::get(a.q, (int64_t)t * d.q_stride[0] + (int64_t)h * d.q_stride[1] + tid);
    const float sc2 = d.sm_scale * kLog2e;
    float mrun = -__FLT_MAX__, lrun = 0.f, acc = 0.f;
    bool seen = false;
    for (int p0 = 0; p0 < positions; p0 += 256) {
        const int v = p0 + tid;
        int64_t row = -1;
        if (v < positions) {
            const int e = sel ? sel[v / P] : v / P;
            const int64_t pos = (int64_t)e * P + v % P;
            if (pos < k.end_max && (pos >= k.lo_min || pos < d.sink)) {
                const int page = e < d.width ? a.table[r * d.table_stride + e] : -1;
                if (page < 0 || page >= d.pages) bad = true;
                else row = page * d.pool_stride[0] + (int64_t)(v % P) * d.pool_stride[1] + (int64_t)kh * d.pool_stride[2];
            } else if (sel && e >= d.width) {
                bad = true;
            }
        }
        at[tid] = row;
        __syncthreads();
        float z = -INFINITY;
        if (row >= 0) {
            float s = 0.f;
            for (int x = 0; x < D; ++x) s += qs[x] * PElem<T>::get(a.kp, row + x);
            z = s * sc2;
        }
        red[tid] = z;
        const int any = __syncthreads_count(row >= 0);
        seen = seen || any;
        for (int s = 128; s > 0; s >>= 1) {
            if (tid < s) red[tid] = fmaxf(red[tid], red[tid + s]);
            __syncthreads();
        }
        const float mnew = fmaxf(mrun, red[0]);
        __syncthreads();
        const float e = row >= 0 ? exp2f(z - mnew) : 0.f;
        ws[tid] = e;
        red[tid] = e;
        __syncthreads();
        for (int s = 128; s > 0; s >>= 1) {
            if (tid < s) red[tid] += red[tid + s];
            __syncthreads();
        }
        const float alpha = exp2f(mrun - mnew);
        lrun = lrun * alpha + red[0];
        mrun = mnew;
        if (tid < D) {
            acc *= alpha;
            const int cnt = min(256, positions - p0);
            for (int x = 0; x < cnt; ++x)
                if (at[x] >= 0) acc += ws[x] * PElem<T>::get(a.vp, at[x] + tid);
        }
        __syncthreads();
    }
    bad = __syncthreads_or(bad);
    const float inv = bad ? NAN : seen ? 1.f / lrun : 0.f;
    if (tid < D) PElem<T>::put(a.out, (int64_t)t * d.o_stride[0] + (int64_t)h * d.o_stride[1] + tid, acc * inv);
    if (a.lse != nullptr && tid == 0) a.lse[(int64_t)h * d.tokens + t] = bad ? NAN : seen ? (mrun + log2f(lrun)) * kLn2 : -INFINITY;
}

size_t paged_workspace_bytes(const sfm_paged_desc&) { return 0; }

int launch_paged_attention(const sfm_paged_desc& d, const void* q, const void* kp, const void* vp, const int32_t* table,
                           const int32_t* past, const int32_t* q_start, const int32_t* selected, void* out, float* lse, void*,
                           size_t, hipStream_t stream) {
    PagedArgs a{d, fast_div(d.page_size / 8), d.width * d.page_size, q, kp, vp, table, past, q_start, selected, out, lse};
    auto kern = d.dtype == SFM_BF16 ? paged_generic_kernel<BF16> : d.dtype == SFM_F16 ? paged_generic_kernel<F16> : paged_generic_kernel<float>;
    if (d.tokens >= (1 << 24) || d.H > 65535) {
        set_error("tokens=%lld, H=%d are more than a launch takes", (long long)d.tokens, d.H);
        return SFM_ERR_UNSUPPORTED;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)d.tokens, d.H), dim3(256), 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err == hipSuccess) return SFM_OK;
    set_error("hip launch failed: %s", hipGetErrorString(err));
    return SFM_ERR_HIP;
}

}  // namespace sfm
