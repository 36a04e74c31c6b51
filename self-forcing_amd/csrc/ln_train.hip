// LayerNorm's training side: the forward that keeps its normalised rows in 8-bit blocks, and the backward of both forms of
// the norm (affine weight / bias: norm3, wan/modules/causal_model.py:1194; per-frame scale / shift: norm1, norm2,
// causal_model.py:1179-1183, 1198-1201).  The reference leaves both to autograd.
//
//   xh = (x - mean) r, r = 1 / sqrt(var + eps);  g = dy w   (w the weight, or 1 + scale of the row's frame)
//   dx = r (g - mean(g) - xh mean(g xh))
//   dw = sum dy xh, db = sum dy   over all rows (affine) or the rows of a frame (scale, shift)
//
// A row is read once into registers: its statistics are formed again from the same values (the row is there anyway; kept
// statistics would be another stream to read), up to 1536 channels in the forward's order, above that over four waves where the
// forward has one, so that their last bits may differ; then the sums of g and g (x - mean) in one exchange.  The column sums
// dw, db stay in registers over all rows of a wave, meet in LDS, and leave as one fp32 partial per workgroup, which a second
// kernel adds in a fixed order: no atomics, the same result every time.
//
// Bound by memory: 21 frames of 1560 x 1536, modulated, 68-70 us and 5 for the partials (302 MB: 4.3 TB/s).  A chunk of 4680 x 1536 from
// 8-bit blocks: 16 us and 4 (36 MB, 8 us at that rate): a wave has two rows, waits for the loads of each and then for its sums, and
// the 768 partials are another 9 MB.

#include "rows8.hpp"

namespace sfm {
namespace {

struct LnBwdArgs {
    const void* x;           // [rows, C], or null with data / scale8 / rstd
    const uint8_t* data;     // normalised rows in 8-bit blocks
    const uint8_t* scale8;
    const float* rstd;       // [rows]
    const void* dy;
    void* dx;                // may be null
    const void* weight;      // [C], or scale rows (MOD) mod_stride apart
    float* part;             // [groups of rows][splits][2][C], unless a group has one workgroup, which stores dw and db itself
    void *dw, *db;
    int64_t xs, dys, dxs, ms, groups8;
    int C, rpg, splits;      // rows per group (of one weight gradient), workgroups per group
    float eps;
};

// WPR waves share a row (1 or 4), NT chunks of 8 channels a lane
template <typename T, int NT, int WPR, bool MOD, bool KEPT>
__global__ __launch_bounds__(256) void ln_bwd_kernel(LnBwdArgs p) {
    using V = V8<T>;
    constexpr int RW = 4 / WPR;              // rows a workgroup has in hand
    __shared__ float xch[2][4][4];
    __shared__ float col[4][64 * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = WPR == 1 ? 0 : wave;     // which part of the row
    const int nch = p.C / 8;
    const int64_t grp = blockIdx.x / p.splits;
    const int split = blockIdx.x % p.splits;
    const int64_t g0 = grp * p.rpg;
    const RowRange mine = rows_of_part(p.rpg, p.splits, split);
    const int64_t r_end = g0 + mine.last;
    int par = 0;
    auto row_sum3 = [&](float& a, float& b, float& c) {
        a = wave_sum(a);
        b = wave_sum(b);
        c = wave_sum(c);
        if (WPR > 1) {
            if (lane == 0) {
                xch[par][wave][0] = a;
                xch[par][wave][1] = b;
                xch[par][wave][2] = c;
            }
            __syncthreads();
            a = xch[par][0][0] + xch[par][1][0] + xch[par][2][0] + xch[par][3][0];
            b = xch[par][0][1] + xch[par][1][1] + xch[par][2][1] + xch[par][3][1];
            c = xch[par][0][2] + xch[par][1][2] + xch[par][2][2] + xch[par][3][2];
            par ^= 1;                        // the other slot is free: everyone has passed the barrier after reading it
        }
    };
    float dw[NT][8], db[NT][8], wv[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int ch = lane + (t * WPR + sub) * 64;
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[t][i] = db[t][i] = wv[t][i] = 0.f;
        if (ch < nch) {
            V::load(p.weight, (MOD ? grp * p.ms : 0) + ch * 8, wv[t]);
            if (MOD) {
#pragma unroll
                for (int i = 0; i < 8; ++i) wv[t][i] += 1.f;
            }
        }
    }
    for (int64_t base = g0 + mine.first; base < r_end; base += RW) {
        const int64_t row = base + (WPR == 1 ? wave : 0);
        const bool live = row < r_end;       // with WPR > 1 the same for the whole workgroup
        if (WPR == 1 && !live) break;
        float x[NT][8], g[NT][8];
        float s0 = 0.f, s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int ch = lane + (t * WPR + sub) * 64;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[t][i] = g[t][i] = 0.f;
            if (ch < nch) {
                if (KEPT) {
                    const u32x2 q = *(const u32x2*)(p.data + row * pad8(p.C) + ch * 8);
                    const float s = two_to((int)p.scale8[scale_at8(row, ch >> 4, p.groups8)] - 127);
                    unpack_e4m3(q.x, x[t]);
                    unpack_e4m3(q.y, x[t] + 4);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[t][i] *= s;
                } else {
                    V::load(p.x, row * p.xs + ch * 8, x[t]);
                }
                V::load(p.dy, row * p.dys + ch * 8, g[t]);
#pragma unroll
                for (int i = 0; i < 8; ++i) s0 += x[t][i];
            }
        }
        float mean = 0.f;
        if (!KEPT) {
            row_sum3(s0, s1, s2);
            mean = s0 / p.C;
        }
        s0 = s1 = s2 = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int ch = lane + (t * WPR + sub) * 64;
            if (ch < nch) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = x[t][i] - mean, gw = g[t][i] * wv[t][i];
                    x[t][i] = d;
                    s0 += d * d;
                    s1 += gw;
                    s2 += gw * d;
                }
            }
        }
        row_sum3(s0, s1, s2);
        // KEPT: x is xh already; otherwise xh = r d
        const float r = KEPT ? p.rstd[row] : 1.0f / sqrtf(s0 / p.C + p.eps);
        const float xr = KEPT ? 1.f : r;
        const float mg = s1 / p.C, mgx = xr * s2 / p.C;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int ch = lane + (t * WPR + sub) * 64;
            if (ch < nch) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float xh = x[t][i] * xr;
                    dw[t][i] += g[t][i] * xh;
                    db[t][i] += g[t][i];
                    o[i] = r * (g[t][i] * wv[t][i] - mg - xh * mgx);
                }
                if (p.dx != nullptr) V::store(p.dx, row * p.dxs + ch * 8, o);
            }
        }
    }
    // column sums of the workgroup
    float* part = p.part + (grp * p.splits + split) * 2 * (int64_t)p.C;
    const bool alone = p.splits == 1;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int ch = lane + (t * WPR + sub) * 64;
            float* v = which == 0 ? dw[t] : db[t];
            void* out = which == 0 ? p.dw : p.db;
            if (WPR > 1) {
                if (ch < nch && alone) V::store(out, grp * p.C + ch * 8, v);
                else if (ch < nch) V8<float>::store(part, which * (int64_t)p.C + ch * 8, v);
            } else {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) col[wave][i * 64 + lane] = v[i];
                __syncthreads();
                for (int e = threadIdx.x; e < 512; e += 256) {
                    const int l = e >> 3, i = e & 7;
                    const float s = col[0][i * 64 + l] + col[1][i * 64 + l] + col[2][i * 64 + l] + col[3][i * 64 + l];
                    const int c = (t * 64 + l) * 8 + i;
                    if (c < p.C && alone) Elem<T>::put(out, grp * p.C + c, s);
                    else if (c < p.C) part[which * (int64_t)p.C + c] = s;
                }
            }
        }
}

// out[g][c] = sum over s of part[g][s][c], c < n; the first `n1` columns of a group go to out1, the rest to out2.  32 columns x SL
// slices of the parts per workgroup, the slices in a fixed order; SL = 32 where there are parts enough: a thread's loads, eight at a
// time, are then few one after the other (512 parts of 2 x 1536 columns: 5 us, with 8 slices 20)
template <typename T, int SL>
__global__ __launch_bounds__(32 * SL) void sum_parts_kernel(const float* part, int64_t parts, int64_t n, int64_t n1, int64_t groups, void* out1,
                                                            void* out2) {
    __shared__ float sl[SL][32];
    const int l = threadIdx.x & 31, sn = threadIdx.x >> 5;
    const int64_t id = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int64_t cols = (n + 31) / 32, g = id / cols, c = (id % cols) * 32 + l;
    if (g >= groups) return;
    float s = 0.f;
    if (c < n) {
        const float* p = part + (g * parts) * n + c;
        int64_t i = sn;
        for (; i + 7 * SL < parts; i += 8 * SL) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[(i + e * SL) * n];
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[e];
        }
        for (; i < parts; i += SL) s += p[i * n];
    }
    sl[sn][l] = s;
    __syncthreads();
    if (sn == 0 && c < n) {
#pragma unroll
        for (int i = 1; i < SL; ++i) s += sl[i][l];
        if (c < n1) Elem<T>::put(out1, g * n1 + c, s);
        else Elem<T>::put(out2, g * (n - n1) + c - n1, s);
    }
}

// y = LayerNorm(x) as ln_modulate_kernel forms it, with xh in 8-bit blocks and r kept besides.  4680 x 1536: 11 us (36 MB: 3.3 TB/s)
template <typename T, int NT>
__global__ __launch_bounds__(256) void ln_keep8_kernel(const void* x, int64_t xs, void* y, int64_t ys, int C, float eps, const void* scale,
                                                       const void* shift, int64_t ms, int rows_per_frame, const void* weight,
                                                       const void* bias, int64_t rows, uint8_t* data, uint8_t* scale8, float* rstd_out) {
    using V = V8<T>;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63, nch = C / 8;
    float v[NT][8];
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int ch = lane + t * 64;
        if (ch < nch) {
            V::load(x, row * xs + ch * 8, v[t]);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += v[t][i];
        }
    }
    const float mean = wave_sum(sum) / C;
    float sq = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int ch = lane + t * 64;
        if (ch < nch) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float d = v[t][i] - mean;
                sq += d * d;
            }
        }
    }
    const float rstd = 1.0f / sqrtf(wave_sum(sq) / C + eps);
    const int64_t moff = (row / rows_per_frame) * ms, kp = pad8(C), groups = (rows + kBlock8 - 1) / kBlock8;
    if (lane == 0) rstd_out[row] = rstd;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int ch = lane + t * 64;
        float n[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = ch < nch ? (v[t][i] - mean) * rstd : 0.f;
        u32x2 q;
        const int s = quantize_block8(n, &q);
        if (ch < kp / 8) {
            *(u32x2*)(data + row * kp + ch * 8) = q;
            if ((lane & 15) == 0) scale8[scale_at8(row, ch >> 4, groups)] = (uint8_t)(s + 127);
        }
        if (ch < nch) {
            float o[8];
            if (weight != nullptr) {
                float w[8], b[8];
                V::load(weight, ch * 8, w);
                V::load(bias, ch * 8, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = (v[t][i] - mean) * rstd * w[i] + b[i];
            } else {
                float sc[8], sh[8];
                V::load(scale, moff + ch * 8, sc);
                V::load(shift, moff + ch * 8, sh);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float m = V::rnd((v[t][i] - mean) * rstd);
                    float g = V::rnd(1.0f + sc[i]);
                    o[i] = V::rnd(m * g) + sh[i];
                }
            }
            V::store(y, row * ys + ch * 8, o);
        }
    }
}

// Workgroups per group of rows: three on every compute unit, or two, where that comes out nearly whole (a few more than two make
// some units run three while the others wait: 21 frames of 1560 x 1536, 525 workgroups 76 us, 756 68), and four rows each at least.
int ln_bwd_splits(int64_t groups, int64_t rpg) {
    const int64_t cus = cu_count(), most = (rpg + 3) / 4;
    for (int64_t k = 3; k >= 2; --k) {
        const int64_t s = k * cus / groups;
        if (s >= 1 && s <= most && groups * s * 10 >= 9 * k * cus) return (int)s;
    }
    const int64_t s = 2 * cus / groups;
    return (int)(s < 1 ? 1 : s < most ? s : most);
}

template <typename T, bool MOD, bool KEPT>
int ln_bwd_t(const LnBwdArgs& a, int64_t groups, hipStream_t st) {
    const dim3 grid((unsigned)(groups * a.splits));
    if (a.C <= 1536) hipLaunchKernelGGL((ln_bwd_kernel<T, 3, 1, MOD, KEPT>), grid, dim3(256), 0, st, a);
    else if (a.C <= 6144) hipLaunchKernelGGL((ln_bwd_kernel<T, 3, 4, MOD, KEPT>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((ln_bwd_kernel<T, 4, 4, MOD, KEPT>), grid, dim3(256), 0, st, a);
    return launched8("sfm_ln_bwd");
}
template <typename T>
int ln_bwd_m(const LnBwdArgs& a, bool mod, int64_t groups, hipStream_t st) {
    if (a.data != nullptr) return mod ? ln_bwd_t<T, true, true>(a, groups, st) : ln_bwd_t<T, false, true>(a, groups, st);
    return mod ? ln_bwd_t<T, true, false>(a, groups, st) : ln_bwd_t<T, false, false>(a, groups, st);
}

template <typename T>
int sum_parts_t(int64_t parts, int64_t n, int64_t n1, int64_t groups, const float* part, void* out1, void* out2, hipStream_t st) {
    const dim3 grid = wide_grid((n + 31) / 32 * groups);
    if (parts >= 64) hipLaunchKernelGGL((sum_parts_kernel<T, 32>), grid, dim3(1024), 0, st, part, parts, n, n1, groups, out1, out2);
    else hipLaunchKernelGGL((sum_parts_kernel<T, 8>), grid, dim3(256), 0, st, part, parts, n, n1, groups, out1, out2);
    return launched8("sum of partials");
}

}  // namespace

int launch_sum_parts(int dtype, int64_t parts, int64_t n, int64_t groups, const float* part, void* out1, void* out2, hipStream_t st) {
    const int64_t n1 = out2 != nullptr ? n / 2 : n;
    return dtype == SFM_BF16 ? sum_parts_t<BF16>(parts, n, n1, groups, part, out1, out2, st)
         : dtype == SFM_F16  ? sum_parts_t<F16>(parts, n, n1, groups, part, out1, out2, st)
                             : sum_parts_t<float>(parts, n, n1, groups, part, out1, out2, st);
}

size_t ln_bwd_workspace_bytes(int64_t rows, int C, int64_t rows_per_group) {
    const int64_t groups = rows / rows_per_group;
    const int splits = ln_bwd_splits(groups, rows_per_group);
    return splits > 1 ? (size_t)groups * splits * 2 * C * sizeof(float) : 0;
}

int launch_ln_bwd(int dtype, int64_t rows, int C, float eps, const void* x, int64_t xs, const void* data, const void* scale8,
                  const float* rstd, const void* dy, int64_t dys, const void* weight, int64_t ms, int64_t rows_per_group, bool mod, void* dx,
                  int64_t dxs, void* dw, void* db, void* workspace, hipStream_t st) {
    const int64_t groups = rows / rows_per_group;
    LnBwdArgs a;
    a.x = x;
    a.data = (const uint8_t*)data;
    a.scale8 = (const uint8_t*)scale8;
    a.rstd = rstd;
    a.dy = dy;
    a.dx = dx;
    a.weight = weight;
    a.part = (float*)workspace;
    a.dw = dw;
    a.db = db;
    a.xs = xs;
    a.dys = dys;
    a.dxs = dxs;
    a.ms = ms;
    a.groups8 = (rows + kBlock8 - 1) / kBlock8;
    a.C = C;
    a.rpg = (int)rows_per_group;
    a.splits = ln_bwd_splits(groups, rows_per_group);
    a.eps = eps;
    int rc = dtype == SFM_BF16 ? ln_bwd_m<BF16>(a, mod, groups, st) : dtype == SFM_F16 ? ln_bwd_m<F16>(a, mod, groups, st) : ln_bwd_m<float>(a, mod, groups, st);
    if (rc || a.splits == 1) return rc;
    return launch_sum_parts(dtype, a.splits, 2 * (int64_t)C, groups, a.part, dw, db, st);
}

#define SFM_LN8(T, NT)                                                                                                              \
    hipLaunchKernelGGL((ln_keep8_kernel<T, NT>), grid, dim3(256), 0, st, x, xs, y, ys, C, eps, scale, shift, ms, rows_per_frame, weight, \
                       bias, rows, (uint8_t*)data, (uint8_t*)scale8, rstd)
#define SFM_LN8_T(T) \
    do { if (nt <= 3) SFM_LN8(T, 3); else if (nt <= 10) SFM_LN8(T, 10); else SFM_LN8(T, 16); } while (0)

int launch_ln_keep8(int dtype, int64_t rows, int C, float eps, const void* x, int64_t xs, void* y, int64_t ys, const void* scale,
                    const void* shift, int64_t ms, int rows_per_frame, const void* weight, const void* bias, void* data, void* scale8,
                    float* rstd, hipStream_t st) {
    const dim3 grid((unsigned)((rows + 3) / 4));
    const int nt = (int)((pad8(C) / 8 + 63) / 64);
    if (dtype == SFM_BF16) SFM_LN8_T(BF16);
    else if (dtype == SFM_F16) SFM_LN8_T(F16);
    else SFM_LN8_T(float);
    return launched8("sfm_ln_keep8");
}

}  // namespace sfm
