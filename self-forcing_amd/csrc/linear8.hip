// y = x w^T + bias with both operands in 8-bit blocks of 128 (rows8.hpp), the linear layers of the causal Wan block
// (wan/modules/model.py:592-650) at the matrix rate of e4m3.  No counterpart of the 8-bit form in the reference.
//
//   y[m, n] = sum_k x8[m, k] w8[n, k] 2^(sx[m, k / 128] + sw[n / 128, k / 128]) + bias[n]
//
// The scaled matrix instructions take a power of two per 32 values of either operand and apply it to the products in
// fp32: a block of 128 is four of those with the same exponent.  Sums are fp32 throughout; bias, GELU and the gated
// residual follow on the fp32 sum, and the result is rounded once.
//
// The e4m3 matrix instructions align the products of 8 neighbouring k to the largest of them and drop what lies below 2^-13 of it
// before the fp32 sum (probed on gfx950; scaled and plain forms alike).  On random rows that is 1.7e-5 of the result, against
// 2.6e-2 for the values' own rounding; the 16-bit instructions, at half the rate, would not do so.
//
// Weight rows are the A operand and activation rows the B operand, so that a lane ends up with neighbouring channels of
// one row.

#include "rows8.hpp"

namespace sfm {
namespace {

struct L8Args {
    const uint8_t* x;        // [M][kp]
    const uint8_t* xscale;   // words by (block column, row group, row % 32)
    const uint8_t* w;        // [N][kp]
    const uint8_t* wscale;   // [ceil(N / 128)][pitch]
    const uint16_t* bias;    // [N] or null
    const uint16_t* res;     // [M, N] rows res_stride apart, may alias out
    const uint16_t* gate;    // [frames, N] rows gate_stride apart, or null
    uint16_t* out;           // [M, N] rows out_stride apart
    int64_t M, groups, kp;
    int N, nkb, pitch;
    int64_t out_stride, res_stride, gate_stride;
    int rows_per_frame;
    int tn;                  // tiles along N
    bool vec;                // rows of out, res, gate and bias allow 8-byte accesses
};

// the tail of four neighbouring channels c.. of a row: bias, epilogue, one rounding, store
template <class E, int EPI>
__device__ __forceinline__ void l8_finish4(const L8Args& p, int64_t row, int c, const float* acc) {
    if (row >= p.M || c >= p.N) return;
    const bool full = p.vec && c + 4 <= p.N;
    float v[4], r[4] = {0.f, 0.f, 0.f, 0.f}, g[4] = {1.f, 1.f, 1.f, 1.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    auto get4 = [&](const uint16_t* s, float* d) {
        if (full) {
            const u32x2 w = *(const u32x2*)s;
            d[0] = E::to_float((uint16_t)(w.x & 0xffffu)); d[1] = E::to_float((uint16_t)(w.x >> 16));
            d[2] = E::to_float((uint16_t)(w.y & 0xffffu)); d[3] = E::to_float((uint16_t)(w.y >> 16));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < p.N) d[i] = E::to_float(s[i]);
        }
    };
    if (p.bias != nullptr) get4(p.bias + c, b);
    if (EPI == SFM_EPI_GATE_RESIDUAL) {
        get4(p.res + row * p.res_stride + c, r);
        if (p.gate != nullptr) get4(p.gate + (row / p.rows_per_frame) * p.gate_stride + c, g);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = acc[i] + b[i];
        if (EPI == SFM_EPI_GELU_TANH) v[i] *= gelu_gate<false>(v[i]);
        if (EPI == SFM_EPI_GATE_RESIDUAL) v[i] = r[i] + v[i] * g[i];
    }
    uint16_t* o = p.out + row * p.out_stride + c;
    if (full) {
        u32x2 w = {pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3])};
        *(u32x2*)o = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < p.N) o[i] = E::from_float(v[i]);
    }
}

__device__ __forceinline__ i32x8 l8_load32(const uint8_t* p) {
    const u32x4 a = *(const u32x4*)p, b = *(const u32x4*)(p + 16);
    i32x8 r = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    return r;
}

// Any size: a workgroup of W waves owns 16 MT rows x 16 NT channels, its waves share the block columns (wave w takes w,
// w + W, ...) and their sums meet in LDS in a fixed order.  Operands come from memory straight into registers, 32 bytes a
// lane of one row: 4 lanes take a row's block of 128 bytes, a whole line.
template <class E, int EPI, int MT, int NT, int W>
__global__ __launch_bounds__(64 * W) void l8_direct_kernel(L8Args p) {
    __shared__ f32x4 part[W][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int64_t m0 = (int64_t)(blockIdx.x / p.tn) * (16 * MT);
    const int n0 = (int)(blockIdx.x % p.tn) * (16 * NT);
    const uint8_t *xp[MT], *wp[NT];
    int64_t xsc[MT];
    int wsc[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t r = min(m0 + 16 * i + l16, p.M - 1);
        xp[i] = p.x + r * p.kp + q * 32;
        xsc[i] = scale_at8(r, 0, p.groups);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = min(n0 + 16 * j + l16, p.N - 1);
        wp[j] = p.w + n * p.kp + q * 32;
        wsc[j] = (n >> 7) * p.pitch;
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = wave; kb < p.nkb; kb += W) {
        i32x8 xf[MT], wf[NT];
        int xe[MT], we[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            wf[j] = l8_load32(wp[j] + (int64_t)kb * kBlock8);
            we[j] = p.wscale[wsc[j] + kb];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            xf[i] = l8_load32(xp[i] + (int64_t)kb * kBlock8);
            xe[i] = p.xscale[xsc[i] + (int64_t)kb * p.groups * kBlock8];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], xf[i], acc[i][j], 0, 0, 0, we[j], 0, xe[i]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    // lane (l16, q) of block (i, j) holds row 16 i + l16, channels 16 j + 4 q ..
    for (int t = wave; t < MT * NT; t += W) {
        f32x4 s = part[0][t][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) s += part[w][t][lane];
        const float v[4] = {s.x, s.y, s.z, s.w};
        l8_finish4<E, EPI>(p, m0 + 16 * (t / NT) + l16, n0 + 16 * (t % NT) + 4 * q, v);
    }
}

template <class E, int EPI, int MT, int NT, int W>
int launch_direct(const L8Args& a0, hipStream_t st) {
    L8Args a = a0;
    a.tn = (a.N + 16 * NT - 1) / (16 * NT);
    const dim3 grid((unsigned)(a.tn * ((a.M + 16 * MT - 1) / (16 * MT))));
    hipLaunchKernelGGL((l8_direct_kernel<E, EPI, MT, NT, W>), grid, dim3(64 * W), 0, st, a);
    return launched8("sfm_linear8");
}

template <class E, int EPI>
int launch_epi(const L8Args& a, hipStream_t st) {
    if (a.M <= 16) return launch_direct<E, EPI, 1, 1, 8>(a, st);
    return launch_direct<E, EPI, 4, 4, 4>(a, st);
}

template <class E>
int launch_dtype(const L8Args& a, int epilogue, hipStream_t st) {
    if (epilogue == SFM_EPI_GELU_TANH) return launch_epi<E, SFM_EPI_GELU_TANH>(a, st);
    if (epilogue == SFM_EPI_GATE_RESIDUAL) return launch_epi<E, SFM_EPI_GATE_RESIDUAL>(a, st);
    return launch_epi<E, SFM_EPI_NONE>(a, st);
}

}  // namespace

int launch_linear8(const sfm_linear8_desc& d, const void* x8, const void* xscale, const void* w8, const void* wscale, const void* bias,
                   const void* res, const void* gate, void* out, hipStream_t stream) {
    L8Args a;
    a.x = (const uint8_t*)x8;
    a.xscale = (const uint8_t*)xscale;
    a.w = (const uint8_t*)w8;
    a.wscale = (const uint8_t*)wscale;
    a.bias = (const uint16_t*)bias;
    a.res = (const uint16_t*)res;
    a.gate = (const uint16_t*)gate;
    a.out = (uint16_t*)out;
    a.M = d.M;
    a.groups = (d.M + kBlock8 - 1) / kBlock8;
    a.kp = pad8(d.K);
    a.N = d.N;
    a.nkb = blocks8(d.K);
    a.pitch = pitch8(d.K);
    a.out_stride = d.out_stride;
    a.res_stride = d.res_stride;
    a.gate_stride = d.gate_stride;
    a.rows_per_frame = d.rows_per_frame > 0 ? d.rows_per_frame : 1;
    auto ok = [](const void* q, int64_t stride) { return q == nullptr || (((uintptr_t)q & 15) == 0 && stride % 8 == 0); };
    a.vec = ok(out, d.out_stride) && ok(res, d.res_stride) && ok(gate, d.gate_stride) && ok(bias, 0);
    return d.dtype == SFM_BF16 ? launch_dtype<BF16>(a, d.epilogue, stream) : launch_dtype<F16>(a, d.epilogue, stream);
}

}  // namespace sfm
