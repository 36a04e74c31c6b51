// y = x w^T + bias with both operands in 8-bit blocks of 128 (rows8.hpp), the linear layers of the causal Wan block
// (wan/modules/model.py:592-650) at the matrix rate of e4m3.  No counterpart of the 8-bit form in the reference.
//
//   y[m, n] = sum_k x8[m, k] w8[n, k] 2^(sx[m, k / 128] + sw[n / 128, k / 128]) + bias[n]
//
// The scaled matrix instructions take a power of two per 32 values of either operand and apply it to the products in
// fp32: a block of 128 is four of those with the same exponent.  Sums are kept in fp32; bias, GELU and the gated
// residual follow on the fp32 sum, and the result is rounded once.
//
// The e4m3 matrix instructions align the products of 8 neighbouring k to the largest of them and drop what lies below 2^-13 of it
// before the fp32 sum (probed on gfx950; scaled and plain forms alike).  On random rows that is 1.7e-5 of the result, against
// 2.6e-2 for the values' own rounding; the 16-bit instructions, at half the rate, would not do so.
//
// Weight rows are the A operand and activation rows the B operand, so that a lane ends up with neighbouring channels of
// one row.

#include <utility>

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
    int tm, tn;              // tiles along M and N
    int half;                // 1: the last strip of tiles has half the rows
};

template <class E>
__device__ __forceinline__ void l8_unpack4(u32x2 w, float* d) {
    d[0] = E::to_float((uint16_t)(w.x & 0xffffu)); d[1] = E::to_float((uint16_t)(w.x >> 16));
    d[2] = E::to_float((uint16_t)(w.y & 0xffffu)); d[3] = E::to_float((uint16_t)(w.y >> 16));
}
template <class E, int EPI>
__device__ __forceinline__ float l8_tail(float sum, float bias, float res, float gate) {
    const float v = sum + bias;
    return EPI == SFM_EPI_GELU_TANH ? v * gelu_gate<false>(v) : EPI == SFM_EPI_GATE_RESIDUAL ? res + v * gate : v;
}

// four neighbouring channels c.. of a row of 16-bit values
template <class E>
__device__ __forceinline__ void l8_get4(const L8Args& p, const uint16_t* s, int c, float* d) {
    if (c + 4 <= p.N) {
        l8_unpack4<E>(*(const u32x2_any*)s, d);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < p.N) d[i] = E::to_float(s[i]);
    }
}
// the bias of four channels, zeros without one or past the last
template <class E>
__device__ __forceinline__ f32x4 l8_bias4(const L8Args& p, int c) {
    float b[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias != nullptr) l8_get4<E>(p, p.bias + c, c, b);
    return f32x4{b[0], b[1], b[2], b[3]};
}
// four neighbouring channels of a row: bias and epilogue on the fp32 sums, rounded once and stored
template <class E, int EPI>
__device__ __forceinline__ void l8_finish4(const L8Args& p, int64_t row, int c, const float* acc, f32x4 b) {
    if (row >= p.M || c >= p.N) return;
    const bool full = c + 4 <= p.N;
    float v[4], r[4] = {0.f, 0.f, 0.f, 0.f}, g[4] = {1.f, 1.f, 1.f, 1.f};
    if (EPI == SFM_EPI_GATE_RESIDUAL) {
        l8_get4<E>(p, p.res + row * p.res_stride + c, c, r);
        if (p.gate != nullptr) l8_get4<E>(p, p.gate + (row / p.rows_per_frame) * p.gate_stride + c, c, g);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = l8_tail<E, EPI>(acc[i], b[i], r[i], g[i]);
    uint16_t* o = p.out + row * p.out_stride + c;
    if (full) {
        u32x2 w = {pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3])};
        *(u32x2_any*)o = w;
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
// w + W, ...) and their sums meet in LDS in a fixed order.  Operands come from memory straight into registers, 32 bytes a lane of one
// row: 4 lanes take a row's block of 128 bytes, a whole line.  Many waves hide the loads: with the next block column's operands held
// besides, 128 x 1536 -> 8960 takes 26 us against 18.
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
        l8_finish4<E, EPI>(p, m0 + 16 * (t / NT) + l16, n0 + 16 * (t % NT) + 4 * q, v, l8_bias4<E>(p, n0 + 16 * (t % NT) + 4 * q));
    }
}

// Up to 16 rows, quantised where they are used: lane (l16, q) forms the operand of its row's 32 values from the 16-bit rows, the four
// lanes of a row agree on the block's scale.  The weights pass once, 16 channels a workgroup, the block columns over its W waves; one
// launch, no rows in memory.  One token, 1536 -> 8960: 9.4 us, of which the weight's 13.8 MB are 2.8 at the rate of a large copy: the
// rest is the launch (3), one trip to memory for a wave's one or two blocks, and the sums' meeting.
template <class E, int EPI, int W>
__global__ __launch_bounds__(64 * W) void l8_few_kernel(L8Args p, const uint16_t* x, int64_t xstride, int K) {
    __shared__ f32x4 part[W][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16, n = min(n0 + l16, p.N - 1);
    const uint8_t* wp = p.w + (int64_t)n * p.kp + q * 32;
    const uint8_t* ws = p.wscale + (int64_t)(n >> 7) * p.pitch;
    const uint16_t* xr = x + min((int64_t)l16, p.M - 1) * xstride;       // lanes past the last row form products that nobody stores
    const f32x4 bias = l8_bias4<E>(p, n0 + 4 * q);                      // on its way from the start
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    struct Ops {
        i32x8 w;
        int we;
        u32x4 v[4];
    };
    const int whole = K / kBlock8;
    auto fetch = [&](Ops& o, int kb) {
        o.w = l8_load32(wp + (int64_t)kb * kBlock8);
        o.we = ws[kb];
        const int c0 = kb * kBlock8 + q * 32;
        if (kb < whole) {
#pragma unroll
            for (int c = 0; c < 4; ++c) o.v[c] = *(const u32x4_any*)(xr + c0 + 8 * c);
        } else {                                                        // the row ends in this block: zeros behind it
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                o.v[c] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c0 + 8 * c + e < K) o.v[c][e >> 1] |= (uint32_t)xr[c0 + 8 * c + e] << (16 * (e & 1));
            }
        }
    };
    auto multiply = [&](const Ops& o) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[2 * i] = E::to_float((uint16_t)(o.v[i >> 2][i & 3] & 0xffffu));
            v[2 * i + 1] = E::to_float((uint16_t)(o.v[i >> 2][i & 3] >> 16));
        }
        auto block_max = [](float m) {
            m = fmaxf(m, __shfl_xor(m, 16));
            return fmaxf(m, __shfl_xor(m, 32));
        };
        float a = block_max(mag_max<32>(v));
        if (__builtin_expect(a >= kTop8, 0)) a = block_max(mag_max_finite<32>(v));
        const int s = block_exp8(a);
        const float inv = two_to(-s);
        i32x8 xf;
#pragma unroll
        for (int c = 0; c < 8; ++c) xf[c] = (int)pack_e4m3(v[4 * c] * inv, v[4 * c + 1] * inv, v[4 * c + 2] * inv, v[4 * c + 3] * inv);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(o.w, xf, acc, 0, 0, 0, o.we, 0, s + 127);
    };
    Ops a, b;
    const int last = p.nkb - 1;
    if (wave <= last) {
        fetch(a, wave);
        for (int kb = wave; kb <= last; kb += 2 * W) {
            fetch(b, min(kb + W, last));
            __builtin_amdgcn_sched_barrier(0);
            multiply(a);
            if (kb + W > last) break;
            fetch(a, min(kb + 2 * W, last));
            __builtin_amdgcn_sched_barrier(0);
            multiply(b);
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
        f32x4 s = part[0][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) s += part[w][lane];
        const float v[4] = {s.x, s.y, s.z, s.w};
        l8_finish4<E, EPI>(p, l16, n0 + 4 * q, v, bias);
    }
}

// 8 or 16 waves a workgroup for up to 16 rows: 16 where the channels make few workgroups and the rows are long enough to share out
// (8960 -> 1536: 96 workgroups of 70 blocks)
bool few_wide(const L8Args& a) { return (a.N + 15) / 16 < 2 * cu_count() && a.nkb >= 16; }
template <class E, int EPI>
int launch_few(const L8Args& a, const void* x, int64_t xstride, int K, hipStream_t st) {
    const unsigned wgs = (unsigned)((a.N + 15) / 16);
    if (few_wide(a))
        hipLaunchKernelGGL((l8_few_kernel<E, EPI, 16>), dim3(wgs), dim3(1024), 0, st, a, (const uint16_t*)x, xstride, K);
    else
        hipLaunchKernelGGL((l8_few_kernel<E, EPI, 8>), dim3(wgs), dim3(512), 0, st, a, (const uint16_t*)x, xstride, K);
    return launched8("sfm_linear8_fwd");
}

template <class E, int EPI, int MT, int NT, int W>
int launch_direct(const L8Args& a0, hipStream_t st) {
    L8Args a = a0;
    a.tn = (a.N + 16 * NT - 1) / (16 * NT);
    const dim3 grid((unsigned)(a.tn * ((a.M + 16 * MT - 1) / (16 * MT))));
    hipLaunchKernelGGL((l8_direct_kernel<E, EPI, MT, NT, W>), grid, dim3(64 * W), 0, st, a);
    return launched8("sfm_linear8");
}

// ---------------------------------------------------------------------------------------------------------------------
// Many rows.  A workgroup of four waves owns 256 weight rows x 64 TB activation rows (TB = 4 or 2), a wave 128 x 32 TB of it: 4 x TB
// matrix instructions 32x32x64 a k step, 64 TB accumulator registers, one wave per SIMD.  A stage is 128 bytes of every row, one
// block and one cache line; both operands go from memory straight into LDS through a ring of nine 16 KB slots of 128 rows: the
// weight rows of a stage are two slots, its activation rows two (TB = 4) or one, so that more than a stage is in flight while one is
// multiplied.  Rows sit two to a 256-byte LDS line with their 16-byte pieces XOR-ed by the line index: the 16 lanes of an
// operand read hit 64 different banks.  A lane's 32 bytes of a step are pieces 4 s + hf and 4 s + 2 + hf of its row for both operands.
//
// Scales: the 64 words of a stage's 256 rows follow the rows into LDS, a lane's word holds those of its row in the four row blocks
// (rows8.hpp), and the matrix instruction picks the byte; the weight's is one for the wave, through the scalar cache.
//
// A stage takes 1.35 us, its matrix instructions 0.98 at the 2.1 GHz of a long run, and a tile 8-10 us besides (launch, first stages,
// its 128 KB on their way out): 8192^3 374-393 us, 2.8-2.9 PFLOP/s; 4680 x 5120 -> 13824 273-285, 2.4; 4680 x 1536 -> 8960, 12 stages a
// tile, 80, 1.6.  (A library's product with one scale per tensor: 2.6 PFLOP/s, 259 us, 85.)  What the stages wait for is the compute
// unit's load path, 64 KB a stage, not the misses of L2 (28 %): lines brought into L2 two stages early cost 8 %, their own requests.
// Patches of 4, 6, 8 or 12 strips: no difference, 19 worse; a workgroup that goes on to further tiles with the operands of its next step
// in flight: slower (they are copied at each tile's end).  With the gated residual the 256-row form spills 11 registers.
constexpr int kTileN = 256, kSlot = 128 * kBlock8, kRing = 9;
constexpr int kScaleAt = kRing * kSlot, kScaleSlot = 256;
constexpr int kLdsBytes = kScaleAt + 4 * kScaleSlot;
constexpr int kGroupM = 8;                   // row tiles per patch of the tile order

// BYTES a lane from base + off to LDS at lds_addr + ADD, lane after lane
template <int BYTES, int ADD>
__device__ __forceinline__ void l8_load_lds(const void* base, uint32_t off, uint32_t lds_addr) {
    static_assert(BYTES == 16 || BYTES == 4, "");
    if constexpr (BYTES == 16)
        asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_addr), "v"(off), "s"(base), "n"(ADD) : "memory", "m0", "scc");
    else
        asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_addr), "v"(off), "s"(base), "n"(ADD) : "memory", "m0", "scc");
}
// waits until at most N of this wave's requests are outstanding (they complete in order) and its LDS reads are done, then the barrier
template <int N>
__device__ __forceinline__ void l8_wait_stage() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }
template <int OFF>
__device__ __forceinline__ u32x4 l8_lds_read16(uint32_t addr) {
    return *(const __attribute__((address_space(3))) u32x4*)(size_t)(addr + OFF);
}
__device__ __forceinline__ uint32_t l8_lds_read4(uint32_t addr) { return *(const __attribute__((address_space(3))) uint32_t*)(size_t)addr; }
__device__ __forceinline__ i32x8 l8_join(u32x4 a, u32x4 b) {
    return __builtin_shufflevector(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), 0, 1, 2, 3, 4, 5, 6, 7);
}

// where a wave's requests go: quarter stages of 128 rows (4 requests each), then the scales
template <int TB>
struct L8Src {
    const uint8_t *w, *x, *s;                // of the stage to be requested next
    uint32_t w_off[8], x_off[2 * TB], s_off;
    uint32_t lds;                            // LDS address of this wave's first 1 KB in slot 0
};
__device__ __forceinline__ uint32_t l8_wrap(uint32_t slot) { return slot >= kRing ? slot - kRing : slot; }
// request J of the quarters Q0, Q0 + 1, .. of a stage whose first quarter is in `slot`; past the last quarter: the scales
template <int TB, int Q0, int J>
__device__ __forceinline__ void l8_request(const L8Src<TB>& src, uint32_t slot, uint32_t scale_addr) {
    constexpr int q = Q0 + J / 4, j = J % 4, NQ = 2 + TB / 2;
    if constexpr (q == NQ) {
        static_assert(j == 0, "one request for the scales");
        l8_load_lds<4, 0>(src.s, src.s_off, scale_addr);
    } else {
        const uint32_t at = src.lds + l8_wrap(slot + q) * kSlot;
        if constexpr (q < 2) l8_load_lds<16, j * 4096>(src.w, src.w_off[4 * q + j], at);
        else l8_load_lds<16, j * 4096>(src.x, src.x_off[4 * (q - 2) + j], at);
    }
}
// piece J of an operand set: two pieces of each weight block, then of each activation block
template <int TB, int J>
__device__ __forceinline__ void l8_fetch(u32x4 (&fn)[8 + 2 * TB], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
    if constexpr (J < 8) fn[J] = l8_lds_read16<(J >> 1) * 4096>(J & 1 ? a1 : a0);
    else fn[J] = l8_lds_read16<((J - 8) >> 1) * 4096>(J & 1 ? b1 : b0);
}
template <int TB, int... J>
__device__ __forceinline__ void l8_fetch_all(std::integer_sequence<int, J...>, u32x4 (&fn)[8 + 2 * TB], uint32_t a0, uint32_t a1, uint32_t b0,
                                             uint32_t b1) {
    (l8_fetch<TB, J>(fn, a0, a1, b0, b1), ...);
}
// One k step: 4 x TB matrix instructions on the operand set fc.  Behind each of them go some of the LDS reads of the next set fn and of
// NLOAD requests (from quarter Q0 on), so that their issue runs under the matrix pipe.
template <int TB, bool FETCH, int NLOAD, int Q0, int I>
__device__ __forceinline__ void l8_kone(f32x16 (&acc)[4][TB], const u32x4 (&fc)[8 + 2 * TB], u32x4 (&fn)[8 + 2 * TB], uint32_t a0, uint32_t a1,
                                        uint32_t b0, uint32_t b1, int we, int xe, const L8Src<TB>& src, uint32_t slot, uint32_t scale_addr) {
    // A matrix instruction takes the time of a dozen others.  The reads are done three of them before the end of the step, where
    // they are waited for; requests go one behind each where there are many, else behind the reads.
    constexpr int kMM = 4 * TB, kReads = 8 + 2 * TB, kTwo = kMM == 16 ? (NLOAD > 4 ? 4 : 8) : kMM;
    constexpr int kR0 = I < kTwo ? 2 * I : kTwo + I, kR1 = I < kTwo ? kR0 + 2 : kR0 + 1;
    constexpr int kLd = NLOAD > kMM ? 2 : 1, kL0 = NLOAD > 4 || kMM < 16 ? kLd * I : I - 8, kL1 = kL0 + kLd;
    constexpr int cb = I / TB, tb = I % TB;
    acc[cb][tb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(l8_join(fc[2 * cb], fc[2 * cb + 1]), l8_join(fc[8 + 2 * tb], fc[9 + 2 * tb]),
                                                                  acc[cb][tb], 0, 0, 0, we, tb, xe);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (FETCH && kR0 < kReads) l8_fetch<TB, kR0>(fn, a0, a1, b0, b1);
    if constexpr (FETCH && kR1 == kR0 + 2 && kR0 + 1 < kReads) l8_fetch<TB, kR0 + 1>(fn, a0, a1, b0, b1);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kL0 >= 0 && kL0 < NLOAD) l8_request<TB, Q0, kL0>(src, slot, scale_addr);
    if constexpr (kL1 == kL0 + 2 && kL0 + 1 < NLOAD) l8_request<TB, Q0, kL0 + 1>(src, slot, scale_addr);
    __builtin_amdgcn_sched_barrier(0);
}
template <int TB, bool FETCH, int NLOAD, int Q0, int... I>
__device__ __forceinline__ void l8_kstep(std::integer_sequence<int, I...>, f32x16 (&acc)[4][TB], const u32x4 (&fc)[8 + 2 * TB],
                                         u32x4 (&fn)[8 + 2 * TB], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1, int we, int xe,
                                         const L8Src<TB>& src, uint32_t slot, uint32_t scale_addr) {
    (l8_kone<TB, FETCH, NLOAD, Q0, I>(acc, fc, fn, a0, a1, b0, b1, we, xe, src, slot, scale_addr), ...);
}

// Four neighbouring values of a row, eight of them: zeros past the last channel.
__device__ __forceinline__ u32x2 l8_raw4(const uint16_t* s, int left) {
    if (left >= 4) return *(const u32x2_any*)s;
    u32x2 w = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) w[i >> 1] |= (uint32_t)s[i] << (16 * (i & 1));
    return w;
}
__device__ __forceinline__ u32x4 l8_raw8(const uint16_t* s, int left) {
    if (left >= 8) return *(const u32x4_any*)s;
    const u32x2 lo = l8_raw4(s, left), hi = l8_raw4(s + 4, left - 4);
    return u32x4{lo.x, lo.y, hi.x, hi.y};
}
// LDS accesses of a wave's lanes before this come before those behind it (a wave's are done in order: nothing to wait for)
__device__ __forceinline__ void l8_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Sums to memory: 4 x TB blocks of 32 channels x 32 rows from channel c0, row r0 on.  Lane (m, hf) of block (cb, tb) holds row
// 32 tb + m, channels 8 g + 4 hf + (i & 3), i = 4 g + ..  32 rows x 128 channels at a time pass through the wave's own `lds`, so that a
// store takes four rows of 256 bytes, whole cache lines; a residual comes in the same way.  (Stored from the registers, 32 rows
// of 32 bytes a time, 32760 x 1536 -> 8960 takes 548 us against 464, 4680 x 5120 -> 13824 294 against 283.)
constexpr int kOutPitch = 256 + 16;                            // the 16-byte pieces of a column of rows sit in different banks
template <class E, int EPI, int TB>
__device__ __forceinline__ void l8_store(const L8Args& p, const f32x16 (&acc)[4][TB], int c0, int64_t r0, int lane, uint8_t* lds) {
    const int m = lane & 31, hf = lane >> 5, l16 = lane & 15, q = lane >> 4;
    const int pc = c0 + 8 * l16, left = p.N - pc;              // a lane's piece of a row in memory
    uint8_t *at_row = lds + q * kOutPitch + l16 * 16, *at_sum = lds + m * kOutPitch + hf * 16;
    u32x2 bia[4][4];
#pragma unroll
    for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = c0 + 32 * cb + 8 * g + 4 * hf;
            bia[cb][g] = p.bias != nullptr ? l8_raw4(p.bias + c, p.N - c) : u32x2{0u, 0u};
        }
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
        const int64_t row0 = r0 + 32 * tb;
        if (EPI == SFM_EPI_GATE_RESIDUAL) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t row = row0 + 4 * i + q;
                u32x4 v = {0u, 0u, 0u, 0u};
                if (row < p.M) v = l8_raw8(p.res + row * p.res_stride + pc, left);
                *(u32x4*)(at_row + 4 * i * kOutPitch) = v;
            }
            l8_wave_sync();
        }
        int64_t row = row0 + m;
        if (row >= p.M) row = p.M - 1;
        const uint16_t* gp = EPI == SFM_EPI_GATE_RESIDUAL && p.gate != nullptr ? p.gate + (row / p.rows_per_frame) * p.gate_stride : nullptr;
#pragma unroll
        for (int cb = 0; cb < 4; ++cb) {
            float bf[16], res[16], gate[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                l8_unpack4<E>(bia[cb][g], bf + 4 * g);
                if (EPI == SFM_EPI_GATE_RESIDUAL) {
                    const int c = c0 + 32 * cb + 8 * g + 4 * hf;
                    l8_unpack4<E>(*(const u32x2*)(lds + m * kOutPitch + (32 * cb + 8 * g + 4 * hf) * 2), res + 4 * g);
                    if (gp != nullptr) {
                        l8_unpack4<E>(l8_raw4(gp + c, p.N - c), gate + 4 * g);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) gate[4 * g + i] = 1.f;
                    }
                }
            }
            if (EPI == SFM_EPI_GATE_RESIDUAL) l8_wave_sync();
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 16; i += 2)
                w[i / 2] = pack2<E>(l8_tail<E, EPI>(acc[cb][tb][i], bf[i], res[i], gate[i]),
                                    l8_tail<E, EPI>(acc[cb][tb][i + 1], bf[i + 1], res[i + 1], gate[i + 1]));
#pragma unroll
            for (int h = 0; h < 2; ++h) {                      // the two lanes of a row exchange halves: 16 bytes each
                auto rx = __builtin_amdgcn_permlane32_swap(w[4 * h], w[4 * h + 2], false, false);
                auto ry = __builtin_amdgcn_permlane32_swap(w[4 * h + 1], w[4 * h + 3], false, false);
                *(u32x4*)(at_sum + cb * 64 + h * 32) = u32x4{(uint32_t)rx[0], (uint32_t)ry[0], (uint32_t)rx[1], (uint32_t)ry[1]};
            }
        }
        l8_wave_sync();
        u32x4 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = *(const u32x4*)(at_row + 4 * i * kOutPitch);
        l8_wave_sync();
        uint16_t* out = p.out + (row0 + q) * p.out_stride + pc;
        const int64_t rows = p.M - row0 - q;                   // those from this lane's first on
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (4 * i < rows && left >= 8) {
                *(u32x4_any*)(out + 4 * i * p.out_stride) = o[i];
            } else if (4 * i < rows) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < left) out[4 * i * p.out_stride + e] = (uint16_t)(o[i][e >> 1] >> (16 * (e & 1)));
            }
        }
    }
}

// One tile: strip rows m0 .., channels n0 ..
template <class E, int EPI, int TB>
__device__ __forceinline__ void l8_tile(const L8Args& p, int64_t m0, int n0) {
    constexpr int kTileM = 64 * TB;
    constexpr int NQ = 2 + TB / 2, kLoads = 4 * NQ + 1;        // slots and a wave's requests of a stage
    constexpr int kAhead = TB == 4 ? 2 : 3;                    // stage s + kAhead is requested while stage s is multiplied ..
    constexpr int kEarly = TB == 4 ? 4 : 0;                    // .. so many of its requests before stage s has been read
    constexpr int kOut = kEarly + (kAhead - 2) * kLoads;       // requests of later stages under way when stage s + 1 is needed
    extern __shared__ __attribute__((aligned(256))) uint8_t l8_lds[];
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)l8_lds;
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave & 1, wm = wave >> 1;

    // request j of a wave fills rows 8 (4 j + wave) .. + 7 of a slot; rows past the end repeat the last
    L8Src<TB> src;
    src.w = p.w + (int64_t)n0 * p.kp;
    src.x = p.x + m0 * p.kp;
    src.s = p.xscale + m0;                                     // 128 bytes of scales per 128 rows
    src.lds = lds0 + (uint32_t)wave * 1024;
    {
        const int g_row = lane >> 3, g_c = (lane & 7) ^ ((((wave & 1) << 2) + (lane >> 4)) & 7);
        const int wlast = p.N - 1 - n0, xlast = (int)min(p.M - 1 - m0, (int64_t)kTileM - 1);
#pragma unroll
        for (int j = 0; j < 8; ++j) src.w_off[j] = (uint32_t)min((4 * j + wave) * 8 + g_row, wlast) * (uint32_t)p.kp + g_c * 16;
#pragma unroll
        for (int j = 0; j < 2 * TB; ++j) src.x_off[j] = (uint32_t)min((4 * j + wave) * 8 + g_row, xlast) * (uint32_t)p.kp + g_c * 16;
        src.s_off = (uint32_t)(lane * 4 - (m0 + 128 < p.M ? 0 : 128 * hf));
    }
    const int64_t s_step = p.groups * 128;
    auto advance = [&]() {
        src.w += kBlock8;
        src.x += kBlock8;
        src.s += s_step;
    };
    const auto* wsp = (const __attribute__((address_space(4))) uint32_t*)(size_t)(p.wscale + (int64_t)min((n0 >> 7) + wn, (p.N - 1) >> 7) * p.pitch);

    f32x16 acc[4][TB];
#pragma unroll
    for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[cb][tb][i] = 0.f;

    // operand read addresses of the pieces of a row, relative to a slot; the wave's weight and activation rows in a stage
    const int sw = (m >> 1) & 7;
    uint32_t kp4[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) kp4[q] = lds0 + (uint32_t)(m * 128) + (uint32_t)(((2 * q + hf) ^ sw) << 4);
    const uint32_t bq = TB == 4 ? 2 + wm : 2, bo = TB == 4 ? 0 : wm * 8192;
    const uint32_t ks = lds0 + kScaleAt + (uint32_t)(((TB == 4 ? wm : 0) * 32 + m) * 4);
    const int xsh = TB == 4 ? 0 : 16 * wm;

    // Quarter q of stage s lives in slot (NQ s + q) % 9.  Iteration s multiplies stage s in two k steps; the operands of a step are
    // read during the step before.  After its first step a wave has read all of stage s: it waits for that and for its own loads
    // of stage s + 1, meets the others, and requests stage s + kAhead into the slots that are free (TB = 4: its first quarter has a slot
    // already before that).
    const int nstage = p.nkb;
    auto whole_stage = [&](int g) {
        const uint32_t slot = (uint32_t)(NQ * g) % kRing, sc = lds0 + kScaleAt + g * kScaleSlot;
#define L8_RQ(J) if constexpr ((J) < kLoads) l8_request<TB, 0, (J) < kLoads ? (J) : 0>(src, slot, sc);
        L8_RQ(0) L8_RQ(1) L8_RQ(2) L8_RQ(3) L8_RQ(4) L8_RQ(5) L8_RQ(6) L8_RQ(7) L8_RQ(8) L8_RQ(9) L8_RQ(10) L8_RQ(11) L8_RQ(12)
        L8_RQ(13) L8_RQ(14) L8_RQ(15) L8_RQ(16)
#undef L8_RQ
        advance();
    };
    whole_stage(0);
    if (nstage > 1) whole_stage(1);
    if (kAhead == 3 && nstage > 2) whole_stage(2);
    if (kAhead == 3 && nstage > 2) l8_wait_stage<2 * kLoads>();
    else if (nstage > 1) l8_wait_stage<kLoads>();
    else l8_wait_stage<0>();
    u32x4 f0[8 + 2 * TB], f1[8 + 2 * TB];
    uint32_t hs = 0;                                           // slot of the first quarter of the stage being multiplied
    uint32_t xe0 = l8_lds_read4(ks);                           // this lane's scales of the stage
    {
        const uint32_t a = wn * kSlot, b = bq * kSlot + bo;
        l8_fetch_all<TB>(std::make_integer_sequence<int, 8 + 2 * TB>{}, f0, kp4[0] + a, kp4[1] + a, kp4[0] + b, kp4[1] + b);
    }
    int s = 0;
    uint32_t wword = wsp[0];                                   // the word with the weight scale of the stage
    // LOAD: request stage s + kAhead; WAIT: requests that may be under way at the barrier; LAST: nothing follows
#define L8_ITER(LOAD, WAIT, LAST)                                                                                              \
    {                                                                                                                          \
        const uint32_t sa = l8_wrap(hs + wn) * kSlot, sb = l8_wrap(hs + bq) * kSlot + bo;                                      \
        const uint32_t ns = l8_wrap(hs + (NQ * kAhead) % kRing);                                                               \
        const uint32_t sc = lds0 + kScaleAt + (uint32_t)((s + kAhead) & 3) * kScaleSlot;                                       \
        __builtin_amdgcn_sched_barrier(0);                                                                                     \
        const int wec = (int)(wword >> (8 * (s & 3))) & 0xff, xe = (int)(xe0 >> xsh);                                          \
        if (!LAST) wword = wsp[(s + 1) >> 2];                                                                                  \
        l8_kstep<TB, true, LOAD ? kEarly : 0, 0>(std::make_integer_sequence<int, 4 * TB>{}, acc, f0, f1, kp4[2] + sa, kp4[3] + sa, \
                                                           kp4[2] + sb, kp4[3] + sb, wec, xe, src, ns, sc);                    \
        __builtin_amdgcn_sched_barrier(0);                                                                                     \
        if (!LAST) {                                                                                                           \
            l8_wait_stage<WAIT>();                                                                                             \
            hs = l8_wrap(hs + NQ);                                                                                             \
            const uint32_t na = l8_wrap(hs + wn) * kSlot, nb = l8_wrap(hs + bq) * kSlot + bo;                                  \
            xe0 = l8_lds_read4(ks + (uint32_t)((s + 1) & 3) * kScaleSlot);                                                     \
            l8_kstep<TB, true, LOAD ? kLoads - kEarly : 0, kEarly / 4>(std::make_integer_sequence<int, 4 * TB>{}, acc, f1, f0, \
                                                                                 kp4[0] + na, kp4[1] + na, kp4[0] + nb, kp4[1] + nb, wec, xe, src, ns, sc); \
            if (LOAD) advance();                                                                                               \
            ++s;                                                                                                               \
        } else {                                                                                                               \
            l8_kstep<TB, false, 0, 0>(std::make_integer_sequence<int, 4 * TB>{}, acc, f1, f0, 0, 0, 0, 0, wec, xe, src, 0, 0); \
        }                                                                                                                      \
    }
    while (s + kAhead < nstage) L8_ITER(true, kOut, false)
    if (kAhead == 3 && nstage >= 3) L8_ITER(false, kLoads, false)
    if (nstage >= 2) L8_ITER(false, 0, false)
    L8_ITER(false, 0, true)
#undef L8_ITER
    __syncthreads();                                           // every wave has read its operands: LDS is free
    l8_store<E, EPI, TB>(p, acc, n0 + wn * 128, m0 + wm * 32 * TB, lane, l8_lds + wave * 32 * kOutPitch);
}

// Every eighth workgroup shares an XCD: each XCD gets a contiguous run of the patch order.  With TB = 4 a last strip of at most 128
// rows is made of half tiles, which come last and fill the last round of the compute units.
template <class E, int EPI, int TB>
__global__ __launch_bounds__(256) void l8_tile_kernel(L8Args p) {
    const int strips = p.tm - p.half, all = strips * p.tn, per_xcd = (all + 7) / 8, blk = (int)blockIdx.x;
    if (blk < 8 * per_xcd) {
        const int v = (blk & 7) * per_xcd + (blk >> 3);
        if (v >= all) return;
        const int patch = v / (kGroupM * p.tn), first = patch * kGroupM, gsize = min(kGroupM, strips - first);
        const int within = v - patch * kGroupM * p.tn;
        const int tn = __builtin_amdgcn_readfirstlane(within / gsize);
        l8_tile<E, EPI, TB>(p, (int64_t)__builtin_amdgcn_readfirstlane(first + within - tn * gsize) * (64 * TB), tn * kTileN);
    } else if (TB == 4) {
        const int per = (p.tn + 7) / 8, h = blk - 8 * per_xcd, v = (h & 7) * per + (h >> 3);
        if (v < p.tn) l8_tile<E, EPI, 2>(p, (int64_t)strips * 256, v * kTileN);
    }
}

template <class E, int EPI, int TB>
int launch_tile(const L8Args& a0, bool half, hipStream_t st) {
    static bool configured = false;          // the attribute belongs to the function; racing callers set the same value
    if (!configured) {
        hipError_t e = hipFuncSetAttribute((const void*)l8_tile_kernel<E, EPI, TB>, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
        if (e != hipSuccess) {
            set_error("sfm_linear8: hipFuncSetAttribute failed: %s", hipGetErrorString(e));
            return SFM_ERR_HIP;
        }
        configured = true;
    }
    L8Args a = a0;
    a.tm = (int)((a.M + 64 * TB - 1) / (64 * TB));
    a.tn = (a.N + kTileN - 1) / kTileN;
    a.half = half;
    const int64_t full = ((int64_t)(a.tm - a.half) * a.tn + 7) / 8 * 8, halves = a.half ? (a.tn + 7) / 8 * 8 : 0;
    hipLaunchKernelGGL((l8_tile_kernel<E, EPI, TB>), dim3((unsigned)(full + halves)), dim3(256), kLdsBytes, st, a);
    return launched8("sfm_linear8");
}

// Which kernel.  Times of a round of tiles over the compute units, fitted to measurements from 12 to 70 stages (us): 256 rows 8 + 1.2
// a stage, 128 rows 7 + 0.9.  Measured on both sides: 4680 x 8960 -> 1536 (114 or 222 tiles, one round) 87 against 67; 4680 x 1536 ->
// 8960 (665 or 1295) 82 against 99; 1560 x 1536 -> 8960 (245 or 455) 27 against 35.  The kernel without LDS runs at up to 0.5
// PFLOP/s behind 6 us, and wins where the tiles are few: 512 x 1536 -> 1536 13 against 15, 1111 x 1000 -> 777 12 against 32.
struct L8Plan {
    int rows;                                // of a tile: 256 or 128; 0: the kernels without LDS tiles
    bool half;                               // the last strip of 256-row tiles is made of half ones
};
L8Plan l8_plan(int64_t M, int N, int nkb) {
    if (M <= 16) return {0, false};
    const double cus = cu_count(), tn = (N + kTileN - 1) / kTileN;
    auto rounds = [&](double tiles) { return tiles < cus ? 1.0 : tiles / cus + 0.3; };
    const double t4 = rounds(tn * (double)((M + 255) / 256)) * (8.0 + 1.2 * nkb);
    const double t2 = rounds(tn * (double)((M + 127) / 128)) * (7.0 + 0.9 * nkb);
    const double flops = 2.0 * M * N * nkb * kBlock8, direct = 6.0 + 0.35 * nkb + flops / 0.5e9;
    if (direct < t2 && direct < t4) return {0, false};
    return t2 < t4 ? L8Plan{128, false} : L8Plan{256, M % 256 != 0 && M % 256 <= 128};
}
template <class E, int EPI>
int launch_epi(const L8Args& a, hipStream_t st) {
    if (a.M <= 16) return few_wide(a) ? launch_direct<E, EPI, 1, 1, 16>(a, st) : launch_direct<E, EPI, 1, 1, 8>(a, st);
    const L8Plan plan = l8_plan(a.M, a.N, a.nkb);
    return plan.rows == 0 ? launch_direct<E, EPI, 4, 2, 8>(a, st) : plan.rows == 128 ? launch_tile<E, EPI, 2>(a, false, st)
                                                                                     : launch_tile<E, EPI, 4>(a, plan.half, st);
}

template <class E>
int launch_dtype(const L8Args& a, int epilogue, hipStream_t st) {
    if (epilogue == SFM_EPI_GELU_TANH) return launch_epi<E, SFM_EPI_GELU_TANH>(a, st);
    if (epilogue == SFM_EPI_GATE_RESIDUAL) return launch_epi<E, SFM_EPI_GATE_RESIDUAL>(a, st);
    return launch_epi<E, SFM_EPI_NONE>(a, st);
}

template <class E>
int few_dtype(const L8Args& a, int epilogue, const void* x, int64_t xstride, int K, hipStream_t st) {
    if (epilogue == SFM_EPI_GELU_TANH) return launch_few<E, SFM_EPI_GELU_TANH>(a, x, xstride, K, st);
    if (epilogue == SFM_EPI_GATE_RESIDUAL) return launch_few<E, SFM_EPI_GATE_RESIDUAL>(a, x, xstride, K, st);
    return launch_few<E, SFM_EPI_NONE>(a, x, xstride, K, st);
}

}  // namespace

int tile_rows8(int64_t M, int N, int K, bool* half_strip) {
    const L8Plan plan = l8_plan(M, N, blocks8(K));
    *half_strip = plan.half;
    return plan.rows;
}

int launch_linear8(const sfm_linear8_desc& d, const void* x, int64_t x_stride, const void* x8, const void* xscale, const void* w8,
                   const void* wscale, const void* bias, const void* res, const void* gate, void* out, hipStream_t stream) {
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
    if (x != nullptr && d.M <= kFewRows8)
        return d.dtype == SFM_BF16 ? few_dtype<BF16>(a, d.epilogue, x, x_stride, d.K, stream) : few_dtype<F16>(a, d.epilogue, x, x_stride, d.K, stream);
    return d.dtype == SFM_BF16 ? launch_dtype<BF16>(a, d.epilogue, stream) : launch_dtype<F16>(a, d.epilogue, stream);
}

}  // namespace sfm
