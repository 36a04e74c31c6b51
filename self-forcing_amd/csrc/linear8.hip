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
    int tm, tn;              // tiles along M and N
    bool vec;                // rows of out, res, gate and bias allow 8-byte accesses
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

// four neighbouring channels c.. of a row: bias and epilogue on the fp32 sums, rounded once and stored
template <class E, int EPI>
__device__ __forceinline__ void l8_finish4(const L8Args& p, int64_t row, int c, const float* acc) {
    if (row >= p.M || c >= p.N) return;
    const bool full = p.vec && c + 4 <= p.N;
    float v[4], r[4] = {0.f, 0.f, 0.f, 0.f}, g[4] = {1.f, 1.f, 1.f, 1.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    auto get4 = [&](const uint16_t* s, float* d) {
        if (full) {
            l8_unpack4<E>(*(const u32x2*)s, d);
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
    for (int i = 0; i < 4; ++i) v[i] = l8_tail<E, EPI>(acc[i], b[i], r[i], g[i]);
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
constexpr int kTileN = 256, kSlot = 128 * kBlock8, kRing = 9;
constexpr int kScaleAt = kRing * kSlot, kScaleSlot = 256, kLdsBytes = kScaleAt + 4 * kScaleSlot;
constexpr int kGroupM = 8;                   // row tiles per patch of the tile order

template <int BYTES>
__device__ __forceinline__ void l8_load_lds(const void* base, uint32_t off, uint32_t lds_addr) {
    static_assert(BYTES == 16 || BYTES == 4, "");
    if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_addr), "v"(off), "s"(base) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_addr), "v"(off), "s"(base) : "memory", "m0");
}
// waits until at most N of this wave's loads are outstanding (they complete in order), then the barrier
template <int N>
__device__ __forceinline__ void l8_wait_stage() { asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory"); }
template <int OFF>
__device__ __forceinline__ u32x4 l8_lds_read16(uint32_t addr) {
    u32x4 r;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
    return r;
}
__device__ __forceinline__ uint32_t l8_lds_read4(uint32_t addr) {
    uint32_t r;
    asm volatile("ds_read_b32 %0, %1" : "=v"(r) : "v"(addr));
    return r;
}
template <int NF>
__device__ __forceinline__ void l8_wait_frags(u32x4 (&f)[NF], uint32_t& xe) {
    static_assert(NF == 16 || NF == 12, "two pieces of 4 weight blocks + 4 or 2 activation blocks");
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]), "+v"(f[4]), "+v"(f[5]), "+v"(f[6]), "+v"(f[7]),
                 "+v"(f[8]), "+v"(f[9]), "+v"(f[10]), "+v"(f[11]), "+v"(xe));
    if constexpr (NF == 16) asm volatile("" : "+v"(f[12]), "+v"(f[13]), "+v"(f[14]), "+v"(f[15]));
}
__device__ __forceinline__ i32x8 l8_join(u32x4 a, u32x4 b) {
    return __builtin_shufflevector(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), 0, 1, 2, 3, 4, 5, 6, 7);
}

// where a wave's loads go: request j of a list of quarter stages (4 requests each), then the scales
template <int TB>
struct L8Src {
    const uint8_t *w, *x, *s;                // stage of the next request
    uint32_t w_off[8], x_off[2 * TB], s_off;
    uint32_t lds;                            // LDS address of this wave's first 1 KB in slot 0
};
// request j (0 ..) of quarters Q0, Q0 + 1, .. of a stage whose first quarter is in slot `slot`; past the last quarter: the scales
template <int TB, int Q0, int J>
__device__ __forceinline__ void l8_request(const L8Src<TB>& src, uint32_t slot, uint32_t scale_addr) {
    constexpr int q = Q0 + J / 4, j = J % 4, NQ = 2 + TB / 2;
    if constexpr (q == NQ) {
        static_assert(j == 0, "one request for the scales");
        l8_load_lds<4>(src.s, src.s_off, scale_addr);
    } else {
        uint32_t at = slot + q;
        at = at >= kRing ? at - kRing : at;
        if constexpr (q < 2) l8_load_lds<16>(src.w, src.w_off[4 * q + j], src.lds + at * kSlot + j * 4096);
        else l8_load_lds<16>(src.x, src.x_off[4 * (q - 2) + j], src.lds + at * kSlot + j * 4096);
    }
}

template <int TB, int J>
__device__ __forceinline__ void l8_fetch(u32x4 (&fn)[8 + 2 * TB], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
    if constexpr (J < 8) fn[J] = l8_lds_read16<(J >> 1) * 4096>(J & 1 ? a1 : a0);
    else if constexpr (J < 8 + 2 * TB) fn[J] = l8_lds_read16<((J - 8) >> 1) * 4096>(J & 1 ? b1 : b0);
}
// One k step: 4 TB matrix instructions on the operand set fc (piece pairs of blocks 0..3: weights, 4..: activations).  Behind each
// of them go some of the LDS reads of the next set fn and of the NLOAD requests (from quarter Q0 on), so that their issue runs
// under the matrix pipe.
#define L8_KS(I)                                                                                                              \
    if constexpr ((I) < 4 * TB) {                                                                                             \
        constexpr int cb = (I) / TB, tb = (I) % TB;                                                                           \
        acc[cb][tb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(l8_join(fc[2 * cb], fc[2 * cb + 1]),                    \
                                                                      l8_join(fc[8 + 2 * tb], fc[9 + 2 * tb]), acc[cb][tb], 0, 0, 0, we, tb, xe); \
        __builtin_amdgcn_sched_barrier(0);                                                                                    \
        if constexpr (FETCH) {                                                                                                \
            l8_fetch<TB, (I) * kRd>(fn, a0, a1, b0, b1);                                                                      \
            if constexpr (kRd == 2) l8_fetch<TB, (I) * kRd + 1>(fn, a0, a1, b0, b1);                                          \
            __builtin_amdgcn_sched_barrier(0);                                                                                \
        }                                                                                                                     \
        if constexpr ((I) * kLd < NLOAD) {                                                                                    \
            l8_request<TB, Q0, (I) * kLd>(src, slot, scale_addr);                                                             \
            if constexpr (kLd == 2 && (I) * kLd + 1 < NLOAD) l8_request<TB, Q0, (I) * kLd + 1>(src, slot, scale_addr);        \
            __builtin_amdgcn_sched_barrier(0);                                                                                \
        }                                                                                                                     \
    }
template <int TB, bool FETCH, int NLOAD, int Q0>
__device__ __forceinline__ void l8_kstep(f32x16 (&acc)[4][TB], const u32x4 (&fc)[8 + 2 * TB], u32x4 (&fn)[8 + 2 * TB], uint32_t a0, uint32_t a1,
                                         uint32_t b0, uint32_t b1, int we, int xe, const L8Src<TB>& src, uint32_t slot, uint32_t scale_addr) {
    constexpr int kRd = TB == 4 ? 1 : 2;                       // LDS reads per matrix instruction
    constexpr int kLd = NLOAD > 4 * TB ? 2 : 1;                // requests per matrix instruction
    static_assert(NLOAD <= kLd * 4 * TB, "requests fit the step");
    L8_KS(0) L8_KS(1) L8_KS(2) L8_KS(3) L8_KS(4) L8_KS(5) L8_KS(6) L8_KS(7)
    L8_KS(8) L8_KS(9) L8_KS(10) L8_KS(11) L8_KS(12) L8_KS(13) L8_KS(14) L8_KS(15)
}
#undef L8_KS

template <class E, int EPI, int TB>
__global__ __launch_bounds__(256) void l8_tile_kernel(L8Args p) {
    constexpr int kTileM = 64 * TB;
    constexpr int NQ = 2 + TB / 2, kLoads = 4 * NQ + 1;        // slots and a wave's load instructions of a stage
    constexpr int kAhead = TB == 4 ? 2 : 3;                    // stage s + kAhead is requested while stage s is multiplied ..
    constexpr int kEarly = TB == 4 ? 4 : 0;                    // .. so many of its requests before stage s has been read
    extern __shared__ __attribute__((aligned(256))) uint8_t l8_lds[];
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)l8_lds;
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave & 1, wm = wave >> 1;

    // every eighth workgroup shares an XCD: each XCD gets a contiguous run of the patch order
    const int ntiles = p.tm * p.tn, per_xcd = (ntiles + 7) / 8;
    const int v = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
    if (v >= ntiles) return;
    const int patch = v / (kGroupM * p.tn), first = patch * kGroupM, gsize = min(kGroupM, p.tm - first);
    const int within = v - patch * kGroupM * p.tn;
    const int tile_n = __builtin_amdgcn_readfirstlane(within / gsize);
    const int64_t m0 = (int64_t)__builtin_amdgcn_readfirstlane(first + within - tile_n * gsize) * kTileM;
    const int n0 = tile_n * kTileN;

    // request j of a wave fills rows 8 (4 j + wave) .. + 7 of a slot; rows past the end repeat the last
    L8Src<TB> src;
    src.w = p.w + (int64_t)n0 * p.kp;
    src.x = p.x + m0 * p.kp;
    src.s = p.xscale;
    src.lds = lds0 + (uint32_t)wave * 1024;
    {
        const int g_row = lane >> 3, g_c = (lane & 7) ^ ((((wave & 1) << 2) + (lane >> 4)) & 7);
        const int wlast = p.N - 1 - n0, xlast = (int)min(p.M - 1 - m0, (int64_t)kTileM - 1);
#pragma unroll
        for (int j = 0; j < 8; ++j) src.w_off[j] = (uint32_t)min((4 * j + wave) * 8 + g_row, wlast) * (uint32_t)p.kp + g_c * 16;
#pragma unroll
        for (int j = 0; j < 2 * TB; ++j) src.x_off[j] = (uint32_t)min((4 * j + wave) * 8 + g_row, xlast) * (uint32_t)p.kp + g_c * 16;
        src.s += min(m0 >> 7, p.groups - 1) * 128;
        src.s_off = (uint32_t)(lane * 4 - ((m0 >> 7) + 1 < p.groups ? 0 : 128 * hf));
    }
    const int64_t s_step = p.groups * 128;
    auto advance = [&]() {
        src.w += kBlock8;
        src.x += kBlock8;
        src.s += s_step;
    };
    const auto* wsp = (const __attribute__((address_space(4))) uint32_t*)(size_t)(p.wscale + (int64_t)min((n0 >> 7) + wn, (p.N - 1) >> 7) * p.pitch);
    auto w_exp = [&](int s) { return (int)(wsp[s >> 2] >> (8 * (s & 3))) & 0xff; };

    f32x16 acc[4][TB];
#pragma unroll
    for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[cb][tb][i] = 0.f;

    // operand read addresses of the pieces of a row, relative to a slot (of the wave's weight rows / activation rows)
    const int sw = (m >> 1) & 7;
    uint32_t ka[4], kb[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t ko = (uint32_t)(((2 * q + hf) ^ sw) << 4);
        ka[q] = lds0 + (uint32_t)(m * 128) + ko;
        kb[q] = lds0 + (uint32_t)(((TB == 4 ? 0 : wm * 64) + m) * 128) + ko;
    }
    const uint32_t ks = lds0 + kScaleAt + (uint32_t)(((TB == 4 ? wm : 0) * 32 + m) * 4);
    const int xsh = TB == 4 ? 0 : 16 * wm;

    // Quarter q of stage s lives in slot (NQ s + q) % 9.  Iteration s multiplies stage s in two k steps; the operands of a step are
    // read during the step before.  After its first step a wave has read all of stage s: it waits for its own loads of stage
    // s + 1, meets the others, and requests the next stage into the slots of stage s (TB = 4: the first quarter of stage s + 2 has
    // a slot already before that).
    const int nstage = p.nkb;
    auto wrap = [](uint32_t h) { return h >= kRing ? h - kRing : h; };
    auto scale_at = [&](int s) { return lds0 + kScaleAt + (uint32_t)(s & 3) * kScaleSlot; };
    auto whole_stage = [&](int s) {
        const uint32_t slot = (uint32_t)(NQ * s) % kRing;
#define L8_RQ(J) if constexpr ((J) < kLoads) l8_request<TB, 0, (J) < kLoads ? (J) : 0>(src, slot, scale_at(s));
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
    uint32_t xe0, xe1;
    xe0 = l8_lds_read4(ks);
    {
        const uint32_t a = wn * kSlot, b = (2 + (TB == 4 ? wm : 0)) * kSlot;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            f0[0 + c] = l8_lds_read16<0>(ka[c] + a);
            f0[2 + c] = l8_lds_read16<4096>(ka[c] + a);
            f0[4 + c] = l8_lds_read16<8192>(ka[c] + a);
            f0[6 + c] = l8_lds_read16<12288>(ka[c] + a);
            f0[8 + c] = l8_lds_read16<0>(kb[c] + b);
            f0[10 + c] = l8_lds_read16<4096>(kb[c] + b);
            if constexpr (TB == 4) {
                f0[12 + c] = l8_lds_read16<8192>(kb[c] + b);
                f0[14 + c] = l8_lds_read16<12288>(kb[c] + b);
            }
        }
    }
    int s = 0, we = w_exp(0);
    // LOAD: request stage s + kAhead; WAIT: loads that may stay outstanding at the barrier; LAST: no barrier
#define L8_ITER(LOAD, WAIT, LAST)                                                                                              \
    {                                                                                                                          \
        const uint32_t sa = wrap(hs + wn) * kSlot, sb = wrap(hs + 2 + (TB == 4 ? wm : 0)) * kSlot;                             \
        const uint32_t ns = wrap(hs + (NQ * kAhead) % kRing);                                                                  \
        const uint32_t sc = scale_at(s + kAhead);                                                                              \
        const int wec = we;                                                                                                    \
        if (!LAST) we = w_exp(s + 1);                                                                                          \
        l8_wait_frags(f0, xe0);                                                                                                \
        const int xe = (int)(xe0 >> xsh);                                                                                      \
        l8_kstep<TB, true, LOAD ? kEarly : 0, 0>(acc, f0, f1, ka[2] + sa, ka[3] + sa, kb[2] + sb, kb[3] + sb, wec, xe, src, ns, sc); \
        l8_wait_frags(f1, xe0);                                /* this wave has read all of the stage */                       \
        if (!LAST) {                                                                                                           \
            l8_wait_stage<WAIT>();                                                                                             \
            hs = wrap(hs + NQ);                                                                                                \
            const uint32_t na = wrap(hs + wn) * kSlot, nb = wrap(hs + 2 + (TB == 4 ? wm : 0)) * kSlot;                         \
            xe1 = l8_lds_read4(ks + (uint32_t)((s + 1) & 3) * kScaleSlot);                                                     \
            l8_kstep<TB, true, LOAD ? kLoads - kEarly : 0, kEarly / 4>(acc, f1, f0, ka[0] + na, ka[1] + na, kb[0] + nb, kb[1] + nb, wec, xe, src, ns, sc); \
            if (LOAD) advance();                                                                                               \
            xe0 = xe1;                                                                                                         \
            ++s;                                                                                                               \
        } else {                                                                                                               \
            l8_kstep<TB, false, 0, 0>(acc, f1, f0, 0, 0, 0, 0, wec, xe, src, 0, 0);                                            \
        }                                                                                                                      \
    }
    if constexpr (TB == 4) {
        while (s + 2 < nstage) L8_ITER(true, 4, false)
    } else {
        while (s + 3 < nstage) L8_ITER(true, kLoads, false)
        if (nstage >= 3) L8_ITER(false, kLoads, false)
    }
    if (nstage >= 2) L8_ITER(false, 0, false)
    L8_ITER(false, 0, true)
#undef L8_ITER

    // lane (m, hf) of block (cb, tb) holds row 32 tb + m, channels 8 g + 4 hf + (i & 3), i = 4 g + ..
    const int64_t row0 = m0 + wm * 32 * TB + m;
    if (p.vec && n0 + wn * 128 + 128 <= p.N) {                 // whole: 16-byte stores, a block column's operands loaded together
#pragma unroll
        for (int cb = 0; cb < 4; ++cb) {
            const int cbase = n0 + wn * 128 + 32 * cb;
            float bia[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                u32x2 b = {0u, 0u};
                if (p.bias != nullptr) b = *(const u32x2*)(p.bias + cbase + 8 * g + 4 * hf);
                l8_unpack4<E>(b, bia + 4 * g);
            }
#pragma unroll
            for (int tb = 0; tb < TB; ++tb) {
                const int64_t row = row0 + 32 * tb, rc = min(row, p.M - 1);
                float res[16], gate[16];
                if (EPI == SFM_EPI_GATE_RESIDUAL) {
                    const uint16_t *rp = p.res + rc * p.res_stride + cbase + 4 * hf;
                    const uint16_t *gp = p.gate != nullptr ? p.gate + (rc / p.rows_per_frame) * p.gate_stride + cbase + 4 * hf : nullptr;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        l8_unpack4<E>(*(const u32x2*)(rp + 8 * g), res + 4 * g);
                        if (gp != nullptr) {
                            l8_unpack4<E>(*(const u32x2*)(gp + 8 * g), gate + 4 * g);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) gate[4 * g + i] = 1.f;
                        }
                    }
                }
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                    w[i / 2] = pack2<E>(l8_tail<E, EPI>(acc[cb][tb][i], bia[i], res[i], gate[i]),
                                        l8_tail<E, EPI>(acc[cb][tb][i + 1], bia[i + 1], res[i + 1], gate[i + 1]));
#pragma unroll
                for (int gp = 0; gp < 2; ++gp) {               // the two lanes of a row exchange halves: 16 bytes each
                    auto rx = __builtin_amdgcn_permlane32_swap(w[4 * gp], w[4 * gp + 2], false, false);
                    auto ry = __builtin_amdgcn_permlane32_swap(w[4 * gp + 1], w[4 * gp + 3], false, false);
                    u32x4 o = {(uint32_t)rx[0], (uint32_t)ry[0], (uint32_t)rx[1], (uint32_t)ry[1]};
                    if (row < p.M) *(u32x4*)(p.out + row * p.out_stride + cbase + 16 * gp + 8 * hf) = o;
                }
            }
        }
    } else {
#pragma unroll
        for (int cb = 0; cb < 4; ++cb)
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float a4[4] = {acc[cb][tb][4 * g], acc[cb][tb][4 * g + 1], acc[cb][tb][4 * g + 2], acc[cb][tb][4 * g + 3]};
                    l8_finish4<E, EPI>(p, row0 + 32 * tb, n0 + wn * 128 + 32 * cb + 8 * g + 4 * hf, a4);
                }
    }
}

template <class E, int EPI, int TB>
int launch_tile(const L8Args& a0, hipStream_t st) {
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
    hipLaunchKernelGGL((l8_tile_kernel<E, EPI, TB>), dim3((unsigned)((a.tm * a.tn + 7) / 8 * 8)), dim3(256), kLdsBytes, st, a);
    return launched8("sfm_linear8");
}

template <class E, int EPI>
int launch_epi(const L8Args& a, hipStream_t st) {
    if (a.M <= 16) return launch_direct<E, EPI, 1, 1, 8>(a, st);
    if (a.M >= 1024 && a.N >= 256) return launch_tile<E, EPI, 4>(a, st);
    if (a.M >= 256 && a.N >= 256) return launch_tile<E, EPI, 2>(a, st);
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
