// Gradient of the weight of a linear layer from the activations its forward kept in 8-bit blocks (rows8.hpp):
//
//   dw[n, k] = sum_m dy[m, n] x8[m, k] 2^sx[m, k / 128]
//
// The sum runs over the rows, along which the scales of x8 change from value to value, so that no scaled matrix instruction
// can take them: a row's bytes become 16-bit values on their way into LDS (exact in bf16: an e4m3 value times a power of
// two has four bits) and the product runs at the 16-bit rate, with dy as it is, unrounded.  The activations' traffic is half
// of what 16-bit ones would need.  No counterpart in the reference.
//
// Both operands lie with the rows (the contraction) outermost: the transposing LDS reads turn 4 rows x 16 columns per 16
// lanes, so that a lane holds 8 rows of one column, in the same row order for both operands.
//
// Calls with few output tiles split the rows; the parts' fp32 sums meet in a fixed order in a second kernel.

#include <type_traits>

#include "rows8.hpp"

namespace sfm {
namespace {

constexpr int kWT = 128;                    // small tiles: 128 channels n x 128 channels k
constexpr int kWR = 64;                     // rows per step
constexpr int kWPitch = kWT * 2;            // LDS bytes per row of a staged tile
constexpr int kWTile = kWR * kWPitch;       // one operand of a step
constexpr int kBT = 256, kBR = 32;          // large tiles: 256 x 256 channels, 32 rows per step
constexpr int kBPitch = kBT * 2, kBTile = kBR * kBPitch;

struct WgradArgs {
    const void* dy;          // [M, N] rows dy_stride apart
    const uint8_t* x;        // [M][kp]
    const uint8_t* xscale;
    void* dw;                // [N, K]
    float* part;             // [splits][N][K] or null
    int64_t M, groups, kp, dy_stride;
    int N, K, tn, tk, splits;
};

typedef short w8_s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 w8_read_tr(const char* lds, uint32_t off) {
    w8_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((w8_s16x4 __attribute__((address_space(3)))*)(lds + off));
    return __builtin_bit_cast(u32x2, v);
}
// 16-byte piece c of row r sits at piece c ^ swz(r): the four rows of a transposing read hit different banks
__device__ __forceinline__ int w8_swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

// eight e4m3 values times 2^(s8 - 127) in the 16-bit type, packed; in fp16 what lies past its range becomes the largest value
template <class E>
__device__ __forceinline__ u32x4 w8_pack8(uint32_t lo, uint32_t hi, uint32_t s8) {
    const float s = two_to((int)s8 - 127);
    if constexpr (std::is_same<E, BF16>::value) {
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true))};
    } else {
        float v[8];
        unpack_e4m3(lo, v);
        unpack_e4m3(hi, v + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] *= s;
            v[i] = v[i] != v[i] ? v[i] : fminf(fmaxf(v[i], -65504.f), 65504.f);
        }
        return u32x4{pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]), pack2<E>(v[4], v[5]), pack2<E>(v[6], v[7])};
    }
}

template <class E>
__global__ __launch_bounds__(256) void wgrad8_kernel(WgradArgs p) {
    __shared__ __attribute__((aligned(256))) char lds[2 * kWTile];       // dy tile, x tile
    const int tid = threadIdx.x, lane = tid & 63, m32 = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = (wave & 1) * 64, wk = (wave >> 1) * 64;
    const int tile = blockIdx.x % (p.tn * p.tk), split = blockIdx.x / (p.tn * p.tk);
    const int n0 = tile % p.tn * kWT, kb = tile / p.tn;
    const int64_t steps = (p.M + kWR - 1) / kWR;
    const int64_t s0 = steps * split / p.splits, s1 = steps * (split + 1) / p.splits;

    // a thread stages rows r8 + 16 i (i < 4) of dy, 8 channels, and rows r4 + 32 i (i < 2) of x, 16 channels
    const int dc = (tid & 15) * 8, dr = tid >> 4;
    const int xc = (tid & 7) * 16, xr = tid >> 3;
    u32x4 dv[4], xv[2];
    uint32_t xs[2];
    auto fetch = [&](int64_t st) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = st * kWR + dr + 16 * i;
            u32x4 z = {0u, 0u, 0u, 0u};
            if (r < p.M) {
                const uint16_t* s = (const uint16_t*)p.dy + r * p.dy_stride + n0 + dc;
                if (n0 + dc + 8 <= p.N) {
                    z = *(const u32x4_any*)s;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (n0 + dc + e < p.N) z[e >> 1] |= (uint32_t)s[e] << (16 * (e & 1));
                }
            }
            dv[i] = z;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t r = st * kWR + xr + 32 * i;
            xv[i] = u32x4{0u, 0u, 0u, 0u};
            xs[i] = 127;
            if (r < p.M) {
                xv[i] = *(const u32x4*)(p.x + r * p.kp + kb * kBlock8 + xc);
                xs[i] = p.xscale[scale_at8(r, kb, p.groups)];
            }
        }
    };
    auto stage = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = dr + 16 * i;
            *(u32x4*)(lds + r * kWPitch + (((dc >> 3) ^ w8_swz(r)) << 4)) = dv[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = xr + 32 * i;
            char* d = lds + kWTile + r * kWPitch;
            *(u32x4*)(d + (((xc >> 3) ^ w8_swz(r)) << 4)) = w8_pack8<E>(xv[i].x, xv[i].y, xs[i]);
            *(u32x4*)(d + (((xc >> 3) + 1 ^ w8_swz(r)) << 4)) = w8_pack8<E>(xv[i].z, xv[i].w, xs[i]);
        }
    };
    // operand [channel 32 b + lane % 32, 16 rows] of a staged tile: rows 4 hf + 0..3 and 8 + 4 hf + 0..3 of the 16
    const int s16 = lane & 15, g16 = lane >> 4;
    auto operand = [&](uint32_t base, int c0, int ks) {
        u32x2 h[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = 16 * ks + 8 * half + 4 * hf + (s16 >> 2);
            const int c = (c0 >> 3) + 2 * (g16 & 1) + ((s16 & 3) >> 1);
            h[half] = w8_read_tr(lds, base + r * kWPitch + ((c ^ w8_swz(r)) << 4) + (s16 & 1) * 8);
        }
        return u32x4{h[0].x, h[0].y, h[1].x, h[1].y};
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
    if (s0 < s1) fetch(s0);
    for (int64_t st = s0; st < s1; ++st) {
        __syncthreads();
        stage();
        __syncthreads();
        if (st + 1 < s1) fetch(st + 1);
#pragma unroll
        for (int ks = 0; ks < kWR / 16; ++ks) {
            u32x4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = operand(kWTile, wk + 32 * i, ks);      // A: rows of the result = channels k, four neighbours a lane
                b[i] = operand(0, wn + 32 * i, ks);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = E::mfma32(a[i], b[j], acc[i][j]);
        }
    }
    // lane: channel n = .. + m32, channels k = 8 g + 4 hf + (0..3) of a 32-block
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = n0 + wn + 32 * j + m32;
            if (n >= p.N) continue;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int k = kb * kBlock8 + wk + 32 * i + 8 * g + 4 * hf;
                const float v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                if (p.part != nullptr) {
                    float* o = p.part + ((int64_t)split * p.N + n) * p.K + k;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k + e < p.K) o[e] = v[e];
                } else {
                    uint16_t* o = (uint16_t*)p.dw + (int64_t)n * p.K + k;
                    if (k + 4 <= p.K) {
                        u32x2 w = {pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3])};
                        *(u32x2_any*)o = w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (k + e < p.K) o[e] = E::from_float(v[e]);
                    }
                }
            }
        }
}

// Large tiles: 256 x 256 channels, a wave 128 x 128 (16 matrix instructions 32x32x16 per 16 rows, 256 accumulator registers, one wave
// per SIMD), 32 rows per step, two LDS buffers.  A thread stages one row: four 16-byte pieces of dy and two of x8, whose 16 values
// become 32 bytes.  The rows of a step are requested five steps ahead into registers (four sets in turn), written to LDS
// a step ahead, behind the matrix instructions of the step's first 16 rows; the operands of the next 16 rows are read behind those
// of the 16 before.  EDGE: a row of dy ends inside a piece of 8 channels of this tile.
//
// Bound by the matrix pipe: 4680 x 1536 x 8960 has 129 GFLOP, 80 us at the 1.6 PFLOP/s of a large bf16 product here, and takes 133 us
// (0.97 PFLOP/s; a library product of 16-bit operands of this shape 158 us); its 210 tiles leave 46 of 256 compute units idle, which
// alone makes 80 us 98.  Requests three steps ahead: 150 us.  It does not fit its registers: with both forms of the tile in one kernel
// the compiler spills 50 vector and some 250 scalar registers (196 bytes of scratch a lane).
template <class E, bool EDGE>
__device__ __forceinline__ void wgrad8_tile(const WgradArgs& p, int n0, int kb, int64_t s0, int64_t s1, int split) {
    extern __shared__ __attribute__((aligned(256))) char w8_lds[];      // [buffer][dy tile | x tile]
    const int tid = threadIdx.x, lane = tid & 63, m32 = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = (wave & 1) * 128, wk = (wave >> 1) * 128;
    const int r = tid >> 3, c8 = tid & 7;                               // this thread's row of a step, its pieces c8 + 8 j
    const int kb1 = (int64_t)(kb + 2) * kBlock8 <= p.kp ? 1 : 0;        // a tile may have one block of channels k only
    struct Raw {
        u32x4 d[4], x[2];
        uint8_t s[2];                                                   // the row's two scales
    };
    // Pieces of dy that lie behind the row's end take what is before it: no store uses their products.  One that the row ends in
    // (EDGE) is loaded from the row's last 8 channels and shifted down by those that are before it.
    int off[4], down[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = n0 + c8 * 8 + 64 * j;
        off[j] = min(c, p.N - 8);
        down[j] = EDGE ? min(c - off[j], 7) : 0;
    }
    struct Rows {                                                       // where a step's row of this thread lies
        const uint8_t *s, *x;
        const uint16_t* d;
    };
    auto find = [&](int64_t st) {
        const int64_t row = min(st * kBR + r, p.M - 1);
        return Rows{p.xscale + scale_at8(row, kb, p.groups), p.x + row * p.kp + (int64_t)kb * kBlock8 + c8 * 16,
                    (const uint16_t*)p.dy + row * p.dy_stride};
    };
    auto load = [&](Raw& w, const Rows& at, int i) {                    // request i of 8
        if (i < 2) w.s[i] = at.s[i * kb1 * p.groups * kBlock8];
        else if (i < 4) w.x[i - 2] = *(const u32x4*)(at.x + (i - 2) * kb1 * kBlock8);
        else w.d[i - 4] = *(const u32x4_any*)(at.d + off[i - 4]);
    };
    auto fetch = [&](Raw& w, int64_t st) {
        const Rows at = find(st);
#pragma unroll
        for (int i = 0; i < 8; ++i) load(w, at, i);
    };
    auto shifted = [&](u32x4 v, int by) {
        if (!EDGE) return v;
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                                   // word i of v >> 16 by
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                lo = i + (by >> 1) == k ? v[k] : lo;
                hi = i + (by >> 1) + 1 == k ? v[k] : hi;
            }
            o[i] = by & 1 ? (lo >> 16) | (hi << 16) : lo;
        }
        return o;
    };
    // Piece c (16 bytes) of row r sits at piece c ^ swz(r), which turns the low four bits of c: what lies above them and the rows'
    // sixteens are offsets in the instructions, and so is the buffer.
    const uint32_t wrow = (uint32_t)(r * kBPitch);
    const uint32_t dp[2] = {wrow + (uint32_t)((c8 ^ w8_swz(r)) << 4), wrow + (uint32_t)(((c8 + 8) ^ w8_swz(r)) << 4)};
    const uint32_t xp[2] = {wrow + (uint32_t)(((2 * c8) ^ w8_swz(r)) << 4), wrow + (uint32_t)(((2 * c8 + 1) ^ w8_swz(r)) << 4)};
    auto put_dy = [&](const Raw& w, int buf, int j, bool live) {
        *(u32x4*)(w8_lds + dp[j & 1] + (buf * 2 * kBTile + (j >> 1) * 256)) = live ? shifted(w.d[j], down[j]) : u32x4{0u, 0u, 0u, 0u};
    };
    auto put_x = [&](const Raw& w, int buf, int i, bool live) {         // half i & 1 of piece i >> 1
        const int j = i >> 1;
        const u32x4 v = w8_pack8<E>(i & 1 ? w.x[j].z : w.x[j].x, i & 1 ? w.x[j].w : w.x[j].y, w.s[j]);
        *(u32x4*)(w8_lds + xp[i & 1] + (buf * 2 * kBTile + kBTile + j * 256)) = live ? v : u32x4{0u, 0u, 0u, 0u};
    };
    // operand [channel 32 b + lane % 32, 16 rows] of a staged tile: rows 4 hf + 0..3 and 8 + 4 hf + 0..3 of the 16
    uint32_t at[4][2];
    {
        const int s16 = lane & 15, g16 = lane >> 4;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int rr = 8 * half + 4 * hf + (s16 >> 2), c = 4 * b + 2 * (g16 & 1) + ((s16 & 3) >> 1);
                at[b][half] = (uint32_t)(rr * kBPitch + ((c ^ w8_swz(rr)) << 4) + (s16 & 1) * 8);
            }
    }
    const char *ldsk = w8_lds + wk * 2, *ldsn = w8_lds + wn * 2;
    auto operand_at = [&](int buf, int ks, int i) {                     // 0..3: channels k (A), 4..7: channels n (B)
        const char* base = (i < 4 ? ldsk : ldsn) + (buf * 2 * kBTile + (i < 4 ? kBTile : 0) + ks * 16 * kBPitch);
        const u32x2 lo = w8_read_tr(base, at[i & 3][0]), hi = w8_read_tr(base, at[i & 3][1]);
        return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    f32x16 acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
    Raw raw[4];
    u32x4 f0[8], f1[8];
    auto last = [&](int64_t st) { return min(st, s1 - 1); };
    auto live = [&](int64_t st) { return st < s1 && st * kBR + r < p.M; };
#pragma unroll
    for (int i = 0; i < 4; ++i) fetch(raw[i], last(s0 + i));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        put_dy(raw[0], 0, j, live(s0));
        put_x(raw[0], 0, j, live(s0));
    }
    fetch(raw[0], last(s0 + 4));
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) f0[i] = operand_at(0, 0, i);
    // Step st from buffer `buf`; the next one's rows are in `w`, which then takes those of step st + 5.  WHOLE: all rows of the next
    // step exist.  Behind the 16 matrix instructions of its first half: the reads for the second, the next step's rows into LDS, the
    // first requests; of its second: the barrier, the reads for the next step (done some instructions before they are waited
    // for), the other requests.
    auto step = [&](int64_t st, Raw& w, int buf, auto whole_c) {
        const bool ok = decltype(whole_c)::value || live(st + 1);
        Rows rows;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            acc[i >> 2][i & 3] = E::mfma32(f0[i >> 2], f0[4 + (i & 3)], acc[i >> 2][i & 3]);
            __builtin_amdgcn_sched_barrier(0);
            if (i < 4) {
                f1[2 * i] = operand_at(buf, 1, 2 * i);
                f1[2 * i + 1] = operand_at(buf, 1, 2 * i + 1);
            } else if (i < 8) {
                put_dy(w, buf ^ 1, i - 4, ok);
            } else if (i < 12) {
                put_x(w, buf ^ 1, i - 8, ok);
            } else if (i == 12) {
                rows = find(last(st + 5));
            } else {
                load(w, rows, i - 13);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            acc[i >> 2][i & 3] = E::mfma32(f1[i >> 2], f1[4 + (i & 3)], acc[i >> 2][i & 3]);
            __builtin_amdgcn_sched_barrier(0);
            if (i == 1) lds_barrier();
            if (i > 1 && i < 10) f0[i - 2] = operand_at(buf ^ 1, 0, i - 2);
            if (i > 9 && i < 15) load(w, rows, i - 7);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int64_t st = s0;
    for (; st + 4 < s1 && (st + 5) * kBR <= p.M; st += 4) {
        step(st, raw[1], 0, std::true_type{});
        step(st + 1, raw[2], 1, std::true_type{});
        step(st + 2, raw[3], 0, std::true_type{});
        step(st + 3, raw[0], 1, std::true_type{});
    }
    // rows behind the last step are zeros (`live`): up to three steps of nothing keep the loop whole
    for (; st < s1; st += 4) {
        step(st, raw[1], 0, std::false_type{});
        step(st + 1, raw[2], 1, std::false_type{});
        step(st + 2, raw[3], 0, std::false_type{});
        step(st + 3, raw[0], 1, std::false_type{});
    }
    // lane: channel n = .. + m32, channels k = 8 g + 4 hf + (0..3) of a 32-block
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            int own = wn + 32 * j + m32;
            asm volatile("" : "+v"(own));                               // addresses block by block: for all they do not fit
            const int n = n0 + own, k0 = kb * kBlock8 + wk + 32 * i;
            if (p.part != nullptr) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int k = k0 + 8 * g + 4 * hf;
                    float* o = p.part + ((int64_t)split * p.N + n) * p.K + k;
                    const f32x4 v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                    if (n < p.N && k + 4 <= p.K) {
                        *(f32x4_any*)o = v;
                    } else if (n < p.N) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (k + e < p.K) o[e] = v[e];
                    }
                }
            } else {
#pragma unroll
                for (int gp = 0; gp < 2; ++gp) {                        // the two lanes of a channel n exchange halves: 16 bytes each
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = pack2<E>(acc[i][j][8 * gp + 2 * e], acc[i][j][8 * gp + 2 * e + 1]);
                    auto rx = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
                    auto ry = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                    const u32x4 o = {(uint32_t)rx[0], (uint32_t)ry[0], (uint32_t)rx[1], (uint32_t)ry[1]};
                    const int k = k0 + 16 * gp + 8 * hf;
                    uint16_t* d = (uint16_t*)p.dw + (int64_t)n * p.K + k;
                    if (n < p.N && k + 8 <= p.K) {
                        *(u32x4_any*)d = o;
                    } else if (n < p.N) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (k + e < p.K) d[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
                    }
                }
            }
        }
}

template <class E>
__global__ __launch_bounds__(256) void wgrad8_big_kernel(WgradArgs p) {
    // neighbouring workgroups of an XCD take the tiles of a few columns n: they share dy's and x8's rows in its L2
    const int ntiles = p.tn * p.tk * p.splits, per = (ntiles + 7) / 8;
    const int v = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (v >= ntiles) return;
    const int split = __builtin_amdgcn_readfirstlane(v / (p.tn * p.tk)), tile = v - split * p.tn * p.tk;
    const int tn = __builtin_amdgcn_readfirstlane(tile / p.tk), kb = (tile - tn * p.tk) * 2, n0 = tn * kBT;
    const int64_t steps = (p.M + kBR - 1) / kBR;
    const int64_t s0 = steps * split / p.splits, s1 = steps * (split + 1) / p.splits;
    if (n0 + kBT <= p.N || p.N % 8 == 0) wgrad8_tile<E, false>(p, n0, kb, s0, s1, split);
    else wgrad8_tile<E, true>(p, n0, kb, s0, s1, split);
}

// Tiles and parts of the rows.  A round of large tiles takes 0.93 us a step of 32 rows, one of small tiles 1.05 a step of 64 (1.6 with
// two on a compute unit), and parts cost what their fp32 sums take to write and read again.
struct WgradPlan {
    bool big;
    int splits;
};
WgradPlan wgrad_plan(int64_t M, int N, int K) {
    const double cus = cu_count();
    WgradPlan best = {false, 1};
    double least = 1e30;
    for (int big = 0; big < (N >= 8 ? 2 : 1); ++big) {
        const double tiles = big ? (double)((N + 255) / 256) * ((K + 255) / 256) : (double)blocks8(N) * blocks8(K);
        const int64_t steps = big ? (M + kBR - 1) / kBR : (M + kWR - 1) / kWR;
        for (int s = 1; s <= 16 && (s == 1 || steps >= 4 * s); ++s) {
            const double wgs = tiles * s, per_cu = big || wgs <= cus ? 1.0 : 2.0;
            const double rounds = wgs <= cus * per_cu ? 1.0 : wgs / (cus * per_cu) + 0.4;
            const double t = 4.0 + rounds * ((double)((steps + s - 1) / s) * (big ? 0.93 : per_cu > 1.0 ? 1.6 : 1.05) + (big ? 5.0 : 3.0)) +
                             (s > 1 ? 3.0 + 8.0 * s * N * K / 4.5e6 : 0.0);
            if (t < least) {
                least = t;
                best = {big != 0, s};
            }
        }
    }
    return best;
}

}  // namespace

int wgrad8_tile_size(int64_t M, int N, int K, int* parts) {
    const WgradPlan plan = wgrad_plan(M, N, K);
    *parts = plan.splits;
    return plan.big ? kBT : kWT;
}

size_t wgrad8_workspace_bytes(int64_t M, int N, int K, bool bias) {
    const int s = wgrad_plan(M, N, K).splits;
    size_t b = s > 1 ? (size_t)s * N * K * sizeof(float) : 0;
    b = (b + 255) / 256 * 256;
    return b + (bias ? (size_t)((M + kColRows8 - 1) / kColRows8) * N * sizeof(float) : 0);
}

int launch_wgrad8(int dtype, int64_t M, int N, int K, const void* dy, int64_t dy_stride, const void* x8, const void* xscale, void* dw,
                  void* dbias, const float* colsum, void* workspace, hipStream_t st) {
    const int64_t groups = (M + kBlock8 - 1) / kBlock8;
    const WgradPlan plan = wgrad_plan(M, N, K);
    const int splits = plan.splits;
    if (dw != nullptr) {
        WgradArgs a;
        a.dy = dy;
        a.x = (const uint8_t*)x8;
        a.xscale = (const uint8_t*)xscale;
        a.dw = dw;
        a.part = splits > 1 ? (float*)workspace : nullptr;
        a.M = M;
        a.groups = groups;
        a.kp = pad8(K);
        a.dy_stride = dy_stride;
        a.N = N;
        a.K = K;
        a.tn = plan.big ? (N + kBT - 1) / kBT : blocks8(N);
        a.tk = plan.big ? (K + kBT - 1) / kBT : blocks8(K);
        a.splits = splits;
        const unsigned wgs = (unsigned)(a.tn * a.tk * splits);
        if (plan.big) {
            static bool configured = false;              // the attribute belongs to the function; racing callers set the same value
            if (!configured) {
                hipError_t e = hipFuncSetAttribute((const void*)wgrad8_big_kernel<BF16>, hipFuncAttributeMaxDynamicSharedMemorySize, 4 * kBTile);
                if (e == hipSuccess) e = hipFuncSetAttribute((const void*)wgrad8_big_kernel<F16>, hipFuncAttributeMaxDynamicSharedMemorySize, 4 * kBTile);
                if (e != hipSuccess) {
                    set_error("sfm_linear8_wgrad: hipFuncSetAttribute failed: %s", hipGetErrorString(e));
                    return SFM_ERR_HIP;
                }
                configured = true;
            }
            const dim3 grid((wgs + 7) / 8 * 8);
            if (dtype == SFM_BF16) hipLaunchKernelGGL((wgrad8_big_kernel<BF16>), grid, dim3(256), 4 * kBTile, st, a);
            else hipLaunchKernelGGL((wgrad8_big_kernel<F16>), grid, dim3(256), 4 * kBTile, st, a);
        } else {
            if (dtype == SFM_BF16) hipLaunchKernelGGL((wgrad8_kernel<BF16>), dim3(wgs), dim3(256), 0, st, a);
            else hipLaunchKernelGGL((wgrad8_kernel<F16>), dim3(wgs), dim3(256), 0, st, a);
        }
        int rc = launched8("sfm_linear8_wgrad");
        if (rc) return rc;
        if (splits > 1 && (rc = launch_sum_parts(dtype, splits, (int64_t)N * K, 1, a.part, dw, nullptr, st))) return rc;
    }
    if (dbias == nullptr) return SFM_OK;
    if (colsum == nullptr) {
        float* cs = (float*)((char*)workspace + (wgrad8_workspace_bytes(M, N, K, false)));
        int rc = launch_quantize8(dtype, M, N, dy, dy_stride, nullptr, nullptr, nullptr, 0, cs, st);
        if (rc) return rc;
        colsum = cs;
    }
    return launch_sum_parts(dtype, (M + kColRows8 - 1) / kColRows8, N, 1, colsum, dbias, nullptr, st);
}

}  // namespace sfm
