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

#include "rows8.hpp"

namespace sfm {
namespace {

constexpr int kWT = 128;                    // tile: 128 channels n x 128 channels k
constexpr int kWR = 64;                     // rows per step
constexpr int kWPitch = kWT * 2;            // LDS bytes per row of a staged tile
constexpr int kWTile = kWR * kWPitch;       // one operand of a step

struct WgradArgs {
    const void* dy;          // [M, N] rows dy_stride apart
    const uint8_t* x;        // [M][kp]
    const uint8_t* xscale;
    void* dw;                // [N, K]
    float* part;             // [splits][N][K] or null
    int64_t M, groups, kp, dy_stride;
    int N, K, tn, tk, splits;
    bool dyvec, dwvec;
};

typedef short w8_s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 w8_read_tr(const char* lds, uint32_t off) {
    w8_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((w8_s16x4 __attribute__((address_space(3)))*)(lds + off));
    return __builtin_bit_cast(u32x2, v);
}
// 16-byte piece c of row r sits at piece c ^ swz(r): the four rows of a transposing read hit different banks
__device__ __forceinline__ int w8_swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

template <class E>
__device__ __forceinline__ u32x4 w8_values8(uint32_t lo, uint32_t hi, float s) {
    float v[8];
    unpack_e4m3(lo, v);
    unpack_e4m3(hi, v + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] *= s;
        if (std::is_same<E, F16>::value) v[i] = v[i] != v[i] ? v[i] : fminf(fmaxf(v[i], -65504.f), 65504.f);
    }
    return u32x4{pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]), pack2<E>(v[4], v[5]), pack2<E>(v[6], v[7])};
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
    float xs[2];
    auto fetch = [&](int64_t st) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = st * kWR + dr + 16 * i;
            u32x4 z = {0u, 0u, 0u, 0u};
            if (r < p.M) {
                const uint16_t* s = (const uint16_t*)p.dy + r * p.dy_stride + n0 + dc;
                if (p.dyvec && n0 + dc + 8 <= p.N) {
                    z = *(const u32x4*)s;
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
            xs[i] = 0.f;
            if (r < p.M) {
                xv[i] = *(const u32x4*)(p.x + r * p.kp + kb * kBlock8 + xc);
                xs[i] = two_to((int)p.xscale[scale_at8(r, kb, p.groups)] - 127);
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
            *(u32x4*)(d + (((xc >> 3) ^ w8_swz(r)) << 4)) = w8_values8<E>(xv[i].x, xv[i].y, xs[i]);
            *(u32x4*)(d + (((xc >> 3) + 1 ^ w8_swz(r)) << 4)) = w8_values8<E>(xv[i].z, xv[i].w, xs[i]);
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
                    if (p.dwvec && k + 4 <= p.K) {
                        u32x2 w = {pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3])};
                        *(u32x2*)o = w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (k + e < p.K) o[e] = E::from_float(v[e]);
                    }
                }
            }
        }
}

int wgrad_splits(int64_t M, int N, int K) {
    const int64_t tiles = (int64_t)blocks8(N) * blocks8(K), steps = (M + kWR - 1) / kWR, cus = cu_count();
    int64_t s = 1;
    while (s < 16 && tiles * s * 2 <= 2 * cus && steps >= s * 2 * 4) s *= 2;      // at least four steps a part
    return (int)s;
}

}  // namespace

size_t wgrad8_workspace_bytes(int64_t M, int N, int K, bool bias) {
    const int s = wgrad_splits(M, N, K);
    size_t b = s > 1 ? (size_t)s * N * K * sizeof(float) : 0;
    b = (b + 255) / 256 * 256;
    return b + (bias ? (size_t)((M + kBlock8 - 1) / kBlock8) * N * sizeof(float) : 0);
}

int launch_wgrad8(int dtype, int64_t M, int N, int K, const void* dy, int64_t dy_stride, const void* x8, const void* xscale, void* dw,
                  void* dbias, const float* colsum, void* workspace, hipStream_t st) {
    const int64_t groups = (M + kBlock8 - 1) / kBlock8;
    const int splits = wgrad_splits(M, N, K);
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
        a.tn = blocks8(N);
        a.tk = blocks8(K);
        a.splits = splits;
        a.dyvec = ((uintptr_t)dy & 15) == 0 && dy_stride % 8 == 0;
        a.dwvec = ((uintptr_t)dw & 15) == 0 && K % 4 == 0;
        const dim3 grid((unsigned)(a.tn * a.tk * splits));
        if (dtype == SFM_BF16) hipLaunchKernelGGL((wgrad8_kernel<BF16>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((wgrad8_kernel<F16>), grid, dim3(256), 0, st, a);
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
    return launch_sum_parts(dtype, groups, N, 1, colsum, dbias, nullptr, st);
}

}  // namespace sfm
