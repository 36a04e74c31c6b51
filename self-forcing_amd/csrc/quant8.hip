// Rows and weights in 8-bit blocks (rows8.hpp says what a block is): quantisation, the values back, weights laid out for
// both products that read them, and GELU with its input kept in 8 bits for the backward.  No counterpart in the reference,
// whose linear layers and activations are 16 bits throughout (wan/modules/model.py:592-650).
//
// All of them read and write every element once and are bound by memory.

#include "rows8.hpp"

namespace sfm {
namespace {

// One workgroup: 32 rows of one block column.  A thread holds 8 neighbouring elements of the rows r0 and r0 + 16; the 16 lanes of a row
// find the block's maximum by rotations.  Small workgroups keep more of them on their way: with 128 rows, whose scales would be
// whole words, 4680 x 5120 takes 22 us (16; 4.5 TB/s) and GELU's forward at 4680 x 8960 48 (39; 5.4 TB/s).
//   GELU: y = gelu_tanh(x) is stored besides.   data NULL: nothing is quantised.
//   colsum: float [ceil(rows / 32)][K], the sums over the workgroup's rows (a bias gradient's first half).
template <typename T, bool GELU>
__global__ __launch_bounds__(256) void quantize8_kernel(const void* x, int64_t xs, int64_t rows, int K, uint8_t* data, uint8_t* scale,
                                                        void* y, int64_t ys, float* colsum) {
    constexpr int NR = 2;
    __shared__ uint8_t sc[kColRows8];
    __shared__ __attribute__((aligned(16))) float cs[16][kBlock8];
    const int64_t groups = (rows + kBlock8 - 1) / kBlock8;
    const int kb = blockIdx.y, l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int c = kb * kBlock8 + l16 * 8;
    const int64_t kp = pad8(K), row0 = (int64_t)blockIdx.x * kColRows8;
    float v[NR][8];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int64_t r = row0 + r0 + 16 * i;
        if (r < rows) {
            load_part8<T>(x, r * xs, c, K, v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        }
    }
    if (colsum != nullptr) {
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[e] = 0.f;
#pragma unroll
            for (int i = 0; i < NR; ++i) s[e] += v[i][e];
        }
        V8<float>::store(&cs[r0][0], l16 * 8, s);
    }
    if (data != nullptr) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int64_t r = row0 + r0 + 16 * i;
            u32x2 q;
            const int s = quantize_block8(v[i], &q);
            if (r < rows) *(u32x2*)(data + r * kp + c) = q;
            if (l16 == 0) sc[r0 + 16 * i] = (uint8_t)(s + 127);
        }
    }
    if (GELU) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int64_t r = row0 + r0 + 16 * i;
            if (r < rows) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= gelu_gate<kWide<T>>(v[i][e]);
                store_part8<T>(y, r * ys, c, K, v[i]);
            }
        }
    }
    __syncthreads();
    if (data != nullptr && threadIdx.x < kColRows8) scale[scale_at8(row0 + threadIdx.x, kb, groups)] = sc[threadIdx.x];
    if (colsum != nullptr && threadIdx.x < kBlock8 && kb * kBlock8 + (int)threadIdx.x < K) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += cs[i][threadIdx.x];
        colsum[(int64_t)blockIdx.x * K + kb * kBlock8 + threadIdx.x] = s;
    }
}

// the values of 8 elements of a row's blocks
__device__ __forceinline__ void values8(const uint8_t* data, const uint8_t* scale, int64_t r, int64_t kp, int64_t groups, int c, float* v) {
    const u32x2 q = *(const u32x2*)(data + r * kp + c);
    const float s = two_to((int)scale[scale_at8(r, c >> 7, groups)] - 127);
    unpack_e4m3(q.x, v);
    unpack_e4m3(q.y, v + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= s;
}

// in fp16 a value past its range (65536 for a 65504 that was rounded up) becomes the largest one
template <typename T>
__global__ __launch_bounds__(256) void dequantize8_kernel(const uint8_t* data, const uint8_t* scale, int64_t rows, int K, void* y,
                                                          int64_t ys) {
    const int64_t kp = pad8(K), groups = (rows + kBlock8 - 1) / kBlock8;
    const int chunks = (K + 7) / 8;
    const int64_t n = rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / chunks;
        const int c = (int)(i - r * chunks) * 8;
        float v[8];
        values8(data, scale, r, kp, groups, c, v);
        if (std::is_same<T, F16>::value) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] != v[e] ? v[e] : fminf(fmaxf(v[e], -65504.f), 65504.f);
        }
        store_part8<T>(y, r * ys, c, K, v);
    }
}

// dx = dy gelu'(x), x from its 8-bit blocks (KEPT) or as it was.  Bound by memory: 4680 x 8960 from blocks 39 us, 5.4 TB/s.
template <typename T, bool KEPT>
__global__ __launch_bounds__(256) void gelu_bwd_kernel(const void* x, int64_t xs, const uint8_t* data, const uint8_t* scale,
                                                       int64_t rows, int K, const void* dy, int64_t dys, void* dx,
                                                       int64_t dxs) {
    const int64_t kp = pad8(K), groups = (rows + kBlock8 - 1) / kBlock8;
    const int chunks = (K + 7) / 8;
    const int64_t n = rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / chunks;
        const int c = (int)(i - r * chunks) * 8;
        float v[8], g[8];
        if (KEPT) values8(data, scale, r, kp, groups, c, v);
        else load_part8<T>(x, r * xs, c, K, v);
        load_part8<T>(dy, r * dys, c, K, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= gelu_slope<kWide<T>>(v[e]);
        store_part8<T>(dx, r * dxs, c, K, g);
    }
}

// One workgroup: a 128 x 128 block of a weight [N, K], one scale.  The block goes out twice, as it lies and transposed (through
// LDS, a thread turning 4 x 4 bytes at a time), so that the product with the gradient of the output reads it along N.  13824 x 5120:
// 58-61 us, 4.8 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void pack8_kernel(const void* w, int64_t ws, int N, int K, uint8_t* data, uint8_t* scale,
                                                    uint8_t* data_t, uint8_t* scale_t, int pitch, int pitch_t) {
    __shared__ float top[4];
    __shared__ __attribute__((aligned(16))) uint8_t tile[kBlock8][kBlock8 + 4];
    const int kb = blockIdx.x, nb = blockIdx.y, l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int c = kb * kBlock8 + l16 * 8;
    const int64_t kp = pad8(K), np = pad8(N);
    float v[8][8], a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = (int64_t)nb * kBlock8 + r0 + 16 * i;
        if (r < N) {
            load_part8<T>(w, r * ws, c, K, v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        }
        a = fmaxf(a, mag_max<8>(v[i]));
    }
    auto block_max = [&](float m) {
        m = max16(m);
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
        __syncthreads();
        return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    };
    a = block_max(a);
    if (a >= kTop8) {                                 // the same for the whole workgroup
        a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, mag_max_finite<8>(v[i]));
        a = block_max(a);
    }
    const int s = block_exp8(a);
    const float inv = two_to(-s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int rr = r0 + 16 * i;
        const int64_t r = (int64_t)nb * kBlock8 + rr;
        u32x2 q;
        q.x = pack_e4m3(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        q.y = pack_e4m3(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
        if (r < N) *(u32x2*)(data + r * kp + c) = q;
        *(uint32_t*)&tile[rr][l16 * 8] = q.x;
        *(uint32_t*)&tile[rr][l16 * 8 + 4] = q.y;
    }
    if (threadIdx.x == 0) {                          // the last block of a row of scales fills the rest of its last word
        uint8_t* o = scale + (int64_t)nb * pitch;
        o[kb] = (uint8_t)(s + 127);
        for (int i = kb + 1; kb + 1 == (int)gridDim.x && i < pitch; ++i) o[i] = 0;
        if (data_t != nullptr) {
            o = scale_t + (int64_t)kb * pitch_t;
            o[nb] = (uint8_t)(s + 127);
            for (int i = nb + 1; nb + 1 == (int)gridDim.y && i < pitch_t; ++i) o[i] = 0;
        }
    }
    if (data_t == nullptr) return;
    __syncthreads();
    // 32 x 32 pieces of 4 rows x 4 columns, 4 a thread: lanes walk the rows, so that a column's bytes leave 4 a lane in a row
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int id = threadIdx.x + 256 * p, r4 = (id & 31) * 4, c4 = (id >> 5) * 4;
        uint32_t w4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w4[i] = *(const uint32_t*)&tile[r4 + i][c4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t o = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) o |= ((w4[i] >> (8 * j)) & 0xffu) << (8 * i);
            if (kb * kBlock8 + c4 + j < K) *(uint32_t*)(data_t + (int64_t)(kb * kBlock8 + c4 + j) * np + nb * kBlock8 + r4) = o;
        }
    }
}

template <typename T>
int quantize_t(int64_t rows, int K, const void* x, int64_t xs, void* data, void* scale, void* y, int64_t ys, float* colsum, hipStream_t st) {
    const dim3 grid((unsigned)((rows + kColRows8 - 1) / kColRows8), (unsigned)blocks8(K));
    if (y != nullptr)
        hipLaunchKernelGGL((quantize8_kernel<T, true>), grid, dim3(256), 0, st, x, xs, rows, K, (uint8_t*)data, (uint8_t*)scale, y, ys, colsum);
    else
        hipLaunchKernelGGL((quantize8_kernel<T, false>), grid, dim3(256), 0, st, x, xs, rows, K, (uint8_t*)data, (uint8_t*)scale, y, ys, colsum);
    return launched8("sfm_quantize8");
}

template <typename T>
int dequantize_t(int64_t rows, int K, const void* data, const void* scale, void* y, int64_t ys, hipStream_t st) {
    const int64_t wgs = (rows * ((K + 7) / 8) + 255) / 256, cap = (int64_t)cu_count() * 16;
    hipLaunchKernelGGL((dequantize8_kernel<T>), dim3((unsigned)(wgs < cap ? wgs : cap)), dim3(256), 0, st, (const uint8_t*)data, (const uint8_t*)scale, rows, K,
                       y, ys);
    return launched8("sfm_dequantize8");
}

template <typename T>
int gelu_bwd_t(int64_t rows, int K, const void* x, int64_t xs, const void* data, const void* scale, const void* dy, int64_t dys, void* dx,
               int64_t dxs, hipStream_t st) {
    const int64_t wgs = (rows * ((K + 7) / 8) + 255) / 256, cap = (int64_t)cu_count() * 16;
    const dim3 grid((unsigned)(wgs < cap ? wgs : cap));
    if (data != nullptr)
        hipLaunchKernelGGL((gelu_bwd_kernel<T, true>), grid, dim3(256), 0, st, nullptr, 0, (const uint8_t*)data, (const uint8_t*)scale,
                           rows, K, dy, dys, dx, dxs);
    else
        hipLaunchKernelGGL((gelu_bwd_kernel<T, false>), grid, dim3(256), 0, st, x, xs, nullptr, nullptr, rows, K, dy, dys, dx, dxs);
    return launched8("sfm_gelu_bwd");
}

template <typename T>
int pack_t(int N, int K, const void* w, int64_t ws, void* data, void* scale, void* data_t, void* scale_t, hipStream_t st) {
    hipLaunchKernelGGL((pack8_kernel<T>), dim3((unsigned)blocks8(K), (unsigned)blocks8(N)), dim3(256), 0, st, w, ws, N, K,
                       (uint8_t*)data, (uint8_t*)scale, (uint8_t*)data_t, (uint8_t*)scale_t, pitch8(K), pitch8(N));
    return launched8("sfm_pack8");
}

}  // namespace

#define SFM_BY_TYPE(dtype, F, ...) \
    ((dtype) == SFM_BF16 ? F<BF16>(__VA_ARGS__) : (dtype) == SFM_F16 ? F<F16>(__VA_ARGS__) : F<float>(__VA_ARGS__))

int launch_quantize8(int dtype, int64_t rows, int K, const void* x, int64_t xs, void* data, void* scale, void* y, int64_t ys, float* colsum,
                     hipStream_t st) {
    return SFM_BY_TYPE(dtype, quantize_t, rows, K, x, xs, data, scale, y, ys, colsum, st);
}
int launch_dequantize8(int dtype, int64_t rows, int K, const void* data, const void* scale, void* y, int64_t ys, hipStream_t st) {
    return SFM_BY_TYPE(dtype, dequantize_t, rows, K, data, scale, y, ys, st);
}
int launch_gelu_bwd(int dtype, int64_t rows, int K, const void* x, int64_t xs, const void* data, const void* scale, const void* dy,
                    int64_t dys, void* dx, int64_t dxs, hipStream_t st) {
    return SFM_BY_TYPE(dtype, gelu_bwd_t, rows, K, x, xs, data, scale, dy, dys, dx, dxs, st);
}
int launch_pack8(int dtype, int N, int K, const void* w, int64_t ws, void* data, void* scale, void* data_t, void* scale_t, hipStream_t st) {
    return SFM_BY_TYPE(dtype, pack_t, N, K, w, ws, data, scale, data_t, scale_t, st);
}

}  // namespace sfm
