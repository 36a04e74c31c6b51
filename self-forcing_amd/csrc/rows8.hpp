// Rows of channels in registers: eight elements at a time for the three tensor types, sums over a wave, and the 8-bit
// blocks that rows and weights are kept in.
//
// 8-bit blocks: 128 consecutive values of a row share a power of two 2^s, the smallest with max |v| <= 448 * 2^s over the
// finite values (s = 0 for a block of zeros, never below -126); a value is kept as e4m3 of v * 2^-s, ties to even, one
// that is not finite as NaN, and one that would round up to 2^128 (from 248 * 2^120, 3.3e38, on) as 240 * 2^120.  Powers of
// two cost up to one bit of the e4m3 range against a free scale and nothing of its relative precision (half a step is 2^-4
// either way), and the scaled matrix instructions apply them: no product needs a multiplication of its own per block, and the
// 8-bit value times its scale is exact in bf16.
//
// Memory: `data` [rows][round_up(K, 128)] bytes, zeros past K; `scale` bytes s + 127, one word of four for the rows
// 128 g + m + 32 t (t = byte) of block column kb at word (kb * groups + g) * 32 + m, groups = ceil(rows / 128): a lane of a
// 32-row matrix instruction finds the scales of its row in four row blocks in one word.
#pragma once

#include <type_traits>

#include "sfm_common.hpp"

namespace sfm {

template <typename T> struct V8;   // 8 consecutive elements <-> 8 floats
template <> struct V8<float> {
    static __device__ __forceinline__ void load(const void* p, int64_t e, float* x) {
        const f32x4* s = (const f32x4*)((const float*)p + e);
        f32x4 a = s[0], b = s[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static __device__ __forceinline__ void store(void* p, int64_t e, const float* x) {
        f32x4* d = (f32x4*)((float*)p + e);
        f32x4 a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
        d[0] = a; d[1] = b;
    }
    static __device__ __forceinline__ float rnd(float x) { return x; }
};
template <class E> struct V8_16 {
    static __device__ __forceinline__ void load(const void* p, int64_t e, float* x) {
        u32x4 w = *(const u32x4*)((const uint16_t*)p + e);
        uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = E::to_float((uint16_t)(ww[i] & 0xffffu));
            x[2 * i + 1] = E::to_float((uint16_t)(ww[i] >> 16));
        }
    }
    static __device__ __forceinline__ void store(void* p, int64_t e, const float* x) {
        u32x4 w;
        w.x = pack2<E>(x[0], x[1]); w.y = pack2<E>(x[2], x[3]); w.z = pack2<E>(x[4], x[5]); w.w = pack2<E>(x[6], x[7]);
        *(u32x4*)((uint16_t*)p + e) = w;
    }
    static __device__ __forceinline__ float rnd(float x) { return E::to_float(E::from_float(x)); }
};
template <> struct V8<BF16> : V8_16<BF16> {};
template <> struct V8<F16> : V8_16<F16> {};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}


typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

template <typename T> constexpr bool kWide = std::is_same<T, float>::value;      // 4-byte elements

constexpr int kBlock8 = 128;
constexpr int kColRows8 = 32;          // rows of one partial column sum (sfm_quantize8)

__host__ __device__ inline int blocks8(int64_t k) { return (int)((k + kBlock8 - 1) / kBlock8); }
__host__ __device__ inline int64_t pad8(int64_t k) { return (k + kBlock8 - 1) / kBlock8 * kBlock8; }
// bytes between the scales of two block rows of a weight: whole words, which a wave reads through the scalar cache
__host__ __device__ inline int pitch8(int64_t k) { return (blocks8(k) + 3) & ~3; }
// byte of row r in block column kb
__device__ __forceinline__ int64_t scale_at8(int64_t r, int kb, int64_t groups) {
    return ((kb * groups + (r >> 7)) << 7) + ((r & 31) << 2) + ((r & 127) >> 5);
}

// exponent s of a block from the largest finite magnitude
__device__ __forceinline__ int block_exp8(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int s = (int)(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u);      // 448 = 1.75 * 2^8
    return u == 0 ? 0 : max(s, -126);
}
__device__ __forceinline__ float two_to(int s) { return __uint_as_float((uint32_t)(s + 127) << 23); }      // -126 <= s <= 127
// |v| where it counts for a block's scale
__device__ __forceinline__ float finite_mag(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.f;
}
// Blocks with a magnitude from here on hold values that are not finite, or finite ones that e4m3 would round up to 2^128
constexpr float kTop8 = 0x1.fp127f;                       // 248 * 2^120
__device__ __forceinline__ float below_top8(float v) {
    const float a = fabsf(v);
    return a >= kTop8 && a <= 3.402823466e38f ? copysignf(0x1.ep127f, v) : v;         // 240 * 2^120
}
// four values, already divided by the block's scale, to e4m3: at most 448, or not finite, which the conversion turns into NaN
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (uint32_t)w;
}
__device__ __forceinline__ void unpack_e4m3(uint32_t w, float* v) {
    auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
}

// Eight elements of a row of n that may end inside them, at any address that suits the elements (gfx950 takes wide accesses off
// their own alignment); zeros past the end
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct Elem {
    static __device__ __forceinline__ float get(const void* p, int64_t e) { return T::to_float(((const uint16_t*)p)[e]); }
    static __device__ __forceinline__ void put(void* p, int64_t e, float v) { ((uint16_t*)p)[e] = T::from_float(v); }
    static __device__ __forceinline__ void get8(const void* p, int64_t e, float* v) {
        const u32x4 w = *(const u32x4_any*)((const uint16_t*)p + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = T::to_float((uint16_t)(w[i] & 0xffffu));
            v[2 * i + 1] = T::to_float((uint16_t)(w[i] >> 16));
        }
    }
    static __device__ __forceinline__ void put8(void* p, int64_t e, const float* v) {
        const u32x4 w = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
        *(u32x4_any*)((uint16_t*)p + e) = w;
    }
};
template <> struct Elem<float> {
    static __device__ __forceinline__ float get(const void* p, int64_t e) { return ((const float*)p)[e]; }
    static __device__ __forceinline__ void put(void* p, int64_t e, float v) { ((float*)p)[e] = v; }
    static __device__ __forceinline__ void get8(const void* p, int64_t e, float* v) {
        const f32x4_any* s = (const f32x4_any*)((const float*)p + e);
        const f32x4 a = s[0], b = s[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void put8(void* p, int64_t e, const float* v) {
        f32x4_any* d = (f32x4_any*)((float*)p + e);
        d[0] = f32x4{v[0], v[1], v[2], v[3]};
        d[1] = f32x4{v[4], v[5], v[6], v[7]};
    }
};
template <typename T>
__device__ __forceinline__ void load_part8(const void* p, int64_t row_off, int c, int n, float* v) {
    if (c + 8 <= n) {
        Elem<T>::get8(p, row_off + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < n ? Elem<T>::get(p, row_off + c + i) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store_part8(void* p, int64_t row_off, int c, int n, const float* v) {
    if (c + 8 <= n) {
        Elem<T>::put8(p, row_off + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < n) Elem<T>::put(p, row_off + c + i, v[i]);
    }
}

// maximum over the 16 lanes that share a block of 128 values (8 a lane), in all of them: rotations within the row of lanes
__device__ __forceinline__ float max16(float a) {
    auto turned = [](float v, auto by) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + decltype(by)::value, 0xf, 0xf, true));
    };
    a = fmaxf(a, turned(a, std::integral_constant<int, 8>{}));
    a = fmaxf(a, turned(a, std::integral_constant<int, 4>{}));
    a = fmaxf(a, turned(a, std::integral_constant<int, 2>{}));
    return fmaxf(a, turned(a, std::integral_constant<int, 1>{}));
}
// largest magnitude of N values, not numbers left out; from kTop8 on a block is redone by `mag_max_finite`, the rare case
template <int N>
__device__ __forceinline__ float mag_max(const float* v) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) a = fmaxf(a, fabsf(v[i]));
    return a;
}
// the same of the finite ones, which are brought below kTop8
template <int N>
__device__ __forceinline__ float mag_max_finite(float* v) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = below_top8(v[i]);
        a = fmaxf(a, finite_mag(v[i]));
    }
    return a;
}
// 8 values of each of 16 lanes that make a block: the block's exponent, and the lane's bytes
__device__ __forceinline__ int quantize_block8(const float* v0, u32x2* q) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v0[i];
    float a = max16(mag_max<8>(v));
    if (__builtin_expect(a >= kTop8, 0)) a = max16(mag_max_finite<8>(v));
    const int s = block_exp8(a);
    const float inv = two_to(-s);
    q->x = pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    q->y = pack_e4m3(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    return s;
}

// GELU in its tanh form, 0.5 x (1 + tanh(u)) with u = sqrt(2/pi) (x + 0.044715 x^3), as x p with p = 1 / (1 + exp(-2u)): no
// cancellation where tanh approaches -1.  FULL (fp32 tensors): expf and a division; otherwise the hardware's 2^x and reciprocal,
// good to a unit of fp32 each, with -2 log2(e) in the constants.
template <bool FULL>
__device__ __forceinline__ float gelu_gate(float x) {
    if (FULL) return 1.f / (1.f + expf(-1.5957691216057308f * (x + 0.044715f * x * x * x)));
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * (-2.3022082f - 0.10294324f * x * x)));
}
// d gelu / dx = p + x p (1 - p) 2 u'(x); past |x| = 16 p is 0 or 1 to fp32
template <bool FULL>
__device__ __forceinline__ float gelu_slope(float x) {
    if (fabsf(x) > 16.f) return x > 0.f ? 1.f : 0.f;
    const float p = gelu_gate<FULL>(x);
    return p + x * p * (1.f - p) * (1.5957691216057308f + 0.21406445f * x * x);
}

// Rows first .. last - 1, of a group of `rows`, that workgroup `part` of `parts` takes (LayerNorm's backward); none where the parts
// before it have all.  Up to 2^31 - 1 rows: in 64 bits, the sums pass 32.
struct RowRange {
    int64_t first, last;
};
__host__ __device__ inline RowRange rows_of_part(int64_t rows, int parts, int part) {
    const int64_t per = (rows + parts - 1) / parts, first = part * per;
    return {first, first + per < rows ? first + per : rows};
}

// `wgs` workgroups of up to 1024 threads as a grid: the runtime refuses 2^32 work-items or more along one dimension.  A kernel numbers
// them blockIdx.y * gridDim.x + blockIdx.x, and those from wgs on have nothing to do.
inline dim3 wide_grid(int64_t wgs) {
    const int64_t x = wgs < (1 << 21) ? wgs : 1 << 21;
    return dim3((unsigned)x, (unsigned)((wgs + x - 1) / x));
}

// the launch that precedes: SFM_OK, or SFM_ERR_HIP with the runtime's message
inline int launched8(const char* what) {
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) return SFM_OK;
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return SFM_ERR_HIP;
}

// quant8.hip
int launch_quantize8(int dtype, int64_t rows, int K, const void* x, int64_t xs, void* data, void* scale, void* y, int64_t ys, float* colsum,
                     hipStream_t st);
int launch_dequantize8(int dtype, int64_t rows, int K, const void* data, const void* scale, void* y, int64_t ys, hipStream_t st);
int launch_gelu_bwd(int dtype, int64_t rows, int K, const void* x, int64_t xs, const void* data, const void* scale, const void* dy,
                    int64_t dys, void* dx, int64_t dxs, hipStream_t st);
int launch_pack8(int dtype, int N, int K, const void* w, int64_t ws, void* data, void* scale, void* data_t, void* scale_t, hipStream_t st);
// linear8.hip; x: the 16-bit rows, or null.  Up to kFewRows8 of them are quantised in the product's own kernel, which reads no blocks
constexpr int kFewRows8 = SFM_LINEAR8_FEW_ROWS;
int launch_linear8(const sfm_linear8_desc& d, const void* x, int64_t x_stride, const void* x8, const void* xscale, const void* w8,
                   const void* wscale, const void* bias, const void* res, const void* gate, void* out, hipStream_t stream);
int tile_rows8(int64_t M, int N, int K, bool* half_strip);
// linear8_wgrad.hip; `colsum`: column sums of dy by kColRows8 rows where a quantisation has formed them, else null
size_t wgrad8_workspace_bytes(int64_t M, int N, int K, bool bias);
int wgrad8_tile_size(int64_t M, int N, int K, int* parts);
int launch_wgrad8(int dtype, int64_t M, int N, int K, const void* dy, int64_t dy_stride, const void* x8, const void* xscale, void* dw,
                  void* dbias, const float* colsum, void* workspace, hipStream_t st);
// ln_train.hip; launch_sum_parts: out[g][c] = sum over s of part[g][s][c], two halves of the columns to out1 and out2 if that is given
int launch_sum_parts(int dtype, int64_t parts, int64_t n, int64_t groups, const float* part, void* out1, void* out2, hipStream_t st);
size_t ln_bwd_workspace_bytes(int64_t rows, int C, int64_t rows_per_group);
int launch_ln_bwd(int dtype, int64_t rows, int C, float eps, const void* x, int64_t xs, const void* data, const void* scale8,
                  const float* rstd, const void* dy, int64_t dys, const void* weight, int64_t ms, int64_t rows_per_group, bool mod, void* dx,
                  int64_t dxs, void* dw, void* db, void* workspace, hipStream_t st);
int launch_ln_keep8(int dtype, int64_t rows, int C, float eps, const void* x, int64_t xs, void* y, int64_t ys, const void* scale,
                    const void* shift, int64_t ms, int rows_per_frame, const void* weight, const void* bias, void* data, void* scale8,
                    float* rstd, hipStream_t st);

}  // namespace sfm
