// Tiles of 64 K / V rows in LDS for the attention kernels: their layout, and how rows get there and back into registers.
#pragma once

#include "sfm_common.hpp"

namespace sfm {

template <int D, int NW = 4>
struct DnLds {
    static constexpr int kCPR = D / 8;                  // 16-byte chunks per row
    static constexpr int kPitch = 2 * D;                // bytes per row
    static constexpr int kMat = 64 * kPitch;            // one 64-row tile
    static constexpr int kK = 0, kV = 2 * kMat;         // K tiles 0/1, then V tiles 0/1
    static constexpr int kStage = NW * 32 * (2 * D + 16);  // output staging, NW waves x 32 rows
    static constexpr int kTotal = 4 * kMat > kStage ? 4 * kMat : kStage;
    // chunk c of row r sits at chunk position c ^ swz(r); depends on r mod 16 only
    static __device__ __forceinline__ int swz(int r) {
        return D >= 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
    }
};

typedef short dn_s16x4 __attribute__((ext_vector_type(4)));

// Transposing LDS read: within each group of 16 lanes, lane i receives element i % 4 of the 8 bytes addressed
// by lanes i/4, i/4 + 4, i/4 + 8, i/4 + 12.  With lane s of a group addressing row s / 4, columns
// 4 (s % 4) .. + 3 of a 4 x 16 block, lane i ends up with column i of the four rows.
__device__ __forceinline__ u32x2 dn_read_tr(const char* lds, uint32_t off) {
    dn_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((dn_s16x4 __attribute__((address_space(3)))*)(lds + off));
    return __builtin_bit_cast(u32x2, v);
}

// 16 bytes per lane from global memory into LDS without passing through registers: lane i of the wave reads
// base + off (off per lane, unsigned 32 bit) and writes LDS bytes [lds_addr + 16 i, + 16).  `base` and `lds_addr`
// are the same in every lane.  The load counts in vmcnt like any other; the compiler does not know that it
// writes LDS, so the code that reads the tile waits (dn_wait_tiles) and synchronises explicitly.
__device__ __forceinline__ void dn_load_lds16(const char* base, uint32_t off, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_addr), "v"(off), "s"(base) : "memory", "m0");
}
// The same past the caches, for rows that are read once
__device__ __forceinline__ void dn_load_lds16_nt(const char* base, uint32_t off, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds_addr), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dn_wait_tiles() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace sfm
