// What the matrix-core kernels share.
#pragma once

#include "ltxk_common.h"

namespace ltxk {

typedef __attribute__((address_space(3))) char lds_char;

// LDS position of 16-byte chunk c of a tile's row of 128 bytes: 16 rows of one
// chunk column, which a fragment read takes at a time, cover all banks.
__device__ __forceinline__ int chunk_pos(int row, int c) { return c ^ ((row >> 1) & 7); }

// 64 lanes x 16 (4) bytes from memory straight to LDS at `lds`, through m0.  In assembly
// because the compiler, which cannot tell the buffers of a ring apart, would wait
// for every load in flight before each LDS read; it has no output register, and its
// wait is step_barrier's.  The wait states cover scalar operands that a vector
// instruction has just written, which the compiler does not see the load read.  It
// does not see m0 change either (a reserved register, whose clobber it ignores with
// a warning): nothing else in a kernel that calls these may use m0, such as an LDS load
// builtin, an indexed register or a message, nor may its assembly.
__device__ __forceinline__ void load_lds16(const u32x4 &rsrc, uint32_t lds, uint32_t off, uint32_t soff)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(lds), "v"(off), "s"(rsrc), "s"(soff)
                 : "memory");
}
__device__ __forceinline__ void load_lds4(const u32x4 &rsrc, uint32_t lds, uint32_t off, uint32_t soff)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 ::"s"(lds), "v"(off), "s"(rsrc), "s"(soff)
                 : "memory");
}

// At most `N` of this wave's loads in flight (none without `more`) and its LDS
// reads returned, then all waves'.
template <int N>
__device__ __forceinline__ void step_barrier(bool more)
{
    asm volatile("" ::: "memory");
    if (more)
        __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4 << 14));  // vmcnt(N) lgkmcnt(0)
    else
        __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A buffer of all memory from `base` on: loads through it go by 32-bit offsets.
__device__ __forceinline__ u32x4 whole_memory(const void *base)
{
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4{static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32) & 0xffff, 0xffffffffu, 0x00020000u};
}

// The rows of x and w from which tile t of a product is made, of TM and TN of them: bands kBand tiles
// of x deep.  8-bit, 24576 x 4096 x 4096 / 6144 x 16384 x 4096, us: 2: 332 / 302, 4: 313 / 300, 8: 317 / 312,
// 16: 323 / 320 (bf16: 8, no difference).
constexpr int kBand = 4;

template <int TM, int TN>
__device__ __forceinline__ void tile_rows(int tiles_m, int tiles_n, int t, int &m0, int &n0)
{
    const int band = t / (kBand * tiles_n), at = t % (kBand * tiles_n);
    const int deep = min(kBand, tiles_m - band * kBand);
    m0 = (band * kBand + at % deep) * TM;
    n0 = at / deep * TN;
}

// A 32 x 32 tile whose lane l holds, of row l % 32, columns 8 q + 4 (l / 32) .. + 3 in v[q]: lanes l
// and l + 32, then l and l + 16, swap, so that lane l holds columns 8 (l / 32) + (l & 16) .. + 7 of
// rows l % 16 (lo) and l % 16 + 16 (hi): a store of 16 rows of 32 columns each (of 32 rows of 16:
// 309 against 302 us on [24576, 4096] x 4096).
__device__ __forceinline__ void rows16(const uint32_t v[4][2], u32x4 &lo, u32x4 &hi)
{
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const auto first = __builtin_amdgcn_permlane32_swap(v[0][e], v[1][e], false, false);
        const auto second = __builtin_amdgcn_permlane32_swap(v[2][e], v[3][e], false, false);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const auto rows = __builtin_amdgcn_permlane16_swap(first[i], second[i], false, false);
            lo[2 * i + e] = rows[0], hi[2 * i + e] = rows[1];
        }
    }
}

}  // namespace ltxk
