// What the attention kernels share: tiles of keys and values in LDS, and a query's row over two lanes.
#pragma once

#include "tiles.h"

namespace ltxk {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;
constexpr int kKeys = 64;         // keys a tile
constexpr float kLarge = 4096.f;  // scaled scores whose products' rounding the weights may show

// LDS position of 16-byte chunk c of a tile's row.  A row is D/8 chunks with no
// padding (the loads write LDS in lane order), so the chunks of a row are
// permuted instead.  K is read 16 bytes a lane down 16 rows of one chunk column,
// V as 4 rows x 64 bytes (a transposed read's four keys): with these
// permutations each such group covers 256 bytes of distinct banks.
template <int D>
__device__ __forceinline__ int k_pos(int row, int c)
{
    return D >= 128 ? c ^ (row & 15) : c ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_pos(int row, int c)
{
    return D >= 128 ? c ^ (((row & 3) << 2) | ((row >> 2) & 3)) : c ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
}

// Part j of a wave's share of a 64-row tile: one load instruction moves 64 lanes
// x 16 bytes straight into LDS.  Rows past the last key repeat it (their scores
// are masked), so nothing outside the tensor is read.
template <int D>
constexpr int kLoads = kKeys * D * 2 / 1024 / kWaves;  // load instructions of a wave for a tile

// The row of a tile that this lane loads in part j.
template <int D>
__device__ __forceinline__ int part_row(int j, int wave, int lane)
{
    return (wave * kLoads<D> + j) * (1024 / (2 * D)) + lane / (D / 8);
}

template <int D, bool V>
__device__ __forceinline__ void load_part(rsrc_t r, char *lds, int j, int key, uint32_t stride, int wave, int lane)
{
    const int at = wave * kLoads<D> + j;
    const int row = part_row<D>(j, wave, lane);
    const int pos = lane % (D / 8);
    const int c = V ? v_pos<D>(row, pos) : k_pos<D>(row, pos);  // the permutations are involutions
    const uint32_t off = static_cast<uint32_t>(key) * stride + c * 16;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_char *)(lds + at * 1024), 16, off, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 cat(bf16x4 a, bf16x4 b)
{
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The larger (sum) of a value over lanes l and l ^ 32, in both.
__device__ __forceinline__ float pair_max(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// This wave's loads have landed and its LDS reads returned, then all waves'.
__device__ __forceinline__ void tile_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace
}  // namespace ltxk
