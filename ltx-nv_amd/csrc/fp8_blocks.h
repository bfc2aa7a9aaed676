// Blocks of 128 e4m3 values with a power-of-two scale each, the operands of the
// 8-bit linear layers.
//
// A row of k values is held as ceil(k / 128) blocks: with a = max |x| of a block,
// e the least integer with a <= 448 * 2^e, at least -127 (448 is e4m3's largest
// value), the block holds q = e4m3(x * 2^-e) and stands for q * 2^e.  x * 2^-e is
// exact (but where it lies under e4m3's smallest step), so q is one rounding to
// four significant bits, the same however the block was made.  A power of two costs
// no precision against a free scale, since e4m3 is itself floating point: only its
// subnormal range starts up to one binade higher.  And the matrix cores take such
// scales as operands of the product.  An infinity or NaN makes its whole block NaN.
//
// In memory: values (rows, 128 * blocks) bytes, zeros past k (but in a NaN block);
// scales e + 127, one byte a block (255: a NaN block), as (ceil(blocks / 4), rows, 4)
// bytes, so that the scales of neighbouring rows over four blocks are contiguous: a
// tile's scales are one load, and a lane's four blocks one register.
#pragma once

#include "ltxk_common.h"

namespace ltxk {

constexpr int kFp8Block = 128;  // values of a scale
constexpr int kFp8Group = 4;    // scales of a row that lie together

inline int64_t fp8_blocks(int64_t k) { return (k + kFp8Block - 1) / kFp8Block; }
inline int64_t fp8_groups(int64_t k) { return (fp8_blocks(k) + kFp8Group - 1) / kFp8Group; }

// The largest of 16 neighbouring lanes' values (bit patterns of non-negative
// floats, which order as integers do, NaN above infinity), in all of them.
__device__ __forceinline__ uint32_t max16(uint32_t v)
{
    auto take = [&](uint32_t o) { v = v > o ? v : o; };
    take(__builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));   // quad_perm 1,0,3,2
    take(__builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));   // quad_perm 2,3,0,1
    take(__builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));  // row_half_mirror
    take(__builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));  // row_mirror
    return v;
}

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// The scale byte of a block whose largest magnitude has the bits `top`:
// 448 = 1.75 * 2^8, so e is the magnitude's exponent less 8, one more past 1.75.
__device__ __forceinline__ uint32_t fp8_scale(uint32_t top)
{
    const int e = static_cast<int>(top >> 23);  // exponent + 127
    if (e == 255) return 255;
    const int s = e - 8 + ((top & 0x7fffffu) > 0x600000u);
    return s < 0 ? 0 : s;
}

// 2^-e of a scale byte e + 127 (at most 247, so the result is normal)
__device__ __forceinline__ float fp8_inverse(uint32_t scale) { return __uint_as_float((254u - scale) << 23); }

// Four values times `inverse` as e4m3, rounded to nearest even.
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float inverse)
{
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a * inverse, b * inverse, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c * inverse, d * inverse, v, true);
}

// The eight values of a lane in a block that 16 neighbouring lanes hold: `scale`
// is the block's byte.
__device__ __forceinline__ uint2 fp8_quantize8(const float f[8], uint32_t &scale)
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude(f[i]));
    scale = fp8_scale(max16(top));
    if (scale == 255) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    const float inv = fp8_inverse(scale);
    return make_uint2(fp8_pack4(f[0], f[1], f[2], f[3], inv), fp8_pack4(f[4], f[5], f[6], f[7], inv));
}

}  // namespace ltxk
