// What the matrix-core kernels share.
#pragma once

#include "ltxk_common.h"

namespace ltxk {

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
