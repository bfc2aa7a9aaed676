// Rows of bf16 activations -> blocks of e4m3 values (fp8_blocks.h):
//   quantize_fp8            q = blocks(x)
//   add_norm_modulate_fp8   x' = round_bf16(x + f*gate*mask); q = blocks(rms(x') * (1 + scale) + shift)
// The second one's norm is not rounded to bf16 before it is rounded to e4m3: the
// blocks are its only output, and a second rounding would only add to their error.
#include "fp8_blocks.h"

namespace ltxk {
namespace {

constexpr int kBlock = 256;
constexpr int kPerCu = 3;   // workgroups a compute unit of the streaming form (2: 34 us, 4: 39 on [6144, 4096])
constexpr int kItems = 64;  // most batch items that it walks

// ------------------------------------------------------------ quantize_fp8 --
// A wave takes 512 columns (four blocks, 16 lanes of 8 columns each) of a row.  Bound by memory: [24576, 4096]
// 60 us, 5.0 TB/s (a large copy 4.9; two rows a wave 57, eight 60), [6144, 4096] 17.5, [1024, 4096] 4.4 (two rows
// 4.6); read without the streaming hint 61, 18.1 and 5.0; written with it 61, 17.4 and 4.0, but the product that
// reads it next takes 4 us longer at [6144, 4096].
struct QuantParams {
    const uint16_t *x;
    uint8_t *q, *scale;
    int64_t rows;
    int k, kp, groups;  // columns, whole blocks' columns, groups of four blocks
};

__global__ void __launch_bounds__(kBlock) quantize_kernel(QuantParams p)
{
    constexpr int kWaves = kBlock / 64;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t row = unit % p.rows;
    const int group = static_cast<int>(unit / p.rows);
    if (group >= p.groups) return;
    const int col = group * 512 + lane * 8;
    u32x4 raw = {};
    if (col < p.k) raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p.x + row * p.k + col));
    float f[8];
    unpack8v(raw, f);
    uint32_t scale;
    const uint2 q = fp8_quantize8(f, scale);
    if (col < p.kp) *reinterpret_cast<uint2 *>(p.q + row * p.kp + col) = q;
    if ((lane & 15) == 0) p.scale[(group * p.rows + row) * kFp8Group + (lane >> 4)] = static_cast<uint8_t>(scale);
}

// --------------------------------------------------- add_norm_modulate_fp8 --
struct NormParams {
    int64_t rows, tokens;
    int dim, kp, blocks;
    const uint16_t *x, *f, *mask;
    uint16_t *x_out;
    uint8_t *q, *q_scale;
    Ada gate, shift, scale;
    float eps;
};

// One workgroup a row, C chunks of 8 columns a thread (chunk u = thread + 256 i, so
// 16 neighbouring lanes hold a block).  Few rows are bound by the latency of its loads, its
// sum over the workgroup and its stores, one after another: [126, 2048] 5 us, of 1.8 MB.
template <int C>
__global__ void __launch_bounds__(kBlock) add_norm_kernel(NormParams p)
{
    __shared__ float lds[kBlock / 64];
    const int64_t row = blockIdx.x;
    const int64_t b = udiv32(row, p.tokens), t = row - b * p.tokens;
    float v[C][8];
    float s2 = 0.f;
    const float m = p.mask ? bf16_to_f32(p.mask[b]) : 1.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int col = (threadIdx.x + i * kBlock) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (col >= p.dim) continue;
        u32x4 raw = *reinterpret_cast<const u32x4 *>(p.x + row * p.dim + col);
        unpack8v(raw, v[i]);
        if (p.f) {
            float f[8], g[8];
            unpack8v(*reinterpret_cast<const u32x4 *>(p.f + row * p.dim + col), f);
            ada_load8(p.gate, b, t, row, col, 1.f, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] += f[j] * g[j] * m;
            raw = pack8v(v[i]);
            *reinterpret_cast<u32x4 *>(p.x_out + row * p.dim + col) = raw;
            unpack8v(raw, v[i]);  // the norm sees the rounded residual
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s2 = __builtin_fmaf(v[i][j], v[i][j], s2);
    }
    const float r = rsqrtf(row_sum<kBlock>(s2, lds) / static_cast<float>(p.dim) + p.eps);
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int col = (threadIdx.x + i * kBlock) * 8;
        float o[8] = {};
        if (col < p.dim) {
            float sh[8], sc[8];
            ada_load8(p.shift, b, t, row, col, 0.f, sh);
            ada_load8(p.scale, b, t, row, col, 0.f, sc);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = v[i][j] * r * (1.f + sc[j]) + sh[j];
        }
        uint32_t scale;
        const uint2 q = fp8_quantize8(o, scale);
        if (col < p.kp) *reinterpret_cast<uint2 *>(p.q + row * p.kp + col) = q;
        const int block = col / kFp8Block;
        // the bytes past a row's last block, which fill its last group, are written too
        if ((threadIdx.x & 15) == 0 && block < (p.blocks + 3) / 4 * 4)
            p.q_scale[(static_cast<int64_t>(block / kFp8Group) * p.rows + row) * kFp8Group + block % kFp8Group] =
                static_cast<uint8_t>(scale);
    }
}

// The same for modulations of one row per batch item: persistent workgroups walk the rows
// of each item with the item's modulation in registers and the next row on its way while
// one is reduced and written, up to 512 chunks a row (their registers).  With a residual, a
// workgroup a row / this form, us: [6144, 4096] 53 / 34 (5.2 TB/s), [4290, 4096] 34 / 26, [3000,
// 2048] 14 / 12, [1024, 4096] 11 / 11; 4 items of [504, 2048], fewer rows than workgroups, 11 / 13.  Without a
// residual this form takes 20-22 on [6144, 4096].  Modulations by token or index, whose rows differ
// from one row of x to the next, are read for each and keep a workgroup a row: 44-45 with a residual, 28-29 without.
template <int C, bool RESIDUAL>
__global__ void __launch_bounds__(kBlock) add_norm_stream_kernel(NormParams p)
{
    __shared__ float lds[2][kBlock / 64];
    const int lane = threadIdx.x;
    const int rows = static_cast<int>(p.rows), tokens = static_cast<int>(p.tokens), G = static_cast<int>(gridDim.x);
    const uint32_t bytes = static_cast<uint32_t>(p.dim) * 2;
    int parity = 0;
    for (int lo = 0; lo < rows; lo += tokens) {
        const int hi = lo + tokens, at = lo % G, w = static_cast<int>(blockIdx.x);
        int r = lo + (w >= at ? w - at : w - at + G);  // the first row of the item that is w modulo G
        if (r >= hi) continue;
        u32x4 cx[2][C], cf[2][C];
        auto load = [&](int row, u32x4 (&x)[C], u32x4 (&f)[C]) __attribute__((always_inline)) {
            const uint32_t range = row < hi ? bytes : 0;  // nothing is read past the item
            const rsrc_t rx = make_rsrc(p.x + static_cast<int64_t>(row < hi ? row : lo) * p.dim, range);
            const rsrc_t rf = make_rsrc((RESIDUAL ? p.f : p.x) + static_cast<int64_t>(row < hi ? row : lo) * p.dim, range);
#pragma unroll
            for (int k = 0; k < C; ++k) {
                x[k] = ldb(rx, (lane + k * kBlock) * 16u);
                if constexpr (RESIDUAL) f[k] = ldb(rf, (lane + k * kBlock) * 16u);
            }
        };
        load(r, cx[0], cf[0]);
        load(r + G, cx[1], cf[1]);
        float gt[RESIDUAL ? C : 1][8], sh[C][8], sc[C][8];
        const int64_t b = lo / tokens;
#pragma unroll
        for (int k = 0; k < C; ++k) {
            const int col = (lane + k * kBlock) * 8;
            const bool in = col < p.dim;
            if constexpr (RESIDUAL) ada_load8(p.gate, b, 0, lo, in ? col : 0, 1.f, gt[k]);
            ada_load8(p.shift, b, 0, lo, in ? col : 0, 0.f, sh[k]);
            ada_load8(p.scale, b, 0, lo, in ? col : 0, 0.f, sc[k]);
            if constexpr (RESIDUAL)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!in) gt[k][j] = 0.f;  // nothing of column 0's reaches the sum of squares
        }
        const float m = RESIDUAL && p.mask ? bf16_to_f32(p.mask[b]) : 1.f;
        auto step = [&](u32x4 (&x)[C], u32x4 (&f)[C]) __attribute__((always_inline)) {
            float v[C][8], s2 = 0.f;
            u32x4 out[C];
#pragma unroll
            for (int k = 0; k < C; ++k) {
                unpack8v(x[k], v[k]);
                if constexpr (RESIDUAL) {
                    float fv[8];
                    unpack8v(f[k], fv);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[k][j] += fv[j] * gt[k][j] * m;
                    out[k] = pack8v(v[k]);
                    unpack8v(out[k], v[k]);  // the norm sees the rounded residual
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) s2 = __builtin_fmaf(v[k][j], v[k][j], s2);
            }
            load(r + 2 * G, x, f);
            if constexpr (RESIDUAL) {
                const rsrc_t rx = make_rsrc(p.x_out + static_cast<int64_t>(r) * p.dim, bytes);
#pragma unroll
                for (int k = 0; k < C; ++k) stb(rx, (lane + k * kBlock) * 16u, out[k]);
            }
            s2 = wave_sum64(s2);
            if ((lane & 63) == 0) lds[parity][lane >> 6] = s2;
            __syncthreads();
            s2 = (lds[parity][0] + lds[parity][1]) + (lds[parity][2] + lds[parity][3]);
            parity ^= 1;  // the other row's sums go elsewhere, so that one barrier a row is enough
            const float rs = rsqrtf(s2 / static_cast<float>(p.dim) + p.eps);
#pragma unroll
            for (int k = 0; k < C; ++k) {
                const int col = (lane + k * kBlock) * 8;
                float o[8];
                // zeros past the last column, whatever the row's norm and the modulation are
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = col < p.dim ? v[k][j] * rs * (1.f + sc[k][j]) + sh[k][j] : 0.f;
                uint32_t scale;
                const uint2 q = fp8_quantize8(o, scale);
                if (col < p.kp) *reinterpret_cast<uint2 *>(p.q + static_cast<int64_t>(r) * p.kp + col) = q;
                const int block = col / kFp8Block;
                if ((lane & 15) == 0 && block < (p.blocks + 3) / 4 * 4)
                    p.q_scale[(static_cast<int64_t>(block / kFp8Group) * p.rows + r) * kFp8Group + block % kFp8Group] =
                        static_cast<uint8_t>(scale);
            }
            r += G;
            return r < hi;
        };
        while (step(cx[0], cf[0]) && step(cx[1], cf[1])) {
        }
    }
}

template <int C>
void launch_norm(const NormParams &p, hipStream_t s)
{
    bool broadcast = true;
    for (const Ada *a : {&p.gate, &p.shift, &p.scale}) broadcast &= !(a->emb && (a->ts != 0 || a->idx));
    if constexpr (C <= 2) {
        const int64_t grid = static_cast<int64_t>(device_cus()) * kPerCu;
        if (broadcast && p.rows / p.tokens <= kItems && p.tokens > grid) {
            if (p.f)
                add_norm_stream_kernel<C, true><<<static_cast<unsigned>(grid), kBlock, 0, s>>>(p);
            else
                add_norm_stream_kernel<C, false><<<static_cast<unsigned>(grid), kBlock, 0, s>>>(p);
            return;
        }
    }
    add_norm_kernel<C><<<static_cast<unsigned>(p.rows), kBlock, 0, s>>>(p);
}

}  // namespace
}  // namespace ltxk

using namespace ltxk;

extern "C" int ltxk_quantize_fp8(void *q, void *q_scale, const void *x, int64_t rows, int64_t k, void *stream)
{
    static const char *what = "quantize_fp8";
    clear_error();
    if (rows < 0 || k <= 0 || k % 8)
        return fail(LTXK_E_ARG, "%s: bad shape rows=%lld k=%lld (k a positive multiple of 8)", what, (long long)rows,
                    (long long)k);
    if (rows == 0) return LTXK_OK;
    if (!q || !q_scale || !x) return fail(LTXK_E_ARG, "%s: null q, q_scale or x", what);
    if (!aligned16(q) || !aligned16(q_scale) || !aligned16(x))
        return fail(LTXK_E_ALIGN, "%s: q, q_scale and x must be 16-byte aligned", what);
    const int64_t kMax = int64_t{1} << 31, kp = fp8_blocks(k) * kFp8Block;
    if (k >= kMax / 2 || rows > (kMax - 1) / kp) return fail(LTXK_E_ARG, "%s: 2^31 values or more", what);
    QuantParams p{static_cast<const uint16_t *>(x), static_cast<uint8_t *>(q), static_cast<uint8_t *>(q_scale), rows,
                  static_cast<int>(k), static_cast<int>(kp), static_cast<int>(fp8_groups(k))};
    const int64_t grid = (rows * p.groups + 3) / 4;
    quantize_kernel<<<static_cast<unsigned>(grid), kBlock, 0, static_cast<hipStream_t>(stream)>>>(p);
    return check_launch(what);
}

extern "C" int ltxk_add_norm_modulate_fp8(void *x_out, void *q, void *q_scale, const void *x, const void *f,
                                          const ltxk_ada *gate, const void *mask, int64_t rows, int64_t tokens,
                                          int64_t dim, float eps, const ltxk_ada *shift, const ltxk_ada *scale,
                                          void *stream)
{
    static const char *what = "add_norm_modulate_fp8";
    clear_error();
    if (rows < 0 || tokens <= 0 || dim <= 0 || dim % 8 || dim > 16384 || rows % tokens)
        return fail(LTXK_E_ARG, "%s: bad shape rows=%lld tokens=%lld dim=%lld (dim a multiple of 8 up to 16384)", what,
                    (long long)rows, (long long)tokens, (long long)dim);
    if (rows == 0) return LTXK_OK;
    if (!q || !q_scale || !x) return fail(LTXK_E_ARG, "%s: null q, q_scale or x", what);
    if (!f != !x_out) return fail(LTXK_E_ARG, "%s: f and x_out go together", what);
    if (!f && (gate || mask)) return fail(LTXK_E_ARG, "%s: a gate or mask without f", what);
    for (const void *v : {static_cast<const void *>(x_out), static_cast<const void *>(q),
                          static_cast<const void *>(q_scale), x, f})
        if (!aligned16(v)) return fail(LTXK_E_ALIGN, "%s: buffers must be 16-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(mask) & 1u) return fail(LTXK_E_ALIGN, "%s: mask must be 2-byte aligned", what);
    NormParams p{};
    p.gate = make_ada(gate);
    p.shift = make_ada(shift);
    p.scale = make_ada(scale);
    for (const Ada *a : {&p.gate, &p.shift, &p.scale}) {
        if (!ada_aligned(*a))
            return fail(LTXK_E_ALIGN, "%s: AdaLN operands must be 16-byte aligned (pointers and strides)", what);
        if (a->idx && (a->idx_rows == 0 || a->idx_rows > 0x7fffffffu))
            return fail(LTXK_E_ARG, "%s: an operand has an index but emb_rows %u is not in [1, 2^31)", what, a->idx_rows);
    }
    p.kp = static_cast<int>(fp8_blocks(dim) * kFp8Block);
    if (rows > 0x7fffffff / p.kp) return fail(LTXK_E_ARG, "%s: 2^31 values or more", what);
    p.rows = rows;
    p.tokens = tokens;
    p.dim = static_cast<int>(dim);
    p.blocks = static_cast<int>(fp8_blocks(dim));
    p.x = static_cast<const uint16_t *>(x);
    p.f = static_cast<const uint16_t *>(f);
    p.mask = static_cast<const uint16_t *>(mask);
    p.x_out = static_cast<uint16_t *>(x_out);
    p.q = static_cast<uint8_t *>(q);
    p.q_scale = static_cast<uint8_t *>(q_scale);
    p.eps = eps;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int chunks = static_cast<int>(fp8_groups(dim)) * 64;  // a row's threads, the last group's padding too
    if (chunks <= kBlock)
        launch_norm<1>(p, s);
    else if (chunks <= 2 * kBlock)
        launch_norm<2>(p, s);
    else if (chunks <= 4 * kBlock)
        launch_norm<4>(p, s);
    else
        launch_norm<8>(p, s);
    return check_launch(what);
}
