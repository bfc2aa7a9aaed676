// y = round_bf16(x w^T + bias), and blocks(gelu_tanh(x w^T + bias)), for x (M, K) and
// w (N, K) in blocks of 128 e4m3 values with a power-of-two scale each (fp8_blocks.h):
//
//   sum[m, n] = sum_b 2^(ex[m, b] + ew[n, b]) sum_{k in block b} qx[m, k] qw[n, k]
//
// The scaled matrix instructions multiply both operands by their power of two, so
// the sums run on in fp32 accumulators over all of K.  Inside an instruction the
// products of 8 neighbouring values of k are cut off at 2^-13 of their largest (measured:
// one large and one small product, all pairs of places), which is what its rate costs; over
// K 4096 of normal inputs the sum is then off by 2^-16 of its value (rms), a hundredth of
// the result's rounding to bf16.  Everything past a group of 8 is fp32.
#include "fp8_blocks.h"

namespace ltxk {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Params {
    const uint8_t *x, *xs, *w, *ws;  // values and scales
    const uint16_t *bias;
    uint16_t *y;       // bf16 result, or
    uint8_t *q, *qs;   // its blocks after GELU
    float *part;       // fp32 sums (m, np)
    int m, n, kp, blocks, np;
};

__device__ __forceinline__ i32x8 cat(i32x4 a, i32x4 b)
{
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// gelu_tanh(x) = 0.5 x (1 + tanh(y)), y = sqrt(2/pi) (x + 0.044715 x^3), as
// x / (1 + 2^(-2 y log2 e)).
__device__ __forceinline__ float gelu(float x)
{
    constexpr float kC1 = -2.0f * 1.4426950408889634f * 0.7978845608028654f, kC2 = kC1 * 0.044715f;
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * __builtin_fmaf(kC2, x * x, kC1)));
}

// ------------------------------------------------------------------ few rows --
// 16 rows of w and 16 * MT of x a workgroup; its waves take every kWaves-th block of
// K, straight from memory to registers, and their sums are added in LDS.
constexpr int kWaves = 8;

template <int MT, bool SUMS>
__global__ void __launch_bounds__(kWaves * 64) few_kernel(Fp8Params p)
{
    __shared__ f32x4 sums[kWaves][MT][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int across = (p.n + 15) / 16;
    const int n0 = blockIdx.x % across * 16, m0 = blockIdx.x / across * 16 * MT;
    const int l16 = lane & 15, quad = lane >> 4;
    // rows past the last repeat it; their results are not stored
    const int nr = min(n0 + l16, p.n - 1);
    const uint8_t *wp = p.w + static_cast<int64_t>(nr) * p.kp + quad * 32;
    const uint8_t *xp[MT];
    int mr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        mr[t] = min(m0 + t * 16 + l16, p.m - 1);
        xp[t] = p.x + static_cast<int64_t>(mr[t]) * p.kp + quad * 32;
    }
    f32x4 acc[MT] = {};
    for (int b = wave; b < p.blocks; b += kWaves) {
        const int64_t off = static_cast<int64_t>(b) * kFp8Block;
        const i32x4 *wv = reinterpret_cast<const i32x4 *>(wp + off);
        const i32x8 wf = cat(wv[0], wv[1]);
        const int ws = p.ws[(static_cast<int64_t>(b >> 2) * p.n + nr) * 4 + (b & 3)];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const i32x4 *xv = reinterpret_cast<const i32x4 *>(xp[t] + off);
            const i32x8 xf = cat(xv[0], xv[1]);
            const int xs = p.xs[(static_cast<int64_t>(b >> 2) * p.m + mr[t]) * 4 + (b & 3)];
            acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[t], 0, 0, 0, ws, 0, xs);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= MT) return;
    // lane l: row l % 16 of x, rows 4 (l / 16) .. + 3 of w
    f32x4 v = sums[0][wave][lane];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v += sums[i][wave][lane];
    const int row = m0 + wave * 16 + l16, col = n0 + quad * 4;
    if (row >= p.m || col >= p.n) return;
    if (p.bias)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += bf16_to_f32(p.bias[col + e]);
    if constexpr (SUMS)
        *reinterpret_cast<f32x4 *>(p.part + static_cast<int64_t>(row) * p.np + col) = v;
    else
        *reinterpret_cast<uint2 *>(p.y + static_cast<int64_t>(row) * p.n + col) =
            make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// blocks(gelu(sums)): 16 lanes a block, as quantize_fp8.
__global__ void __launch_bounds__(256) gelu_quantize_kernel(Fp8Params p)
{
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, row = static_cast<int>(unit % p.m);
    const int group = static_cast<int>(unit / p.m), col = group * 512 + lane * 8;
    if (group * 512 >= p.np) return;
    float f[8] = {};
    if (col < p.n) {
        const f32x4 *s = reinterpret_cast<const f32x4 *>(p.part + static_cast<int64_t>(row) * p.np + col);
        const f32x4 lo = s[0], hi = s[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = gelu(lo[e]);
            f[4 + e] = gelu(hi[e]);
        }
    }
    uint32_t scale;
    const uint2 q = fp8_quantize8(f, scale);
    if (col < p.np) *reinterpret_cast<uint2 *>(p.q + static_cast<int64_t>(row) * p.np + col) = q;
    if ((lane & 15) == 0)
        p.qs[(static_cast<int64_t>(group) * p.m + row) * 4 + (lane >> 4)] = static_cast<uint8_t>(scale);
}

template <bool SUMS>
void launch_few(const Fp8Params &p, hipStream_t s)
{
    const unsigned across = static_cast<unsigned>((p.n + 15) / 16);
    if (p.m <= 16)
        few_kernel<1, SUMS><<<across, kWaves * 64, 0, s>>>(p);
    else if (p.m <= 32)
        few_kernel<2, SUMS><<<across, kWaves * 64, 0, s>>>(p);
    else
        few_kernel<4, SUMS><<<across * static_cast<unsigned>((p.m + 63) / 64), kWaves * 64, 0, s>>>(p);
}

int64_t workspace_bytes(int64_t m, int64_t n, int64_t k, bool gelu)
{
    return gelu ? m * fp8_blocks(n) * kFp8Block * 4 : 0;
}

// The checks and the launch of both entry points.
int linear(const char *what, void *y, void *y_scale, bool gelu, const void *x, const void *x_scale, const void *w,
           const void *w_scale, const void *bias, int64_t m, int64_t n, int64_t k, void *workspace,
           int64_t workspace_size, void *stream)
{
    clear_error();
    if (m < 0 || n <= 0 || k <= 0 || n % 8 || k % 8)
        return fail(LTXK_E_ARG, "%s: bad shape m=%lld n=%lld k=%lld (n and k positive multiples of 8)", what,
                    (long long)m, (long long)n, (long long)k);
    if (m == 0) return LTXK_OK;
    if (!y || (gelu && !y_scale) || !x || !x_scale || !w || !w_scale)
        return fail(LTXK_E_ARG, "%s: null operand", what);
    for (const void *v : {static_cast<const void *>(y), static_cast<const void *>(y_scale), x, x_scale, w, w_scale, bias})
        if (!aligned16(v)) return fail(LTXK_E_ALIGN, "%s: operands must be 16-byte aligned", what);
    // operands are read through 32-bit offsets, outputs counted by 32-bit tiles
    const int64_t kMax = int64_t{1} << 31;
    if (k >= kMax / 2 || n >= kMax / 2) return fail(LTXK_E_ARG, "%s: n or k of 2^30 or more", what);
    const int64_t kp = fp8_blocks(k) * kFp8Block, np = fp8_blocks(n) * kFp8Block;
    if (m > (kMax - 1) / kp || n > (kMax - 1) / kp || m > (kMax - 1) / np)
        return fail(LTXK_E_ARG, "%s: x, w or y holds 2^31 values or more", what);
    const int64_t need = workspace_bytes(m, n, k, gelu);
    if (need && (!workspace || !aligned16(workspace) || workspace_size < need))
        return fail(LTXK_E_ARG, "%s: the workspace must hold ltxk_linear_fp8_workspace_bytes, 16-byte aligned", what);
    Fp8Params p{};
    p.x = static_cast<const uint8_t *>(x);
    p.xs = static_cast<const uint8_t *>(x_scale);
    p.w = static_cast<const uint8_t *>(w);
    p.ws = static_cast<const uint8_t *>(w_scale);
    p.bias = static_cast<const uint16_t *>(bias);
    p.y = gelu ? nullptr : static_cast<uint16_t *>(y);
    p.q = gelu ? static_cast<uint8_t *>(y) : nullptr;
    p.qs = static_cast<uint8_t *>(y_scale);
    p.part = static_cast<float *>(workspace);
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.kp = static_cast<int>(kp);
    p.blocks = static_cast<int>(kp / kFp8Block);
    p.np = static_cast<int>(np);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (gelu) {
        launch_few<true>(p, s);
        gelu_quantize_kernel<<<static_cast<unsigned>((m * fp8_groups(n) + 3) / 4), 256, 0, s>>>(p);
    } else {
        launch_few<false>(p, s);
    }
    return check_launch(what);
}

}  // namespace
}  // namespace ltxk

using namespace ltxk;

extern "C" int64_t ltxk_linear_fp8_workspace_bytes(int64_t m, int64_t n, int64_t k, int gelu)
{
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    return workspace_bytes(m, n, k, gelu != 0);
}

extern "C" int ltxk_linear_fp8(void *y, const void *x, const void *x_scale, const void *w, const void *w_scale,
                               const void *bias, int64_t m, int64_t n, int64_t k, void *workspace,
                               int64_t workspace_bytes, void *stream)
{
    return linear("linear_fp8", y, nullptr, false, x, x_scale, w, w_scale, bias, m, n, k, workspace, workspace_bytes,
                  stream);
}

extern "C" int ltxk_linear_gelu_fp8(void *q, void *q_scale, const void *x, const void *x_scale, const void *w,
                                    const void *w_scale, const void *bias, int64_t m, int64_t n, int64_t k,
                                    void *workspace, int64_t workspace_bytes, void *stream)
{
    return linear("linear_gelu_fp8", q, q_scale, true, x, x_scale, w, w_scale, bias, m, n, k, workspace,
                  workspace_bytes, stream);
}
