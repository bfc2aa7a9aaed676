// Attention over sequences laid end to end, and over a prefix that a batch shares: grouped
// heads (query head h reads key head h / (heads / kv_heads)), causal or not, fp32 scores,
// softmax and sums, one rounding to bf16.
//
// A query at position i of its sequence's own n keys (its newest ones are the queries')
// sees keys [lo, hi) of them, hi = i + 1 and lo = max(0, i + 1 - window) where the mask is
// causal and [0, n) else, behind all of the prefix (if i >= 0).
#include "ltxk_common.h"

#include <cfloat>

namespace ltxk {
namespace {

constexpr int kWaves = 4;

struct Params {
    const uint16_t *q, *k, *v, *pk, *pv;
    uint16_t *out;
    const int *qo, *ko;   // packed: where the sequences' queries and keys begin
    const int *lengths;   // batch: how many keys of its own an item has (null: tk)
    int64_t qbs, kbs, vbs;  // batch strides, bytes
    uint32_t qts, kts, vts, pkts, pvts;  // token strides, bytes
    int tq, tk;           // tokens: all (packed) or of an item
    int seqs, prefix, heads, kv_heads, group, window;  // window 0: none
    bool causal;
    float scale2;         // scale * log2(e)
};

// What one sequence's queries attend to, at one key head.
struct Sequence {
    const char *q;        // its first query, at the first head of the group
    int64_t first;        // and that query's row of the output
    const char *k, *v;    // its first own key
    int queries, n;       // queries and own keys
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Sequence s, its lengths cut to what the tensors hold whatever the offsets say.
template <bool PACKED>
__device__ __forceinline__ Sequence sequence(const Params &p, int s, int kvh, int dim)
{
    Sequence r;
    const int64_t qh = static_cast<int64_t>(kvh) * p.group * dim * 2, kh = static_cast<int64_t>(kvh) * dim * 2;
    if constexpr (PACKED) {
        const int q0 = min(max(uniform(p.qo[s]), 0), p.tq), q1 = min(uniform(p.qo[s + 1]), p.tq);
        const int k0 = min(max(uniform(p.ko[s]), 0), p.tk), k1 = min(uniform(p.ko[s + 1]), p.tk);
        r.queries = max(q1 - q0, 0);
        r.n = max(k1 - k0, 0);
        r.first = q0;
        r.q = reinterpret_cast<const char *>(p.q) + static_cast<int64_t>(q0) * p.qts + qh;
        r.k = reinterpret_cast<const char *>(p.k) + static_cast<int64_t>(k0) * p.kts + kh;
        r.v = reinterpret_cast<const char *>(p.v) + static_cast<int64_t>(k0) * p.vts + kh;
    } else {
        r.queries = p.tq;
        r.n = p.lengths ? min(max(uniform(p.lengths[s]), 0), p.tk) : p.tk;
        r.first = static_cast<int64_t>(s) * p.tq;
        r.q = reinterpret_cast<const char *>(p.q) + s * p.qbs + qh;
        r.k = reinterpret_cast<const char *>(p.k) + s * p.kbs + kh;
        r.v = reinterpret_cast<const char *>(p.v) + s * p.vbs + kh;
    }
    return r;
}

// The last s with offsets[s] <= token, of `count` sequences (0 if there is none).
__device__ __forceinline__ int sequence_of(const int *offsets, int count, int token)
{
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (uniform(offsets[mid]) <= token) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Adds keys [from, to) to a row's running maximum, sum and weighted values: a lane has the
// score of one key of 64, then 2 or more columns of the values.
template <int D>
__device__ __forceinline__ void attend_keys(const char *q, const char *k, uint32_t ks, const char *v, uint32_t vs, int from,
                                            int to, float scale2, float &mx, float &sum, float (&acc)[D / 64])
{
    const int lane = threadIdx.x & 63;
    for (int j0 = from; j0 < to; j0 += 64) {
        const int j = min(j0 + lane, to - 1);
        float dot = 0.f;
        for (int c = 0; c < D / 8; ++c) {
            float a[8], b[8];
            unpack8(ld16(q + c * 16), a);
            unpack8(ld16(k + static_cast<int64_t>(j) * ks + c * 16), b);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = __builtin_fmaf(a[e], b[e], dot);
        }
        const float s = j0 + lane < to ? dot * scale2 : -INFINITY;
        float m = s;
#pragma unroll
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        m = fmaxf(m, mx);
        const float fade = __builtin_amdgcn_exp2f(mx - m);
        mx = m;
        sum *= fade;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] *= fade;
        const float w = __builtin_amdgcn_exp2f(s - m);
        sum += wave_sum64(w);
        for (int i = 0; i < min(64, to - j0); ++i) {
            const float wi = __shfl(w, i, 64);
            const uint16_t *row = reinterpret_cast<const uint16_t *>(v + static_cast<int64_t>(j0 + i) * vs) + lane * (D / 64);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) acc[c] = __builtin_fmaf(wi, bf16_to_f32(row[c]), acc[c]);
        }
    }
}

// A wave for each query and head.
template <int D, bool PACKED>
__global__ void __launch_bounds__(kWaves * 64) row_kernel(Params p)
{
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + uniform(threadIdx.x >> 6);
    const int64_t token = row / p.heads;
    const int head = static_cast<int>(row % p.heads), kvh = head / p.group;
    if (token >= static_cast<int64_t>(PACKED ? 1 : p.seqs) * p.tq) return;
    const int s = PACKED ? sequence_of(p.qo, p.seqs, static_cast<int>(token)) : static_cast<int>(token / p.tq);
    const Sequence r = sequence<PACKED>(p, s, kvh, D);
    const int64_t t = token - r.first;
    if (t < 0 || t >= r.queries) return;  // a row of no sequence
    const int pos = r.n - r.queries + static_cast<int>(t);
    const int hi = p.causal ? pos + 1 : r.n, lo = p.window ? max(0, hi - p.window) : 0;
    const char *q = r.q + t * p.qts + (head - kvh * p.group) * D * 2;
    float mx = -FLT_MAX, sum = 0.f, acc[D / 64] = {};
    if (!p.causal || pos >= 0) {
        const int64_t kh = static_cast<int64_t>(kvh) * D;
        attend_keys<D>(q, reinterpret_cast<const char *>(p.pk + kh), p.pkts, reinterpret_cast<const char *>(p.pv + kh), p.pvts,
                       0, p.prefix, p.scale2, mx, sum, acc);
        attend_keys<D>(q, r.k, p.kts, r.v, p.vts, lo, hi, p.scale2, mx, sum, acc);
    }
    const bool none = p.causal ? pos < 0 : p.prefix + r.n == 0;
    uint16_t *out = p.out + (token * p.heads + head) * D + (threadIdx.x & 63) * (D / 64);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) out[c] = f32_to_bf16(none ? 0.f : acc[c] / sum);
}

constexpr int64_t kMost = 0x7fffffff - 1024;  // rows that are counted in int
constexpr int64_t kStride = 1 << 23;          // elements of a token stride: 64 rows within 2^31 bytes

template <bool PACKED>
void launch(const Params &p, int dim, int64_t rows, hipStream_t s)
{
    const unsigned blocks = static_cast<unsigned>((rows + kWaves - 1) / kWaves);
    if (dim == 64) row_kernel<64, PACKED><<<blocks, kWaves * 64, 0, s>>>(p);
    else if (dim == 128) row_kernel<128, PACKED><<<blocks, kWaves * 64, 0, s>>>(p);
    else row_kernel<256, PACKED><<<blocks, kWaves * 64, 0, s>>>(p);
}

// The checks that both entry points share.
int check_sizes(const char *what, int64_t tokens_q, int64_t tokens_k, int64_t heads, int64_t kv_heads, int64_t head_dim,
                float scale, float *scale2)
{
    if (tokens_q < 0 || tokens_k < 0 || heads <= 0 || kv_heads <= 0 || heads > (1 << 16) || heads % kv_heads)
        return fail(LTXK_E_ARG, "%s: bad shape tokens_q=%lld tokens_k=%lld heads=%lld kv_heads=%lld", what,
                    (long long)tokens_q, (long long)tokens_k, (long long)heads, (long long)kv_heads);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(LTXK_E_ARG, "%s: head_dim must be 64, 128 or 256 (got %lld)", what, (long long)head_dim);
    *scale2 = scale * 1.4426950408889634f;
    if (!(scale > 0.f && *scale2 <= FLT_MAX))
        return fail(LTXK_E_ARG, "%s: scale must be positive and finite (got %g)", what, static_cast<double>(scale));
    return LTXK_OK;
}

int check_rows(const char *what, const char *name, const void *x, int64_t stride, int64_t width)
{
    if (!x) return fail(LTXK_E_ARG, "%s: null %s", what, name);
    if (!aligned16(x) || stride % 8)
        return fail(LTXK_E_ALIGN, "%s: %s must be 16-byte aligned, with strides that are multiples of 8", what, name);
    if (stride < width || stride > kStride)
        return fail(LTXK_E_ARG, "%s: %s's token stride must be between its width (%lld) and 2^23", what, name,
                    (long long)width);
    return LTXK_OK;
}

}  // namespace
}  // namespace ltxk

using namespace ltxk;

extern "C" int64_t ltxk_packed_attention_workspace_bytes(int64_t tokens_q, int64_t tokens_k, int64_t sequences,
                                                         int64_t heads, int64_t kv_heads, int64_t head_dim)
{
    return 0;
}

extern "C" int ltxk_packed_attention(void *out, const void *q, int64_t q_tstride, const void *k, int64_t k_tstride,
                                     const void *v, int64_t v_tstride, const int32_t *offsets, const int32_t *k_offsets,
                                     int64_t sequences, int64_t tokens_q, int64_t tokens_k, int64_t heads,
                                     int64_t kv_heads, int64_t head_dim, int causal, int64_t window, float scale,
                                     void *workspace, int64_t workspace_bytes, void *stream)
{
    static const char *what = "packed_attention";
    clear_error();
    Params p{};
    if (int rc = check_sizes(what, tokens_q, tokens_k, heads, kv_heads, head_dim, scale, &p.scale2)) return rc;
    if (sequences < 0 || sequences > (1 << 20))
        return fail(LTXK_E_ARG, "%s: between 0 and 2^20 sequences (got %lld)", what, (long long)sequences);
    if (window < 0 || (window && !causal))
        return fail(LTXK_E_ARG, "%s: a window must be positive, and needs the causal mask", what);
    if (sequences == 0 || tokens_q == 0) return LTXK_OK;
    const int64_t group = heads / kv_heads;
    if (tokens_q > kMost / heads || tokens_k > kMost)
        return fail(LTXK_E_ARG, "%s: too many tokens", what);
    if (!out || !aligned16(out)) return fail(out ? LTXK_E_ALIGN : LTXK_E_ARG, "%s: out must be 16-byte aligned memory", what);
    if (int rc = check_rows(what, "q", q, q_tstride, heads * head_dim)) return rc;
    if (tokens_k) {
        if (int rc = check_rows(what, "k", k, k_tstride, kv_heads * head_dim)) return rc;
        if (int rc = check_rows(what, "v", v, v_tstride, kv_heads * head_dim)) return rc;
    }
    if (!offsets || !k_offsets) return fail(LTXK_E_ARG, "%s: null offsets", what);
    if ((reinterpret_cast<uintptr_t>(offsets) | reinterpret_cast<uintptr_t>(k_offsets)) & 3)
        return fail(LTXK_E_ALIGN, "%s: offsets must be 4-byte aligned", what);
    p.q = static_cast<const uint16_t *>(q);
    p.k = static_cast<const uint16_t *>(k);
    p.v = static_cast<const uint16_t *>(v);
    p.out = static_cast<uint16_t *>(out);
    p.qo = offsets;
    p.ko = k_offsets;
    p.qts = static_cast<uint32_t>(q_tstride * 2);
    p.kts = static_cast<uint32_t>(k_tstride * 2);
    p.vts = static_cast<uint32_t>(v_tstride * 2);
    p.tq = static_cast<int>(tokens_q);
    p.tk = static_cast<int>(tokens_k);
    p.seqs = static_cast<int>(sequences);
    p.heads = static_cast<int>(heads);
    p.kv_heads = static_cast<int>(kv_heads);
    p.group = static_cast<int>(group);
    p.causal = causal != 0;
    p.window = static_cast<int>(window < kMost ? window : 0);  // a window of everything is none
    launch<true>(p, static_cast<int>(head_dim), tokens_q * heads, static_cast<hipStream_t>(stream));
    return check_launch(what);
}

extern "C" int64_t ltxk_prefix_attention_workspace_bytes(int64_t batch, int64_t tokens_q, int64_t tokens_k, int64_t prefix,
                                                         int64_t heads, int64_t kv_heads, int64_t head_dim)
{
    return 0;
}

extern "C" int ltxk_prefix_attention(void *out, const void *q, int64_t q_bstride, int64_t q_tstride, const void *k,
                                     int64_t k_bstride, int64_t k_tstride, const void *v, int64_t v_bstride,
                                     int64_t v_tstride, const void *prefix_k, int64_t prefix_k_tstride,
                                     const void *prefix_v, int64_t prefix_v_tstride, const int32_t *lengths,
                                     int64_t batch, int64_t tokens_q, int64_t tokens_k, int64_t prefix, int64_t heads,
                                     int64_t kv_heads, int64_t head_dim, int causal, float scale, void *workspace,
                                     int64_t workspace_bytes, void *stream)
{
    static const char *what = "prefix_attention";
    clear_error();
    Params p{};
    if (int rc = check_sizes(what, tokens_q, tokens_k, heads, kv_heads, head_dim, scale, &p.scale2)) return rc;
    if (batch < 0 || batch > (1 << 20) || prefix < 0)
        return fail(LTXK_E_ARG, "%s: bad shape batch=%lld prefix=%lld", what, (long long)batch, (long long)prefix);
    if (batch == 0 || tokens_q == 0) return LTXK_OK;
    const int64_t group = heads / kv_heads;
    if (tokens_q > kMost / heads / batch || tokens_k > kMost || prefix > kMost)
        return fail(LTXK_E_ARG, "%s: too many tokens", what);
    if (!out || !aligned16(out)) return fail(out ? LTXK_E_ALIGN : LTXK_E_ARG, "%s: out must be 16-byte aligned memory", what);
    if (int rc = check_rows(what, "q", q, q_tstride, heads * head_dim)) return rc;
    const int64_t width = kv_heads * head_dim;
    if (tokens_k) {
        if (int rc = check_rows(what, "k", k, k_tstride, width)) return rc;
        if (int rc = check_rows(what, "v", v, v_tstride, width)) return rc;
    }
    if (prefix) {
        if (int rc = check_rows(what, "prefix_k", prefix_k, prefix_k_tstride, width)) return rc;
        if (int rc = check_rows(what, "prefix_v", prefix_v, prefix_v_tstride, width)) return rc;
    }
    for (int64_t st : {q_bstride, k_bstride, v_bstride})
        if (st < 0 || st % 8 || st > (int64_t{1} << 40))
            return fail(LTXK_E_ALIGN, "%s: batch strides must be non-negative multiples of 8", what);
    if (reinterpret_cast<uintptr_t>(lengths) & 3) return fail(LTXK_E_ALIGN, "%s: lengths must be 4-byte aligned", what);
    p.q = static_cast<const uint16_t *>(q);
    p.k = static_cast<const uint16_t *>(k);
    p.v = static_cast<const uint16_t *>(v);
    p.pk = static_cast<const uint16_t *>(prefix_k);
    p.pv = static_cast<const uint16_t *>(prefix_v);
    p.out = static_cast<uint16_t *>(out);
    p.lengths = lengths;
    p.qbs = q_bstride * 2;
    p.kbs = k_bstride * 2;
    p.vbs = v_bstride * 2;
    p.qts = static_cast<uint32_t>(q_tstride * 2);
    p.kts = static_cast<uint32_t>(k_tstride * 2);
    p.vts = static_cast<uint32_t>(v_tstride * 2);
    p.pkts = static_cast<uint32_t>(prefix_k_tstride * 2);
    p.pvts = static_cast<uint32_t>(prefix_v_tstride * 2);
    p.tq = static_cast<int>(tokens_q);
    p.tk = static_cast<int>(tokens_k);
    p.seqs = static_cast<int>(batch);
    p.prefix = static_cast<int>(prefix);
    p.heads = static_cast<int>(heads);
    p.kv_heads = static_cast<int>(kv_heads);
    p.group = static_cast<int>(group);
    p.causal = causal != 0;
    launch<false>(p, static_cast<int>(head_dim), batch * tokens_q * heads, static_cast<hipStream_t>(stream));
    return check_launch(what);
}
