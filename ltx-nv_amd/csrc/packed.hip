// Attention over sequences laid end to end, and over a prefix that a batch shares: grouped
// heads (query head h reads key head h / (heads / kv_heads)), causal or not:
//
//   out[t, h, :] = round_bf16(sum_j p_j v_j / sum_j p_j),  p_j = 2^(scale log2(e) q.k_j - r)
//
// over the keys j that query t sees, r a reference that the quotient does not depend on.
// A query at position i of its sequence's own n keys (its newest ones are the queries')
// sees keys [lo, hi) of them, hi = i + 1 and lo = max(0, i + 1 - window) where the mask is
// causal and [0, n) else, behind all of the prefix (if i >= 0).  Scores, references, sums
// and output are fp32; p is rounded to bf16 for the second product, and so are the p that
// are summed.
//
// A row is a query at one head of its group, so that one tile of keys serves all heads of
// the group, few queries fill a tile of rows, and a causal tile spans few of them.  Tiles of
// 128 rows share key tiles in LDS, 32 rows a wave (the scores transposed, so that a lane has a
// row's weights as the second product takes them).  Up to 32 rows are attended by all four
// waves, each over keys of its own.  What bounds them:
// * Tiles, long: with half of the time what is not a product (the matrix cores are busy 48 %, with heads of
//   256 42 %), then power.  6144 x 6144 tokens, 32 heads of 128, no mask, 610 us (1.01 PFLOP/s; ltxk_attention
//   599-621), of which the products at a large one's 1.5 PFLOP/s would take 412 and zeros, which draw less power,
//   521 (ltxk_attention 427).  Causal, 12288 tokens over 8 key heads: 1140-1260 us from card to card, 0.98-1.08.
//   Heads of 256 in a window of 1024: 353-430 us for 20078 tokens, 0.68-0.83.
// * Tiles, few: the latency of a tile's chain of products, exponentials and products again, about
//   1.4 us for 64 keys (32 with heads of 256) where no second workgroup shares the unit, with 3 us ahead (which
//   sequence, first keys, queries) and 1-2 behind.  Deeper rings of tiles (three on their way instead of one) change
//   nothing; the weights of a tile beside the scores of the next, 47 against 51 us on prompts of 1024 and
//   333 tokens, heads of 256, but 5 % slower where the chip is full; two groups of waves, 38.
// * Few rows: memory, 5.3-5.4 TB/s on 64 tokens over 125624 keys (516 MB in 95-98 us with the join of their parts, 5;
//   5.7 without); short ones the same latencies.
// * A prefix beside own keys: 64 items of a query, 32 heads of 128 over 8, prefix 8192, own up to 1024, 33 us and 6.5 to
//   join: the latencies of both kinds of tile on places that they share.
// * Units that turn out to be none, which lengths on the device cost: 2-3 us of a workgroup's place each.  A call is
//   cut by its keys, of which a window leaves few, and its join then finds nothing to do: 4 tokens of 16 heads of 256 in
//   a window of 1024 of 4096 keys 18.4 us, over these 1024 alone 16.1; one of 8 heads of 128, of 100000, 12.7 / 12.6.
#include "flash_tiles.h"

#include <cfloat>
#include <type_traits>

namespace ltxk {
namespace {

// Rows (a query at one head of the group) of a tile: 32 a wave, which share its keys, or 32
// that all waves attend with, each over keys of its own.
constexpr int kRows = 32 * kWaves, kFewRows = 32;
// Keys that the former take at a time, and a wave of the latter.  (32 with heads of 256 let two
// workgroups share a unit: 20078 tokens in a window of 1024 367 us, 475 with 64 and one.)
template <int D>
constexpr int kTileKeys = D == 256 ? 32 : 64;
template <int D>
constexpr int kFewKeys = D == 64 ? 64 : 32;

// Tiles of kRows rows take a row's maximum so far, or up to kLag below it, as the reference, so that
// what was summed is rarely rescaled: 12288 causal tokens 1141 us, 1225 with the maximum in every
// tile, four clips 1730 / 1925, a window with heads of 256 359 / 391.  The largest weight is then not
// always 1, and its rounding adds to the error: 1.92e-3 to 2.33e-3 in all against 1.87e-3 to 2.18e-3
// (the output's own rounding is 1.66e-3).  Few rows, which wait for memory, take the maximum.
// The weights are summed as the second product takes them, so that their rounding cancels where
// one of them is most of the sum.  References past kHuge round by more than 2^-4: there the scores
// round first, as the reference did.
constexpr float kLag = 6.f, kHuge = 1048576.f;

// sum + the two bf16 values of `pair`.
__device__ __forceinline__ float add_pair(uint32_t pair, float sum)
{
    const bf16x2_t ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), ones, sum, false);
}

// The keys of a launch: a sequence's (behind the prefix, if there is one), an item's own
// alone, or the prefix alone, for the queries of all items.
enum Keys { kBoth, kOwn, kCommon };

// Parts of cut tiles.
struct Parts {
    float *sums;          // each part's weighted sums of v (rows x D)
    float2 *stats;        // and each of its rows' maximum and sum of weights
    int units, slots;     // parts of all tiles of a key head (with some that are none), and places for them on an XCD
    int rows;             // a part's, as many as a tile has at most
    int parts, least;     // a tile's keys are cut into up to `parts`, of at least `least` key tiles each
    int chunk;            // and of about `chunk` keys (packed: for each row tile of the sequence) each
};

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
    Keys keys;
    bool joined, few;     // every tile is written as parts; tiles of kFewRows rows
    Parts cut;
};

// Values that are the same in all lanes, in scalar registers, as the loads' buffers have to be.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ const char *uniform(const char *x)
{
    const uint64_t a = reinterpret_cast<uint64_t>(x);
    return reinterpret_cast<const char *>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(a >> 32)))) << 32 |
                                          static_cast<uint32_t>(uniform(static_cast<int>(a))));
}

// A tile of rows, what its rows attend to, and where they go.  Rows are a sequence's
// queries, each at all heads of the group in turn, so that few queries fill a tile's rows
// and a causal tile spans few of them.
struct Tile {
    const char *q;        // the sequence's first query, at the group's first head
    int64_t token;        // and that query's row of the output
    const char *k, *v;    // its first own key
    int queries, n;       // its queries and own keys
    int first, rows;      // the tile's first row, and the rows of the whole sequence
    int from, to;         // own keys that some of its rows see
    int np, tiles;        // key tiles: of the prefix, and in all
    int parts, each;      // into which these are cut, and key tiles of a part
    int unit, step;       // the first part's unit, and from each to the next
    bool stacked;         // the queries are those of all items
};

// Packed sequences: of a sequence with r row tiles and m keys, whose parts take about c r keys
// (the more tiles, the longer), all parts number r ceil(m / (c r)), at most floor(m / c) +
// floor(rows / ROWS) + 1.  So unit floor(keys before / c) + floor(rows before / ROWS) + s is
// behind the last one of the sequences before s, and known without their lengths.
template <int ROWS>
__device__ __forceinline__ int first_unit(const Params &p, int s)
{
    const int64_t rows = static_cast<int64_t>(min(max(p.qo[s], 0), p.tq)) * p.group;
    return static_cast<int>(rows / ROWS) + s + (p.cut.parts > 1 ? min(max(p.ko[s], 0), p.tk) / p.cut.chunk : 0);
}

// The last sequence whose first(s) is at most `x`, 64 of them at a time.
template <typename F>
__device__ __forceinline__ int sequence_of(int seqs, int x, F first)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, count = seqs;
    while (count > 1) {
        const int step = (count + 63) / 64, i = lane * step;
        const uint64_t under = __ballot(i < count && first(lo + min(i, count - 1)) <= x);
        const int at = under ? (63 - __builtin_clzll(under)) * step : 0;
        lo += at;
        count = min(step, count - at);
    }
    return uniform(lo);
}

// Sequence (item) s at key head kvh: its operands, and its units, of which there are `parts`
// for a tile at most.
template <int D, int ROWS, int KEYS>
__device__ __forceinline__ void find_sequence(const Params &p, int s, int kvh, Tile &r)
{
    const int64_t qh = static_cast<int64_t>(kvh) * p.group * D * 2, kh = static_cast<int64_t>(kvh) * D * 2;
    r.parts = p.cut.parts;
    r.stacked = p.keys == kCommon;
    if (p.qo) {
        // lengths are cut to what the tensors hold, whatever the offsets say
        const int q0 = min(max(uniform(p.qo[s]), 0), p.tq), q1 = min(uniform(p.qo[s + 1]), p.tq);
        const int k0 = min(max(uniform(p.ko[s]), 0), p.tk), k1 = min(uniform(p.ko[s + 1]), p.tk);
        r.queries = max(q1 - q0, 0);
        r.n = max(k1 - k0, 0);
        r.token = q0;
        r.q = reinterpret_cast<const char *>(p.q) + static_cast<int64_t>(q0) * p.qts + qh;
        r.k = reinterpret_cast<const char *>(p.k) + static_cast<int64_t>(k0) * p.kts + kh;
        r.v = reinterpret_cast<const char *>(p.v) + static_cast<int64_t>(k0) * p.vts + kh;
        r.step = (r.queries * p.group + ROWS - 1) / ROWS;
        r.unit = uniform(first_unit<ROWS>(p, s));
        if (r.parts > 1) {
            const int64_t each = static_cast<int64_t>(p.cut.chunk) * max(r.step, 1);
            r.parts = static_cast<int>(min((r.n + each - 1) / each, static_cast<int64_t>(r.parts)));
        }
    } else {
        const int items = r.stacked ? 1 : p.seqs;
        r.queries = r.stacked ? p.seqs * p.tq : p.tq;
        r.n = r.stacked ? 0 : p.lengths ? min(max(uniform(p.lengths[s]), 0), p.tk) : p.tk;
        r.token = static_cast<int64_t>(s) * p.tq;
        r.q = reinterpret_cast<const char *>(p.q) + s * p.qbs + qh;
        r.k = reinterpret_cast<const char *>(p.k) + s * p.kbs + kh;
        r.v = reinterpret_cast<const char *>(p.v) + s * p.vbs + kh;
        r.step = (r.queries * p.group + ROWS - 1) / ROWS * items;
        r.unit = s;
    }
    r.rows = r.queries * p.group;
}

// Into how many parts `tiles` key tiles are cut, of `each` but the last: `most`, if they are long enough.
__device__ __forceinline__ int parts_of(const Parts &c, int most, int tiles, int &each)
{
    const int parts = max(min(most, tiles / c.least), 1);
    each = (tiles + parts - 1) / parts;
    return parts > 1 ? (tiles + each - 1) / each : 1;
}
template <int KEYS>
__device__ __forceinline__ int batch_parts(const Parts &c, int tiles)
{
    return c.parts > 1 ? min(c.parts, (tiles * KEYS + c.chunk - 1) / c.chunk) : 1;
}

// Row tile `tile` of the sequence: what it attends to, and its parts.
template <int ROWS, int KEYS>
__device__ __forceinline__ void take_tile(const Params &p, int tile, Tile &r)
{
    r.first = tile * ROWS;
    r.unit += tile * (p.qo || r.stacked ? 1 : p.seqs);
    const int behind = r.n - r.queries;  // keys in front of the first query's
    const int last = min(r.first + ROWS, r.rows) - 1;
    r.to = p.causal && !r.stacked ? max(behind + last / p.group + 1, 0) : r.n;
    r.from = p.window ? min(max(behind + r.first / p.group + 1 - p.window, 0), r.to) : 0;
    r.np = r.stacked || (p.keys == kBoth && (r.to || !p.causal)) ? (p.prefix + KEYS - 1) / KEYS : 0;
    r.tiles = r.np + (r.to - r.from + KEYS - 1) / KEYS;
    r.parts = parts_of(p.cut, p.qo ? r.parts : batch_parts<KEYS>(p.cut, r.tiles), r.tiles, r.each);
}

// Unit `unit` of key head kvh: its tile and part, or false if there is none.
template <int D, int ROWS, int KEYS>
__device__ __forceinline__ bool find_tile(const Params &p, int unit, int kvh, Tile &r, int &part)
{
    int tile;
    if (p.qo) {
        const int s = sequence_of(p.seqs, unit, [&](int i) { return first_unit<ROWS>(p, i); });
        find_sequence<D, ROWS, KEYS>(p, s, kvh, r);
        if (unit < r.unit || r.step == 0) return false;
        tile = unit - r.unit;
        part = p.cut.parts > 1 ? tile / r.step : 0;
        tile -= part * r.step;
    } else {
        const int items = p.keys == kCommon ? 1 : p.seqs, x = unit / items;
        find_sequence<D, ROWS, KEYS>(p, unit - x * items, kvh, r);
        const int tiles = r.step / items;
        part = x / tiles;
        tile = x - part * tiles;
    }
    if (tile * ROWS >= r.rows) return false;
    take_tile<ROWS, KEYS>(p, tile, r);
    return part < r.parts;
}

// Row `row` of a tile: its query, head of the group, and the own keys [lo, hi) it sees (and
// the prefix, if any).
struct Row {
    int query, member, lo, hi;
    bool any;
};
__device__ __forceinline__ Row find_row(const Params &p, const Tile &r, int row)
{
    Row w;
    w.query = row / p.group;
    w.member = row - w.query * p.group;
    const int pos = r.n - r.queries + w.query;
    w.hi = p.causal ? max(pos + 1, 0) : r.n;
    w.lo = p.window ? max(w.hi - p.window, 0) : 0;
    w.any = w.hi > w.lo || (p.prefix > 0 && !p.causal);
    return w;
}

// A row's query.
__device__ __forceinline__ const char *query(const Params &p, const Tile &r, const Row &w, int dim)
{
    const char *q = r.q + w.member * dim * 2;
    if (!r.stacked) return q + static_cast<int64_t>(w.query) * p.qts;
    const int item = w.query / p.tq;
    return q + item * p.qbs + static_cast<int64_t>(w.query - item * p.tq) * p.qts;
}

// The keys (values) of key tile g, from `base` on, `valid` of them.
struct Span {
    const char *base;
    uint32_t stride;
    int valid;
};
template <int D, int KEYS, bool V>
__device__ __forceinline__ Span key_span(const Params &p, const Tile &r, int kvh, int g)
{
    Span s;
    if (g < r.np) {
        s.valid = min(KEYS, p.prefix - g * KEYS);
        s.stride = V ? p.pvts : p.pkts;
        s.base = reinterpret_cast<const char *>(V ? p.pv : p.pk) + static_cast<int64_t>(kvh) * D * 2 +
                 static_cast<int64_t>(g) * KEYS * s.stride;
    } else {
        const int at = r.from + (g - r.np) * KEYS;
        s.valid = min(KEYS, r.to - at);
        s.stride = V ? p.vts : p.kts;
        s.base = (V ? r.v : r.k) + static_cast<int64_t>(at) * s.stride;
    }
    s.base = uniform(s.base);
    s.valid = uniform(s.valid);
    s.stride = uniform(s.stride);
    return s;
}

// Bytes that a span's loads may reach.
template <int D>
__device__ __forceinline__ uint32_t reach(const Span &s)
{
    return static_cast<uint32_t>(s.valid - 1) * s.stride + 2 * D;
}

// Adds keys [from, to) to a row's maximum, sum and weighted values: a lane has the
// score of one key of 64, then one or more columns of the values.
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

// One row over key tiles t0 .. t1 - 1 by a whole wave, only what it sees: for rows whose
// matrix products met a masked value that is not finite (its weight of zero makes NaN).
template <int D, int KEYS>
__device__ __forceinline__ void attend_row(const Params &p, const Tile &r, int kvh, int row, int t0, int t1, float &mx,
                                           float &sum, float (&acc)[D / 64])
{
    const Row w = find_row(p, r, row);
    const char *q = query(p, r, w, D);
    const int64_t kh = static_cast<int64_t>(kvh) * D;
    mx = -FLT_MAX;
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = 0.f;
    if (!w.any && !r.stacked) return;
    attend_keys<D>(q, reinterpret_cast<const char *>(p.pk + kh), p.pkts, reinterpret_cast<const char *>(p.pv + kh), p.pvts,
                   min(t0, r.np) * KEYS, min(min(t1, r.np) * KEYS, p.prefix), p.scale2, mx, sum, acc);
    attend_keys<D>(q, r.k, p.kts, r.v, p.vts, max(w.lo, r.from + (max(t0, r.np) - r.np) * KEYS),
                   min(w.hi, r.from + (max(t1, r.np) - r.np) * KEYS), p.scale2, mx, sum, acc);
}

// Unit and key head of this workgroup.  Workgroups are dealt to the 8 XCDs in turn: of the key
// heads, as many at a time as divide 8 go to XCDs of their own, whose L2 then holds their
// keys and values, and each head's units are dealt among its XCDs, in turn where they are
// whole tiles (those with the most keys, a sequence's last ones, first), else in runs.
__device__ __forceinline__ bool find_work(const Params &p, int block, int &unit, int &kvh)
{
    const int xcd = block & 7, j = block >> 3;
    const int beside = p.kv_heads & -p.kv_heads & 7 ? p.kv_heads & -p.kv_heads : 8, each = 8 / beside;
    const Parts &c = p.cut;
    kvh = j / c.slots * beside + xcd % beside;
    unit = c.units - 1 - (c.parts > 1 ? xcd / beside * c.slots + j % c.slots : j % c.slots * each + xcd / beside);
    return unit >= 0;
}

// The place of a part's first row.
__device__ __forceinline__ int64_t part_rows(const Params &p, const Tile &r, int kvh, int part)
{
    return ((r.unit + static_cast<int64_t>(part) * r.step) * p.kv_heads + kvh) * p.cut.rows;
}

// A sum of weights that says that a part has no key, and has written no weighted values.
constexpr float kNoKeys = -1.f;

// A tile without any key: its rows weigh nothing, or are zero.
template <int D, int ROWS, int WAVES>
__device__ __forceinline__ void no_keys(const Params &p, const Tile &r, int kvh, int64_t u, bool joined)
{
    for (int i = threadIdx.x; i < ROWS * (D / 8); i += WAVES * 64) {
        const int at = i / (D / 8), c = i % (D / 8);
        if (r.first + at >= r.rows) break;
        const Row w = find_row(p, r, r.first + at);
        if (!joined)
            *reinterpret_cast<u32x4 *>(p.out + ((r.token + w.query) * p.heads + kvh * p.group + w.member) * D + c * 8) = u32x4{};
        else if (c == 0)
            p.cut.stats[u + at] = make_float2(-FLT_MAX, kNoKeys);
    }
}

// One row over again by a wave: its sums, or its output.
template <int D, int KEYS>
__device__ __forceinline__ void again_row(const Params &p, const Tile &r, int kvh, int row, int t0, int t1, int64_t u, bool joined)
{
    const int lane = threadIdx.x & 63;
    float mx, sum, acc[D / 64];
    attend_row<D, KEYS>(p, r, kvh, row, t0, t1, mx, sum, acc);
    const Row w = find_row(p, r, row);
    if (joined && lane == 0) p.cut.stats[u] = make_float2(mx, sum);
    uint16_t *out = p.out + ((r.token + w.query) * p.heads + kvh * p.group + w.member) * D;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
        const int col = lane * (D / 64) + c;
        if (joined)
            p.cut.sums[u * D + col] = acc[c];
        else
            out[col] = f32_to_bf16(w.any ? acc[c] / sum : 0.f);
    }
}

// The buffer of a span, for load_lds16.
template <int D>
__device__ __forceinline__ u32x4 buffer(const Span &s)
{
    const uint64_t a = reinterpret_cast<uint64_t>(s.base);
    return u32x4{static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32) & 0xffff, reach<D>(s), 0x00020000u};
}

__device__ __forceinline__ uint32_t lds_address(const void *x)
{
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)x));
}

// At most N loads of this wave in flight; nothing moves over it.
template <int N>
__device__ __forceinline__ void wait_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4 << 14));
    asm volatile("" ::: "memory");
}
// This wave's LDS reads have returned; nothing moves over it.
__device__ __forceinline__ void wait_lds()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    asm volatile("" ::: "memory");
}

// LDS of tiles of kRows rows: two stages of keys and values a group, or in the end its sums.
template <int D, int GROUPS>
struct TileLds {
    static constexpr int kBytes = kTileKeys<D> * D * 2;
    union {
        struct {
            char k0[kBytes], k1[kBytes], v0[kBytes], v1[kBytes];
        } of[GROUPS];
        float sums[GROUPS == 1 ? 1 : kRows * D];
    };
    float2 stats[GROUPS == 1 ? 1 : kRows];
};

// A tile of kRows rows by GROUPS times four waves: each group takes every so many key tiles,
// through LDS of its own, and their sums are added up in the end.  Two groups on a unit of their
// own overlap one's products with the other's weights.
template <int D, int GROUPS>
__device__ __forceinline__ void attend_tile(const Params &p, int block, TileLds<D, GROUPS> &whole)
{
    constexpr int KS = D / 16;               // contraction steps of the scores
    constexpr int MT = D / 32;               // output tiles
    constexpr int KT = kTileKeys<D>, KU = KT / 32;
    constexpr int NK = KU * KS, NV = KT / 16 * MT;  // K and V fragments of a tile
    constexpr int kAhead = D == 256 ? 2 : 4;        // fragments read ahead of the products
    constexpr int kTileBytes = KT * D * 2, kParts = kTileBytes / 1024 / kWaves;  // of a tile, and a wave's loads for it

    int unit, kvh, part;
    Tile r;
    if (!find_work(p, block, unit, kvh) || !find_tile<D, kRows, KT>(p, unit, kvh, r, part)) return;
    const bool joined = r.parts > 1 || p.joined;
    const int64_t place = part_rows(p, r, kvh, part);
    const int t0 = part * r.each, all = min(r.each, r.tiles - t0);
    const int any = uniform(threadIdx.x >> 6), group = GROUPS == 1 ? 0 : any / kWaves, wave = GROUPS == 1 ? any : any % kWaves;
    const int lane = threadIdx.x & 63, n = (all - group + GROUPS - 1) / GROUPS;  // the group's tiles
    auto &lds = whole.of[group];
    const int l32 = lane & 31, half = lane >> 5;
    const int first = r.first + wave * 32, last = r.rows - 1;
    const Row own = find_row(p, r, min(first + l32, last));
    const int64_t at = (r.token + own.query) * p.heads + kvh * p.group + own.member;  // this row of the output
    // rows first .. first + 31 all see own keys up to sure_hi from sure_lo on
    const int sure_hi = uniform(own.hi), sure_lo = __builtin_amdgcn_readlane(own.lo, 31);
    uint16_t *const out = p.out;

    if (all == 0) return no_keys<D, kRows, GROUPS * kWaves>(p, r, kvh, place, joined);

    // The keys (values) of tile g on their way into `dst`, a load instruction a call.
    auto load = [&](auto is_v, const u32x4 &rsrc, const Span &s, int c, const char *dst) __attribute__((always_inline)) {
        constexpr bool V = decltype(is_v)::value;
        const int at = wave * kParts + c, row = at * (1024 / (2 * D)) + lane / (D / 8), pos = lane % (D / 8);
        const uint32_t off = __umul24(min(row, s.valid - 1), s.stride) + (V ? v_pos<D>(row, pos) : k_pos<D>(row, pos)) * 16;
        load_lds16(rsrc, lds_address(dst) + at * 1024, off, 0);
    };
    Span ks = key_span<D, KT, false>(p, r, kvh, t0 + min(group, all - 1)), vs = key_span<D, KT, true>(p, r, kvh, t0 + min(group, all - 1));
    // on to the group's tile i
    auto next = [&](auto is_v, Span &s, int i) __attribute__((always_inline)) {
        const int g = t0 + group + i * GROUPS;
        if (GROUPS > 1 || g == r.np) {
            s = key_span<D, KT, decltype(is_v)::value>(p, r, kvh, g);
        } else {
            s.base += static_cast<uint64_t>(s.stride) * KT;
            s.valid = min(KT, g < r.np ? p.prefix - g * KT : r.to - r.from - (g - r.np) * KT);
        }
    };
    auto load_all = [&](auto is_v, Span &s, const char *dst) __attribute__((always_inline)) {
        const u32x4 rsrc = buffer<D>(s);
#pragma unroll
        for (int c = 0; c < kParts; ++c) load(is_v, rsrc, s, c, dst);
    };
    if (n) load_all(std::false_type{}, ks, lds.k0);

    // Queries: lane l holds row l % 32, elements 16 s + 8 (l/32) .. + 7.
    bf16x8 qf[KS];
    {
        const char *qp = query(p, r, own, D) + half * 16;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const bf16x8 *>(qp + s * 32);
    }

    // LDS addresses of this lane's fragments in the first buffers.  K: row l % 32 (+ 32 u),
    // chunk 2 s + half.  V (transposed reads of 4 keys x 16 columns by 16 lanes): rows
    // 16 s + 8 e + 4 half + (l%16)/4, columns 32 m + 16 (l/16 % 2) + 4 (l % 4).  The chunks'
    // permutations are over 16 of them: what is 256 bytes on in heads of 256 keeps its place.
    // (In heads of 256 the first chunk's address gives the others': registers are short.)
    constexpr int KO = KS < 8 ? KS : 8, VO = MT < 4 ? MT : 4, KA = D == 256 ? 1 : KO, VA = D == 256 ? 1 : VO;
    uint32_t k_at[KA], v_at[VA][2];
#pragma unroll
    for (int s = 0; s < KA; ++s) k_at[s] = lds_address(lds.k0) + l32 * 2 * D + k_pos<D>(l32, 2 * s + half) * 16;
    const int vi = lane & 15;
#pragma unroll
    for (int m = 0; m < VA; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = 8 * e + 4 * half + (vi >> 2);
            const int c = 4 * m + 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);
            v_at[m][e] = lds_address(lds.v0) + row * 2 * D + v_pos<D>(row, c) * 16 + (vi & 1) * 8;
        }

    struct Scores {
        f32x16 x[KU];      // transposed: register i of x[u] is key 32 u + 8 (i/4) + 4 half + i % 4 of row l % 32
    };
    f32x16 o[MT] = {};
    u32x4 w[KT / 16];      // weights, two a register, in the order of the scores
    float mx = -FLT_MAX;   // running maximum of the scaled scores (the same in lanes l and l ^ 32)
    float fade = 1.f, scale2 = p.scale2;
    float sum = 0.f;       // this lane's share of the weights' sum

    // Fragment i of a K tile (contraction step i / KU of keys 32 (i % KU) ..) and of a
    // V tile (keys 16 (i / MT) .., columns 32 (i % MT) ..), in the first or second buffer.
    auto k_frag = [&](int buf, int i) {
        typedef const __attribute__((address_space(3))) bf16x8 lds8;
        const int st = i / KU;
        return *(lds8 *)((k_at[st % KA] ^ (KA == 1 ? st % KO * 32 : 0)) + (buf * kTileBytes + i % KU * 64 * D + st / KO * 256));
    };
    auto v_frag = [&](int buf, int i) {
        typedef __attribute__((address_space(3))) bf16x4 lds4;
        const int m = i % MT, x = VA == 1 ? m % VO * 64 : 0, at = buf * kTileBytes + i / MT * 32 * D + m / VO * 256;
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4 *)((v_at[m % VA][0] ^ x) + at));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4 *)((v_at[m % VA][1] ^ x) + at));
        return cat(lo, hi);
    };
    // Matrix phase: a run of the stream of products that a tile takes, the weights
    // times V of the tile before (0 .. NV - 1), then its scores (NV .. NV + NK - 1),
    // with the LDS fragments read ahead of them and `loads(j)` between them.
    auto products = [&](auto from, auto to, int vbuf, int kbuf, Scores &s, auto loads) __attribute__((always_inline)) {
        bf16x8 f[NV + NK];
        auto frag = [&](int j) { f[j] = j < NV ? v_frag(vbuf, j) : k_frag(kbuf, j - NV); };
#pragma unroll
        for (int j = from; j < from + kAhead; ++j) frag(j);
#pragma unroll
        for (int j = from; j < to; ++j) {
            if (j + kAhead < to) frag(j + kAhead);
            loads(j - from);
            if (j < NV) {
                o[j % MT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], __builtin_bit_cast(bf16x8, w[j / MT]), o[j % MT], 0, 0, 0);
            } else {
                const int i = j - NV;
                s.x[i % KU] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], qf[i / KU], i < KU ? f32x16{} : s.x[i % KU], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Weights 2 j and 2 j + 1 of a lane's.
    auto weigh = [&](const Scores &s, int j) __attribute__((always_inline)) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s.x[j >> 3][2 * (j & 7)], scale2, -mx));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s.x[j >> 3][2 * (j & 7) + 1], scale2, -mx));
        w[j >> 2][j & 3] = pack_bf16x2(x, y);
        sum = add_pair(w[j >> 2][j & 3], sum);
    };
    // Keys of tile g that not all of the wave's rows see (or that are none) get weight zero.
    auto mask = [&](Scores &s, int g) __attribute__((always_inline)) {
        const int key = r.from + (g - r.np) * KT;
        const bool common = g < r.np;
        if (common ? p.prefix - g * KT < KT : key + KT > sure_hi || key < sure_lo) {
            const int hi = (common ? p.prefix - g * KT : own.hi - key) - 4 * half;
            const int lo = (common ? 0 : own.lo - key) - 4 * half;
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = 32 * u + 8 * (e >> 2) + (e & 3);
                    if (j >= hi || j < lo) s.x[u][e] = -INFINITY;
                }
        }
    };
    // The reference of the weights after a tile, and what is left of the sums before it.
    auto raise = [&](Scores &s) __attribute__((always_inline)) {
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16 * KU; ++e) m = __builtin_elementwise_maximum(m, s.x[e >> 4][e & 15]);
        m = pair_max(m) * p.scale2;
        const float nm = m > mx + kLag ? m : mx;  // finite, so that scores of -inf weigh zero
        fade = __builtin_amdgcn_exp2f(mx - nm);
        mx = nm;
        scale2 = p.scale2;
        if (__any(fabsf(mx) > kHuge && mx != -FLT_MAX)) {
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) s.x[u][e] *= scale2;
            scale2 = 1.f;
        }
    };
    auto rescale = [&]() __attribute__((always_inline)) {
        if (!__any(fade != 1.f)) return;
        sum *= fade;
#pragma unroll
        for (int c = 0; c < MT; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[c][e] *= fade;
    };

    // Tile i, whose keys are in buffer b: the weights of the tile before times its values, then
    // the scores; its values and the next tile's keys load into the other buffers between the
    // products.
    using std::integral_constant;
    Scores s;
    auto tile = [&](int i, auto from, auto b) __attribute__((always_inline)) {
        constexpr int kEvery = from == 0 ? 3 : 2;
        u32x4 kr = {};  // (an empty buffer: the load gets nothing)
        if (i + 1 < n) {
            next(std::false_type{}, ks, i + 1);
            kr = buffer<D>(ks);
        }
        if (from == 0) next(std::true_type{}, vs, i);
        const u32x4 vr = buffer<D>(vs);
        if (D == 256) asm volatile("" : "+v"(k_at[0]), "+v"(v_at[0][0]), "+v"(v_at[0][1]));
        products(from, integral_constant<int, NV + NK>{}, 1 - b, b, s, [&](int j) __attribute__((always_inline)) {
            if (j % kEvery) return;
            const int c = j / kEvery;
            if (c < kParts) load(std::true_type{}, vr, vs, c, b ? lds.v1 : lds.v0);
            else if (c < 2 * kParts) load(std::false_type{}, kr, ks, c - kParts, b ? lds.k0 : lds.k1);
        });
        mask(s, t0 + group + i * GROUPS);
        raise(s);
        rescale();
#pragma unroll
        for (int j = 0; j < 8 * KU; ++j) weigh(s, j);
    };
    constexpr integral_constant<int, 0> whole_tile, first_buffer;
    constexpr integral_constant<int, 1> second_buffer;
    tile_barrier();
    const int turns = (all + GROUPS - 1) / GROUPS;  // as many barriers for each group
    if (GROUPS == 1 || n) tile(0, integral_constant<int, NV>{}, first_buffer);
    tile_barrier();
    for (int i = 1; i < turns; i += 2) {
        if (GROUPS == 1 || i < n) tile(i, whole_tile, second_buffer);
        tile_barrier();
        if (i + 1 < turns) {
            if (GROUPS == 1 || i + 1 < n) tile(i + 1, whole_tile, first_buffer);
            tile_barrier();
        }
    }
    if (!(n & 1)) {
#pragma unroll
        for (int m = 0; m < VA; ++m) v_at[m][0] += kTileBytes, v_at[m][1] += kTileBytes;
    }
    if (GROUPS == 1 || n) products(whole_tile, integral_constant<int, NV>{}, 0, 0, s, [](int) {});

    // Lane l: row l % 32, columns 32 m + 8 j + 4 half + (0..3) in registers 4 j ..
    float total = pair_sum(sum);
    if constexpr (GROUPS > 1) {
        // The second group's sums on the first one's: 16-byte chunks of a row permuted by the row.
        tile_barrier();
        const int at = wave * 32 + l32;
        f32x4 *const row = reinterpret_cast<f32x4 *>(whole.sums + at * D);
        if (group) {
            if (half == 0) whole.stats[at] = make_float2(mx, total);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    row[(8 * m + 2 * c + half) ^ (l32 & (D / 4 - 1))] = f32x4{o[m][4 * c], o[m][4 * c + 1], o[m][4 * c + 2], o[m][4 * c + 3]};
        }
        tile_barrier();
        if (group) return;
        const float2 other = whole.stats[at];
        const float top = fmaxf(mx, other.x), f = __builtin_amdgcn_exp2f(mx - top), g = __builtin_amdgcn_exp2f(other.x - top);
        mx = top;
        total = total * f + other.y * g;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const f32x4 x = row[(8 * m + 2 * c + half) ^ (l32 & (D / 4 - 1))];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][4 * c + e] = __builtin_fmaf(x[e], g, o[m][4 * c + e] * f);
            }
    }
    float size = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 16; ++e) size = __builtin_elementwise_maximum(size, fabsf(o[m][e]));  // (NaN stays NaN)
    const uint64_t odd = __ballot(!(size <= FLT_MAX));
    uint32_t again = static_cast<uint32_t>(odd) | static_cast<uint32_t>(odd >> 32);  // rows to be done once more
    if (joined) {
        const int64_t u = place + wave * 32 + l32;
        if (first + l32 <= last) {
            if (half == 0) p.cut.stats[u] = make_float2(mx, total);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<f32x4 *>(p.cut.sums + u * D + 32 * m + 8 * c + 4 * half) =
                        f32x4{o[m][4 * c], o[m][4 * c + 1], o[m][4 * c + 2], o[m][4 * c + 3]};
        }
    } else {
        const float inv = own.any ? 1.f / total : 0.f;
        // stored as 64 bytes of 16 rows each
        const int64_t at0 = __shfl(at, lane & 15, 64), at1 = __shfl(at, (lane & 15) + 16, 64);
        const int col = 8 * half + (lane & 16);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            uint32_t v[4][2];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = o[m][4 * c + e] * inv;
                v[c][0] = pack_bf16x2(f[0], f[1]);
                v[c][1] = pack_bf16x2(f[2], f[3]);
            }
            u32x4 lo, hi;
            rows16(v, lo, hi);
            if (first + (lane & 15) <= last)
                __builtin_nontemporal_store(lo, reinterpret_cast<u32x4 *>(out + at0 * D + col + 32 * m));
            if (first + (lane & 15) + 16 <= last)
                __builtin_nontemporal_store(hi, reinterpret_cast<u32x4 *>(out + at1 * D + col + 32 * m));
        }
    }
    if (again) {
        __builtin_amdgcn_s_waitcnt(0x0070);
        asm volatile("" ::: "memory");
        for (; again; again &= again - 1) {
            const int i = __builtin_ctz(again);
            if (first + i <= last)
                again_row<D, KT>(p, r, kvh, first + i, t0, t0 + all, place + wave * 32 + i, joined);
        }
    }
}

// LDS of tiles of few rows: keys and values of each wave, then its sums.
template <int D>
struct FewLds {
    char tile[kWaves][2][kFewKeys<D> * D * 2];
    float2 stat[kWaves][kFewRows];
    uint32_t odd;
};

// A tile of few rows: each wave takes every fourth tile of kFewKeys keys, through LDS of its own
// and without barriers, the next keys on their way while the weights are made and the next
// values while the next scores are; the waves' sums are added up in the end.  What is read is read
// by no other workgroup: streaming loads, 95 against 109 us on 64 tokens over 125624 keys.
template <int D>
__device__ __forceinline__ void attend_few(const Params &p, int block, FewLds<D> &lds)
{
    constexpr int KT = kFewKeys<D>, KU = KT / 32;
    constexpr int KS = D / 16, MT = D / 32;
    constexpr int kBytes = KT * D * 2, NL = kBytes / 1024;  // of a tile, and its load instructions
    auto &stat = lds.stat;
    uint32_t &odd = lds.odd;

    int unit, kvh, part;
    Tile r;
    if (!find_work(p, block, unit, kvh) || !find_tile<D, kFewRows, KT>(p, unit, kvh, r, part)) return;
    const bool joined = r.parts > 1 || p.joined;
    const int64_t place = part_rows(p, r, kvh, part);
    const int t0 = part * r.each, t1 = min(t0 + r.each, r.tiles);
    if (t0 == t1) return no_keys<D, kFewRows, kWaves>(p, r, kvh, place, joined);
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int l32 = lane & 31, half = lane >> 5;
    const int rows = min(kFewRows, r.rows - r.first);
    const Row own = find_row(p, r, r.first + min(l32, rows - 1));
    const int sure_hi = uniform(own.hi), sure_lo = __builtin_amdgcn_readlane(own.lo, 31);
    if (threadIdx.x == 0) odd = 0;

    char *const kt = lds.tile[wave][0], *const vt = lds.tile[wave][1];
    auto load = [&](auto is_v, int g) __attribute__((always_inline)) {
        constexpr bool V = decltype(is_v)::value;
        const Span s = key_span<D, KT, V>(p, r, kvh, g);
        const u32x4 rsrc = buffer<D>(s);
        const uint32_t to = lds_address(V ? vt : kt);
#pragma unroll
        for (int c = 0; c < NL; ++c) {
            const int row = c * (1024 / (2 * D)) + lane / (D / 8), pos = lane % (D / 8);
            const uint32_t off = __umul24(min(row, s.valid - 1), s.stride) + (V ? v_pos<D>(row, pos) : k_pos<D>(row, pos)) * 16;
            load_lds16_stream(rsrc, to + c * 1024, off);
        }
    };
    int g = t0 + wave;
    if (g < t1) {
        load(std::false_type{}, g);
        load(std::true_type{}, g);
    }
    bf16x8 qf[KS];
    {
        const char *qp = query(p, r, own, D) + half * 16;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const bf16x8 *>(qp + s * 32);
    }
    const int vi = lane & 15;
    f32x16 o[MT] = {};
    float mx = -FLT_MAX, sum = 0.f;
    for (; g < t1; g += kWaves) {
        const bool more = g + kWaves < t1;
        wait_loads<NL>();  // the keys are there; the values may be on their way
        f32x16 s[KU] = {};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                const bf16x8 f = *reinterpret_cast<const bf16x8 *>(kt + (l32 + 32 * u) * 2 * D + k_pos<D>(l32, 2 * i + half) * 16);
                s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, qf[i], s[u], 0, 0, 0);
            }
        wait_lds();
        if (more) load(std::false_type{}, g + kWaves);

        const int key = r.from + (g - r.np) * KT;
        const bool common = g < r.np;
        if (common ? p.prefix - g * KT < KT : key + KT > sure_hi || key < sure_lo) {
            const int hi = (common ? p.prefix - g * KT : own.hi - key) - 4 * half;
            const int lo = (common ? 0 : own.lo - key) - 4 * half;
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = 32 * u + 8 * (e >> 2) + (e & 3);
                    if (j >= hi || j < lo) s[u][e] = -INFINITY;
                }
        }
        float m = s[0][0];
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) m = __builtin_elementwise_maximum(m, s[u][e]);
        m = pair_max(m) * p.scale2;
        if (__any(m > mx)) {
            const float nm = m > mx ? m : mx, a = __builtin_amdgcn_exp2f(mx - nm);
            mx = nm;
            sum *= a;
#pragma unroll
            for (int c = 0; c < MT; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[c][e] *= a;
        }
        u32x4 w[KU * 2];
#pragma unroll
        for (int j = 0; j < KU * 8; ++j) {
            // (the scores round before the maximum is taken off, as it did)
            const float x = __builtin_amdgcn_exp2f(s[j >> 3][2 * (j & 7)] * p.scale2 - mx);
            const float y = __builtin_amdgcn_exp2f(s[j >> 3][2 * (j & 7) + 1] * p.scale2 - mx);
            w[j >> 2][j & 3] = pack_bf16x2(x, y);
            sum = add_pair(w[j >> 2][j & 3], sum);
        }

        if (more) wait_loads<NL>();  // the values are there
        else wait_loads<0>();
        typedef __attribute__((address_space(3))) bf16x4 lds4;
#pragma unroll
        for (int st = 0; st < KT / 16; ++st)
#pragma unroll
            for (int c = 0; c < MT; ++c) {
                bf16x4 f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 8 * e + 4 * half + (vi >> 2);
                    const int pos = 4 * c + 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);
                    f[e] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                        (lds4 *)(vt + (row + 16 * st) * 2 * D + v_pos<D>(row, pos) * 16 + (vi & 1) * 8));
                }
                o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cat(f[0], f[1]), __builtin_bit_cast(bf16x8, w[st]), o[c], 0, 0, 0);
            }
        wait_lds();
        if (more) load(std::true_type{}, g + kWaves);
    }

    // The waves' sums on one maximum, side by side in LDS: row l % 32, columns
    // 32 m + 8 j + 4 half + (0..3) in registers 4 j .., 16-byte chunks permuted by the row.
    const float total = pair_sum(sum);
    if (half == 0) stat[wave][l32] = make_float2(mx, total);
    __syncthreads();
    float top = stat[0][l32].x;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, stat[i][l32].x);
    const float fade = __builtin_amdgcn_exp2f(mx - top);
    float *const mine = reinterpret_cast<float *>(lds.tile[wave]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<f32x4 *>(mine + l32 * D + ((8 * m + 2 * c + half) ^ (l32 & (D / 4 - 1))) * 4) =
                f32x4{o[m][4 * c] * fade, o[m][4 * c + 1] * fade, o[m][4 * c + 2] * fade, o[m][4 * c + 3] * fade};
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (D / 8); i += kWaves * 64) {
        const int at = i / (D / 8), c = i % (D / 8);
        float2 st[kWaves];
        float high = -FLT_MAX, all = 0.f, f[8] = {};
#pragma unroll
        for (int k = 0; k < kWaves; ++k) st[k] = stat[k][at], high = fmaxf(high, st[k].x);
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            all += st[k].y * __builtin_amdgcn_exp2f(st[k].x - high);
            const float *x = reinterpret_cast<const float *>(lds.tile[k]) + at * D;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 y = *reinterpret_cast<const f32x4 *>(x + ((2 * c + h) ^ (at & (D / 4 - 1))) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[4 * h + e] += y[e];
            }
        }
        bool fine = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) fine = fine && fabsf(f[e]) <= FLT_MAX;
        if (!fine) atomicOr(&odd, 1u << at);
        if (joined) {
            if (c == 0) p.cut.stats[place + at] = make_float2(high, all);
            f32x4 *x = reinterpret_cast<f32x4 *>(p.cut.sums + (place + at) * D + c * 8);
            x[0] = f32x4{f[0], f[1], f[2], f[3]};
            x[1] = f32x4{f[4], f[5], f[6], f[7]};
        } else {
            const Row w = find_row(p, r, r.first + at);
            const float inv = 1.f / all;
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = w.any ? f[e] * inv : 0.f;
            *reinterpret_cast<u32x4 *>(p.out + ((r.token + w.query) * p.heads + kvh * p.group + w.member) * D + c * 8) = pack8v(f);
        }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);
    __syncthreads();
    for (uint32_t again = uniform(odd); again; again &= again - 1) {
        const int i = __builtin_ctz(again);
        if (i % kWaves == wave) again_row<D, KT>(p, r, kvh, r.first + i, t0, t1, place + i, joined);
    }
}

// Parameters of which the compiler knows what the kind of call fixes, so that it keeps fewer in
// scalar registers, of which up to 88 spill all the same, 96-156 with a prefix and own keys side by side (guidance
// 38.7 -> 37.7 us, 12288 tokens 1220 -> 1213; side by side 50.6 -> 46.7, 42.9 -> 40, 43.4 -> 37.9).
enum Call { kSequences, kItems, kItemsOwn, kPrefixOfAll };
template <Call CALL>
__device__ __forceinline__ Params known(const Params &given)
{
    Params p = given;
    if (CALL == kSequences) {
        __builtin_assume(p.qo != nullptr);
    } else {
        p.qo = p.ko = nullptr;
        p.window = 0;
    }
    if (CALL == kSequences || CALL == kItemsOwn) {
        p.pk = p.pv = nullptr;
        p.prefix = 0;
    }
    if (CALL == kPrefixOfAll) {
        p.lengths = nullptr;
        p.causal = false;
    }
    p.keys = CALL == kPrefixOfAll ? kCommon : CALL == kItemsOwn ? kOwn : kBoth;
    p.joined = CALL == kPrefixOfAll || CALL == kItemsOwn;
    return p;
}

// One kind of tile, or both for a prefix and the items' own keys, side by side.
template <int D, int GROUPS, Call CALL>
__global__ void __launch_bounds__(GROUPS * kWaves * 64, 2) tile_kernel(Params given)
{
    __shared__ __attribute__((aligned(1024))) TileLds<D, GROUPS> lds;
    const Params p = known<CALL>(given);
    attend_tile<D, GROUPS>(p, blockIdx.x, lds);
}
template <int D, Call CALL>
__global__ void __launch_bounds__(kWaves * 64, D == 256 ? 1 : 2) few_kernel(Params given)
{
    __shared__ __attribute__((aligned(1024))) FewLds<D> lds;
    const Params p = known<CALL>(given);
    attend_few<D>(p, blockIdx.x, lds);
}
struct BothParams {
    Params prefix, own;  // for the prefix's tiles, the first `commons` workgroups, and for the others
    int commons;
};
template <int D>
__global__ void __launch_bounds__(kWaves * 64, D == 256 ? 1 : 2) both_kernel(BothParams both)
{
    __shared__ __attribute__((aligned(1024))) union {
        TileLds<D, 1> tile;
        FewLds<D> few;
    } lds;
    const int block = blockIdx.x;
    if (block < both.commons) {
        const Params p = known<kPrefixOfAll>(both.prefix);
        if (p.few) attend_few<D>(p, block, lds.few);
        else attend_tile<D, 1>(p, block, lds.tile);
    } else {
        const Params p = known<kItemsOwn>(both.own);
        if (p.few) attend_few<D>(p, block - both.commons, lds.few);
        else attend_tile<D, 1>(p, block - both.commons, lds.tile);
    }
}

// Joins the parts of the cut tiles, and of a prefix's (`common`, tiles of COMMON rows) with
// those of the items' own keys: a row a wave, whose lanes first have a part's maximum and sum
// each, then 8 columns of every so many parts each.
template <int D, int ROWS, int KEYS, int COMMON>
__global__ void __launch_bounds__(kWaves * 64) join_kernel(Params p, Parts common, int64_t rows)
{
    constexpr int kLanes = D / 8, kBeside = 64 / kLanes;  // lanes of a part, and parts at a time
    const int lane = threadIdx.x & 63, c = lane % kLanes, g = lane / kLanes;
    const int64_t to = static_cast<int64_t>(blockIdx.x) * kWaves + uniform(threadIdx.x >> 6);  // this row of the output
    if (to >= rows) return;
    const int token = static_cast<int>(to / p.heads), head = static_cast<int>(to - static_cast<int64_t>(token) * p.heads);
    const int kvh = head / p.group;
    Tile r;
    find_sequence<D, ROWS, KEYS>(p, p.qo ? sequence_of(p.seqs, token, [&](int i) { return p.qo[i]; }) : token / p.tq, kvh, r);
    if (token < r.token || token >= r.token + r.queries) return;  // of no sequence
    const int in = static_cast<int>(token - r.token) * p.group + head - kvh * p.group, at = in % ROWS;
    take_tile<ROWS, KEYS>(p, in / ROWS, r);
    if (r.parts == 1 && !p.joined) return;  // the tile's only part has written the output
    if (r.unit + (r.parts - 1) * r.step >= p.cut.units) return;  // (offsets that do not ascend)
    const Row w = find_row(p, r, in);
    // the place of a row's first part, and how far it is to the next part's
    const int64_t u = part_rows(p, r, kvh, 0) + at, step = static_cast<int64_t>(r.step) * p.kv_heads * p.cut.rows;
    int64_t cu = 0, cstep = 0;
    int commons = 0;
    if (COMMON) {
        const int all = p.seqs * p.tq * p.group, row = token * p.group + w.member;
        cu = (static_cast<int64_t>(row / COMMON) * p.kv_heads + kvh) * common.rows + row % COMMON;
        cstep = static_cast<int64_t>((all + COMMON - 1) / COMMON) * p.kv_heads * common.rows;
        constexpr int CK = COMMON == kFewRows ? kFewKeys<D> : kTileKeys<D>;
        const int tiles = (p.prefix + CK - 1) / CK;
        int each;
        commons = parts_of(common, batch_parts<CK>(common, tiles), tiles, each);
    }
    const int count = r.parts + commons;
    auto stat = [&](int k) {
        return k < r.parts ? p.cut.stats[u + k * step] : k < count ? common.stats[cu + (k - r.parts) * cstep] : make_float2(-FLT_MAX, kNoKeys);
    };
    float m = -FLT_MAX, sum = 0.f, acc[8] = {};
    for (int k = lane; k < count; k += 64) m = fmaxf(m, stat(k).x);
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    for (int k0 = 0; k0 < count; k0 += 64) {
        // (a part whose weights are all zero still brings the values that are not finite)
        const float2 st = stat(k0 + lane);
        const bool none = st.y == kNoKeys;
        const float f = none ? kNoKeys : __builtin_amdgcn_exp2f(st.x - m);
        sum += none ? 0.f : f * st.y;
        const int here = min(64, count - k0);
#pragma unroll 4
        for (int k = g; k < here + g; k += kBeside) {  // as many turns for every lane
            const int at_k = k0 + min(k, here - 1);
            const float x = __shfl(f, min(k, here - 1), 64);
            const float *sums = at_k < r.parts ? p.cut.sums + (u + at_k * step) * D : common.sums + (cu + (at_k - r.parts) * cstep) * D;
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(sums + c * 8), hi = *reinterpret_cast<const f32x4 *>(sums + c * 8 + 4);
            const bool take = k < here && x != kNoKeys;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[e] = take ? __builtin_fmaf(x, lo[e], acc[e]) : acc[e];
                acc[4 + e] = take ? __builtin_fmaf(x, hi[e], acc[4 + e]) : acc[4 + e];
            }
        }
    }
    sum = wave_sum64(sum);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int o = kLanes; o < 64; o <<= 1) acc[e] += __shfl_xor(acc[e], o, 64);
    const bool any = w.any || (COMMON && !p.causal);
    const float inv = 1.f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = any ? acc[e] * inv : 0.f;
    if (g == 0) *reinterpret_cast<u32x4 *>(p.out + to * D + c * 8) = pack8v(acc);
}

constexpr int64_t kMost = 1 << 29;            // rows and keys, which are counted in int (a prefix's and own keys together)
constexpr int64_t kMostItems = 1 << 20;       // sequences, or items of a batch
constexpr int64_t kMostBlocks = (int64_t{1} << 32) / (kWaves * 64);  // workgroups: a launch holds fewer than 2^32 threads
// Bytes of a prefix not read again that are worth their sums and a second launch.  32 heads of 128 over 8, own keys
// 64, us, shared / not: one query, 4 items, prefix 4096 11.8 / 14.4 (48 MB; not shared), 16384 22 / 31; 32 items, 512
// 20 / 10, 1024 15.7 / 16.4 (124 MB), 4096 19 / 32, 16384 36 / 122; 16 items of 8 queries, 2048 22 / 21 (120 MB), 8192
// 38 / 44, of 28, 42 / 41 and 88 / 89.
constexpr int64_t kShared = 96 << 20;
constexpr int64_t kStride = (1 << 23) - 8;    // elements of a token stride: its bytes are 24 bits

// How the tiles of a launch are cut.  Where they are too few to fill half of the chip (two
// workgroups a compute unit of few rows, but one with heads of 256; one, of two groups, of other
// tiles), their keys go into parts of at least kLeast, if there are enough of them: joining takes a
// second launch, 4-5 us.  One row of 8 key heads over n keys, us, cut / whole: heads of 64, 1024 9.4 / 8.9,
// 1536 9.4 / 11; of 128, 512 10.4 / 8.7, 768 10.5 / 10.8, 1024 10.4 / 12.8; of 256, 300 15.5 / 13.3, 512
// 15.2 / 15.8, 1024 15 / 25.  100 queries, heads of 128, 512 22 / 17, 768 21 / 20, 1536 22 / 31.
// Few rows of packed sequences, whose lengths may differ, go into parts of 3/4 of the average, so that the
// longest do not end last: 64 tokens over 100 to 8192 keys 97 us, in parts of 5/4 108, whole 140; over 300 to
// 3000 (one row a key head, heads of 128) 61 / 66 / -, over 900 to 1100 56 / 56 / -, of exactly 1024 58 / - / 45.
constexpr int64_t kLeast = 256;

// The places, and the keys that a tile's waves take in turn.
int64_t places(int64_t rows, int64_t head_dim) { return rows == kFewRows && head_dim != 256 ? 512 : 256; }
int64_t turns(int64_t rows, int64_t keys, int64_t head_dim)
{
    const int64_t turn = rows == kFewRows ? kWaves * (head_dim == 64 ? 64 : 32) : head_dim == 256 ? 32 : 64;
    return (keys + turn - 1) / turn;
}

struct Cut {
    bool few;             // tiles of kFewRows rows
    int64_t rows, units, parts, least, chunk, slots, blocks;
    int64_t used;         // rows of a tile at most
};

// `tiles` row tiles of a key head over up to `keys` keys each, or (sequences > 0) packed ones over
// all of `keys` together, for `room` places of a key head.
Cut cut(int64_t rows, int64_t tiles, int64_t keys, int64_t sequences, int64_t kv_heads, int64_t head_dim, int64_t room)
{
    Cut c{};
    c.rows = c.used = rows;
    c.few = rows == kFewRows;
    const int64_t per = head_dim == 256 || (c.few && head_dim == 128) ? 32 : 64;  // keys of a key tile
    const int64_t average = sequences ? keys / sequences : keys;
    c.least = kLeast / per;
    c.parts = 1;
    c.chunk = keys > 0 ? keys : 1;
    c.units = tiles;
    const bool worth = average >= (!c.few ? 768 : head_dim == 64 ? 1280 : head_dim == 128 ? 768 : 512), fills = tiles * 2 > room;
    if (worth && sequences && !(fills && !c.few) && tiles <= 4 * room) {
        // (a sequence's row tiles take longer parts instead of more)
        const int64_t each = (tiles + sequences - 1) / sequences;
        c.chunk = fills ? average * 3 / 4 : keys / (room - tiles) + 1;
        if (c.chunk <= kLeast / each) c.chunk = kLeast / each + 1;
        c.parts = (keys + c.chunk - 1) / c.chunk;
        c.units = tiles + keys / c.chunk;
    } else if (worth && !sequences && !fills) {
        const int64_t most = room / tiles;  // (parts without a place would end last: 36 items of 30 queries, 859 keys, heads of 256 54 us, now 35)
        c.chunk = ((keys + per + most - 1) / most + per - 1) / per * per;
        if (c.chunk < kLeast) c.chunk = kLeast;
        c.parts = (keys + per + c.chunk - 1) / c.chunk;
        c.units = tiles * c.parts;
    }
    if (c.parts < 2) c.parts = 1, c.units = tiles;
    const int64_t low = kv_heads & -kv_heads, beside = low < 8 ? low : 8;
    c.slots = (c.units + 8 / beside - 1) / (8 / beside);
    c.blocks = 8 * c.slots * (kv_heads / beside);
    return c;
}

int64_t parts_bytes(const Cut &c, int64_t kv_heads, int64_t head_dim)
{
    return (c.units * kv_heads * c.used * (head_dim + 2) * 4 + 15) / 16 * 16;
}

// Two groups of waves a tile where a unit has no other tile beside it (causal ones are half as
// long as the longest, on average), but for a few keys, which take less than adding up: one sequence,
// 32 heads over 8, us, one / two groups: causal, heads of 64, 128 tokens 7.4 / 7.9, 500 14 / 12, 1000 23 / 19,
// 2000 39 / 35; of 256, 13 / 16, 26 / 25, 46 / 40, 98 / 86; without a mask, heads of 128, 1000 29 / 25, 2000 75 / 82.
int groups_of(const Cut &c, int64_t keys, bool causal, int64_t kv_heads)
{
    return c.units * kv_heads <= (causal ? 512 : 256) && keys >= 256 ? 2 : 1;
}

// A call: one launch over all keys, or one over the prefix for all items and over their own
// keys, whose parts are joined.
struct Plan {
    bool shared;
    int groups;           // of a tile's waves
    Cut own, common;
    int64_t bytes;  // of the workspace
};

// Whether a call's launches hold its workgroups and, joined, a wave for each of its rows.
bool launches_fit(const Plan &c, int64_t rows)
{
    return c.own.blocks + c.common.blocks < kMostBlocks && (c.bytes == 0 || rows < kMostBlocks * kWaves);
}

// Tiles of few rows, where the sequences have few on average.  64 sequences of 1024 keys, us, few / 128 rows, whole:
// heads of 128, 4 rows 45 / 46, 16 53 / 47, 32 64 / 48; of 64, 20 / 28, 19 / 28, 22 / 28; of 256, 88 / 103, 112 / 103, 134 / 103.
// (A sequence has floor(rows / 32) + 1 units, so that 32 rows make one of two units none.)
Plan plan_packed(int64_t tokens_q, int64_t tokens_k, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
                 bool causal)
{
    Plan c{};
    const int64_t rows = tokens_q * (heads / kv_heads), tile = rows * head_dim <= 2048 * sequences ? kFewRows : kRows;
    c.own = cut(tile, rows / tile + sequences, tokens_k, sequences, kv_heads, head_dim, places(tile, head_dim) / kv_heads);
    c.bytes = c.own.parts > 1 ? parts_bytes(c.own, kv_heads, head_dim) : 0;
    c.groups = groups_of(c.own, tokens_k / sequences, causal, kv_heads);
    return c;
}

// The tiles over a shared prefix and those over the items' own keys share the places by the turns that their waves
// take (for all of the items' room, as their lengths are not known here), so that they end together; heads of 64, whose
// few rows wait for memory, halve them.  The prefix's are cut in two at least where there is place, and into 64 at most.
// Against as many places for each as if alone, 80 calls of random sizes take 0.97 of the time: heads of 128 over 8,
// 64 items of 1 query, prefix 8192, own 1024 46.4 -> 40.5 us, 6 of 8 over 34625, own 372 100 -> 76; heads of 256, 7
// items of 5, 4290, own 1536 38 -> 34; but 116 of 8 over 35576, own 774 428 -> 455.
Plan plan_batch(int64_t batch, int64_t tokens_q, int64_t tokens_k, int64_t prefix, int64_t heads, int64_t kv_heads,
                int64_t head_dim, bool causal, bool may_share)
{
    Plan c{};
    const int64_t rows = tokens_q * (heads / kv_heads), tile = rows <= kFewRows ? kFewRows : kRows;
    const int64_t tiles = (rows + tile - 1) / tile * batch;
    if (may_share && batch > 1 && rows < kRows && prefix) {
        const int64_t of_all = batch * rows <= kFewRows ? kFewRows : kRows;
        const int64_t stacked = (batch * rows + of_all - 1) / of_all, room = places(kFewRows, head_dim) / kv_heads;
        const int64_t theirs = stacked * turns(of_all, prefix, head_dim), others = tiles * turns(tile, tokens_k, head_dim);
        int64_t share = head_dim == 64 ? room / 2 : room * theirs / (theirs + others);
        if (share < 2 * stacked && 2 * stacked <= room) share = 2 * stacked;
        if (share > 64 * stacked) share = 64 * stacked;
        c.common = cut(of_all, stacked, prefix, 0, kv_heads, head_dim, share);
        const int64_t sums = 2 * batch * rows * c.common.parts * kv_heads * head_dim * 4;
        c.shared = (batch - 1) * prefix * kv_heads * head_dim * 4 > kShared + sums;
        if (!c.shared) c.common = Cut{};
    }
    const int64_t left = c.shared && head_dim != 64 ? places(kFewRows, head_dim) / kv_heads - c.common.units : places(tile, head_dim) / kv_heads;
    c.own = cut(tile, tiles, (c.shared ? 0 : prefix) + tokens_k, 0, kv_heads, head_dim, left);
    if (rows < tile) c.own.used = rows;
    if (c.shared || c.own.parts > 1) c.bytes = parts_bytes(c.own, kv_heads, head_dim);
    if (c.shared) c.bytes += parts_bytes(c.common, kv_heads, head_dim);
    c.groups = groups_of(c.own, prefix + tokens_k, causal, kv_heads);
    return c;
}

// A prefix is shared where its join and its tiles beside the items' own still fit.
Plan plan_prefix(int64_t batch, int64_t tokens_q, int64_t tokens_k, int64_t prefix, int64_t heads, int64_t kv_heads,
                 int64_t head_dim, bool causal)
{
    const Plan c = plan_batch(batch, tokens_q, tokens_k, prefix, heads, kv_heads, head_dim, causal, true);
    if (!c.shared || launches_fit(c, batch * tokens_q * heads)) return c;
    return plan_batch(batch, tokens_q, tokens_k, prefix, heads, kv_heads, head_dim, causal, false);
}

Parts place(const Cut &c, int64_t kv_heads, int64_t head_dim, void *workspace)
{
    Parts r;
    r.sums = static_cast<float *>(workspace);
    r.stats = reinterpret_cast<float2 *>(r.sums + c.units * kv_heads * c.used * head_dim);
    r.units = static_cast<int>(c.units);
    r.slots = static_cast<int>(c.slots);
    r.parts = static_cast<int>(c.parts);
    r.rows = static_cast<int>(c.used);
    r.least = static_cast<int>(c.least);
    r.chunk = static_cast<int>(c.chunk);
    return r;
}

template <int D, int ROWS, int KEYS>
void join(const Params &p, const Plan &c, const Parts &common, hipStream_t s)
{
    const int64_t rows = static_cast<int64_t>(p.qo ? 1 : p.seqs) * p.tq * p.heads;
    const unsigned blocks = static_cast<unsigned>((rows + kWaves - 1) / kWaves);
    if (!c.shared) join_kernel<D, ROWS, KEYS, 0><<<blocks, kWaves * 64, 0, s>>>(p, common, rows);
    // (stacked rows are few only where an item's are)
    else if (c.common.few) join_kernel<D, kFewRows, kFewKeys<D>, kFewRows><<<blocks, kWaves * 64, 0, s>>>(p, common, rows);
    else join_kernel<D, ROWS, KEYS, kRows><<<blocks, kWaves * 64, 0, s>>>(p, common, rows);
}

template <int D, Call CALL>
void attend(const Params &p, const Plan &c, hipStream_t s)
{
    const unsigned blocks = static_cast<unsigned>(c.own.blocks);
    if (c.own.few) few_kernel<D, CALL><<<blocks, kWaves * 64, 0, s>>>(p);
    else if (c.groups == 2) tile_kernel<D, 2, CALL><<<blocks, 2 * kWaves * 64, 0, s>>>(p);
    else tile_kernel<D, 1, CALL><<<blocks, kWaves * 64, 0, s>>>(p);
}

template <int D>
void launch(Params &p, const Plan &c, void *workspace, hipStream_t s)
{
    p.cut = place(c.own, p.kv_heads, D, workspace);
    p.few = c.own.few;
    Parts common{};
    if (c.shared) {
        common = place(c.common, p.kv_heads, D, static_cast<char *>(workspace) + parts_bytes(c.own, p.kv_heads, D));
        p.joined = true;
        p.keys = kOwn;
        Params all = p;
        all.cut = common;
        all.few = c.common.few;
        all.keys = kCommon;
        const unsigned commons = static_cast<unsigned>(c.common.blocks), owns = static_cast<unsigned>(c.own.blocks);
        both_kernel<D><<<commons + owns, kWaves * 64, 0, s>>>(BothParams{all, p, static_cast<int>(commons)});
    } else if (p.qo) {
        attend<D, kSequences>(p, c, s);
    } else {
        attend<D, kItems>(p, c, s);
    }
    if (c.shared || c.own.parts > 1) c.own.few ? join<D, kFewRows, kFewKeys<D>>(p, c, common, s) : join<D, kRows, kTileKeys<D>>(p, c, common, s);
}

// The launches, once the operands are checked and p holds them.
int run(const char *what, Params &p, const Plan &c, int64_t head_dim, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (!launches_fit(c, (p.qo ? 1 : p.seqs) * static_cast<int64_t>(p.tq) * p.heads))
        return fail(LTXK_E_ARG, "%s: too many row tiles", what);
    if (c.bytes && (!workspace || !aligned16(workspace) || workspace_bytes < c.bytes))
        return fail(LTXK_E_ARG, "%s: the workspace must hold ltxk_%s_workspace_bytes, 16-byte aligned", what, what);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (head_dim == 64) launch<64>(p, c, workspace, s);
    else if (head_dim == 128) launch<128>(p, c, workspace, s);
    else launch<256>(p, c, workspace, s);
    return check_launch(what);
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

// Sizes that a call takes and has work with.
bool sizes_fit(int64_t batch, int64_t tokens_q, int64_t tokens_k, int64_t prefix, int64_t heads, int64_t kv_heads, int64_t head_dim)
{
    return heads > 0 && heads <= (1 << 16) && kv_heads > 0 && heads % kv_heads == 0 && tokens_q > 0 && tokens_q <= kMost / heads / batch &&
           tokens_k >= 0 && tokens_k <= kMost && prefix >= 0 && prefix <= kMost && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

int check_rows(const char *what, const char *name, const void *x, int64_t stride, int64_t width)
{
    if (!x) return fail(LTXK_E_ARG, "%s: null %s", what, name);
    if (!aligned16(x) || stride % 8)
        return fail(LTXK_E_ALIGN, "%s: %s must be 16-byte aligned, with strides that are multiples of 8", what, name);
    if (stride < width || stride > kStride)
        return fail(LTXK_E_ARG, "%s: %s's token stride must be between its width (%lld) and 2^23 - 8", what, name,
                    (long long)width);
    return LTXK_OK;
}

}  // namespace
}  // namespace ltxk

using namespace ltxk;

extern "C" int64_t ltxk_packed_attention_workspace_bytes(int64_t tokens_q, int64_t tokens_k, int64_t sequences,
                                                         int64_t heads, int64_t kv_heads, int64_t head_dim)
{
    if (sequences <= 0 || sequences > kMostItems || !sizes_fit(1, tokens_q, tokens_k, 0, heads, kv_heads, head_dim)) return 0;
    const Plan c = plan_packed(tokens_q, tokens_k, sequences, heads, kv_heads, head_dim, false);
    return launches_fit(c, tokens_q * heads) ? c.bytes : 0;
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
    if (sequences < 0 || sequences > kMostItems)
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
    return run(what, p, plan_packed(tokens_q, tokens_k, sequences, heads, kv_heads, head_dim, p.causal), head_dim, workspace,
               workspace_bytes, stream);
}

extern "C" int64_t ltxk_prefix_attention_workspace_bytes(int64_t batch, int64_t tokens_q, int64_t tokens_k, int64_t prefix,
                                                         int64_t heads, int64_t kv_heads, int64_t head_dim)
{
    if (batch <= 0 || batch > kMostItems || !sizes_fit(batch, tokens_q, tokens_k, prefix, heads, kv_heads, head_dim)) return 0;
    const Plan c = plan_prefix(batch, tokens_q, tokens_k, prefix, heads, kv_heads, head_dim, false);
    return launches_fit(c, batch * tokens_q * heads) ? c.bytes : 0;
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
    if (batch < 0 || batch > kMostItems || prefix < 0)
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
    return run(what, p, plan_prefix(batch, tokens_q, tokens_k, prefix, heads, kv_heads, head_dim, p.causal), head_dim, workspace,
               workspace_bytes, stream);
}
