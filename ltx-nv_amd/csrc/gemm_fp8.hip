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
//
// What bounds it, by the rows of x: memory up to about 32 (the weights are read once: 4 x 36864 x
// 4096 of 151 MB in 31 us, 4.8 TB/s, where kernels that stream rows reach 5.2-6.6: its 1152 workgroups
// have 768 places, a round and a half); the latency of a launch's one round
// up to a few hundred (126 x 2048 x 2048 in 5 us); for one round of tiles its first loads, stores and launch, about 8 us,
// and LDS, whose reads and writes take 0.32 us of a step's 0.46 (1024 x 4096 x 4096 in 23-26 us, on zeros 22); the
// card's power beyond (24576 x 4096 x 4096 in 287-331 us from card to card, 2.5-2.9 PFLOP/s, on zeros 227 us, 3.63; the
// library's product with a single scale for each operand 270-292 and 212).
#include "fp8_blocks.h"
#include "tiles.h"

#include <algorithm>
#include <type_traits>

namespace ltxk {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Params {
    const uint8_t *x, *xs, *w, *ws;  // values and scales
    const uint16_t *x16;             // x in bf16 instead, rows of k
    const uint16_t *bias;
    uint16_t *y;       // bf16 result, or
    uint8_t *q, *qs;   // its blocks after GELU
    float *part;       // fp32 sums (m, np)
    int m, n, k, kp, blocks, np;
    int tiles_m, tiles_n;
    int whole, rest, parts;  // tiles that one workgroup takes alone; the others, cut into parts over K
    int per;                 // units of the cut tiles an XCD
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

// --------------------------------------------------------------------- tiles --
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Tiles of TM x 128, four waves of TM / 2 x 64, the steps of 128 values as deep in LDS as fit.
// Two teams of four waves that take turns at the steps (two waves a SIMD) are 2-6 % slower: LDS bounds
// a step, not the loads' latency.
constexpr int kTile = 128, kTileWaves = 4;

template <int TM, bool GELU>
__global__ void __launch_bounds__(kTileWaves * 64, 1) tile_kernel(Fp8Params p)
{
    constexpr int MT = TM / 64, NT = kTile / 64, ROWS = TM + kTile;
    constexpr int kRing = TM == kTile ? 4 : 3, kLoads = ROWS / 8 / kTileWaves;  // of a wave for a step
    constexpr int kStep = ROWS * 128, kScalesAt = kRing * kStep, kGroup = ROWS * 4;
    __shared__ __attribute__((aligned(1024))) char smem[kScalesAt + 2 * kGroup];  // two groups' scales
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int l32 = lane & 31, half = lane >> 5;

    // A run of neighbouring tiles per XCD (workgroups are dealt to the XCDs in
    // turn), so that its L2 serves a tile of either side to several workgroups.
    const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3, whole_per = p.whole >> 3;
    int tile, part = -1;
    if (j < whole_per) {
        tile = xcd * whole_per + j;
    } else {
        const int unit = xcd * p.per + j - whole_per;
        if (unit >= p.rest * p.parts) return;
        part = p.parts == 1 ? -1 : unit / p.rest;
        tile = p.whole + unit % p.rest;
    }
    int m0, n0;
    tile_rows<TM, kTile>(p.tiles_m, p.tiles_n, tile, m0, n0);
    // parts * blocks stays below 2^32: 256 parts at most of fewer than 2^24 blocks
    auto from = [&](int i) { return static_cast<int>(static_cast<uint32_t>(i) * p.blocks / static_cast<uint32_t>(p.parts)); };
    const int first = part < 0 ? 0 : from(part), n = (part < 0 ? p.blocks : from(part + 1)) - first;

    const u32x4 xr = whole_memory(p.x), wr = whole_memory(p.w);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)smem));
    // Load c of a step: rows (4 c + wave) * 8 .. + 7 of the tile's x and w together.
    // Rows past the last repeat it; their results are not stored.
    uint32_t at[kLoads];
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
        const int row = (c * kTileWaves + wave) * 8 + (lane >> 3);
        const bool is_x = c * kTileWaves * 8 < TM;
        at[c] = static_cast<uint32_t>(is_x ? min(m0 + row, p.m - 1) : min(n0 + row - TM, p.n - 1)) *
                    static_cast<uint32_t>(p.kp) + chunk_pos(row, lane & 7) * 16;
    }
    // Scales, 64 rows a load: x's, then w's, some of them by two waves.
    const u32x4 xsr = whole_memory(p.xs), wsr = whole_memory(p.ws);
    constexpr int kX = TM / 64, kW = kTile / 64;
    const int sx = wave % kX * 64, sw = wave % kW * 64;
    const uint32_t xso = static_cast<uint32_t>(min(m0 + sx + lane, p.m - 1)) * 4;
    const uint32_t wso = static_cast<uint32_t>(min(n0 + sw + lane, p.n - 1)) * 4;
    const int groups = (p.blocks + 3) >> 2;
    // A group's scales, into its half of their place; past the last group the last one's, which nothing reads.
    // Every step loads them (2 of a wave's 10 loads), not one in four, so that the steps are the same code.
    auto load_scales = [&](int group) {
        const uint32_t to = lds0 + kScalesAt + (group & 1) * kGroup, g = min(group, groups - 1);
        load_lds4(xsr, __builtin_amdgcn_readfirstlane(to + sx * 4), xso, __builtin_amdgcn_readfirstlane(g * p.m * 4));
        load_lds4(wsr, __builtin_amdgcn_readfirstlane(to + (TM + sw) * 4), wso, __builtin_amdgcn_readfirstlane(g * p.n * 4));
    };
    // Load c of step i, into place `slot` of the ring.
    auto load = [&](int i, int c, int slot) {
        load_lds16(c * kTileWaves * 8 < TM ? xr : wr,
                   __builtin_amdgcn_readfirstlane(lds0 + slot * kStep + (c * kTileWaves + wave) * 1024), at[c],
                   __builtin_amdgcn_readfirstlane((first + i) * kFp8Block));
    };
    load_scales(first >> 2);
    load_scales((first >> 2) + 1);
    for (int i = 0; i < kRing && i < n; ++i)
#pragma unroll
        for (int c = 0; c < kLoads; ++c) load(i, c, i);

    int off[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) off[s] = l32 * 128 + chunk_pos(l32, 2 * s + half) * 16;
    const int wm = (wave >> 1) * (TM / 2), wn = (wave & 1) * 64;  // this wave's rows

    // acc[i][j]: lane l holds row 32 i + l % 32 of x; register r row 32 j + 8 (r/4) + 4 half + r % 4 of w
    f32x16 acc[MT][NT] = {};
    // Fragments of a half step (64 values): x's in two sets, w's in one whose second half is
    // read while the first is multiplied, which is what the registers hold.
    constexpr int kEarly = NT / 2;
    i32x8 xf[2][MT], wf[NT];
    int xs[MT], ws[NT], xs_next[MT], ws_next[NT];  // scales of this step and the next
    auto fragment = [&](int base, int s) {
        const i32x4 *lo = reinterpret_cast<const i32x4 *>(smem + base + off[2 * s]);
        const i32x4 *hi = reinterpret_cast<const i32x4 *>(smem + base + off[2 * s + 1]);
        return cat(*lo, *hi);
    };
    auto read_x = [&](int base, int s, int t) { xf[s][t] = fragment(base + t * 4096, s); };
    auto read_w = [&](int base, int s, int t) { wf[t] = fragment(base + t * 4096, s); };
    const int scale_row = kScalesAt + (wm + l32) * 4, scale_row_w = kScalesAt + (TM + wn + l32) * 4;
    auto read_scales = [&](int abs) {
        const char *at = smem + (abs >> 2 & 1) * kGroup + (abs & 3);
#pragma unroll
        for (int t = 0; t < MT; ++t) xs_next[t] = *reinterpret_cast<const uint8_t *>(at + scale_row + t * 128);
#pragma unroll
        for (int t = 0; t < NT; ++t) ws_next[t] = *reinterpret_cast<const uint8_t *>(at + scale_row_w + t * 128);
    };

    // Loads that may be in flight when a step has to be there: those issued after its last
    constexpr int kNewer = (kRing - 2) * kLoads;
    step_barrier<kNewer + kLoads>(n >= kRing);
    read_scales(first);
    int slot = 0, x_at = wm * 128, w_at = (TM + wn) * 128;  // this step's place, and this wave's rows there
#pragma unroll
    for (int t = 0; t < MT; ++t) read_x(x_at, 0, t);
#pragma unroll
    for (int t = 0; t < kEarly; ++t) read_w(w_at, 0, t);

    // Step i, without a branch inside (the compiler would move the products past it).  With
    // `more`, the loads of the step that takes its place are between its products.
    auto step = [&](int i, auto more) __attribute__((always_inline)) {
        // Products before the turn: beside one each the second half of this half step's w is
        // read, the last one covers those reads.  Past it the next half step's x and first half of w.
        constexpr int kProducts = MT * NT, kTurn = NT - kEarly + 1, kSlots = kProducts - kTurn;
        constexpr int kReads = (MT + kEarly + kSlots - 1) / kSlots, kEach = (kLoads + kSlots - 1) / kSlots;
        const int slot_next = slot + 1 == kRing ? 0 : slot + 1;
        const int x_next = slot_next * kStep + wm * 128, w_next = slot_next * kStep + (TM + wn) * 128;
#pragma unroll
        for (int t = 0; t < MT; ++t) xs[t] = xs_next[t];
#pragma unroll
        for (int t = 0; t < NT; ++t) ws[t] = ws_next[t];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < kProducts; ++e) {
                if (e < kTurn) {
                    if (kEarly + e < NT) read_w(w_at, s, kEarly + e);
                } else {
                    // step i + 1 is there, and all waves have read step i whole, so its place
                    // goes to step i + kRing
                    if (s == 1 && e == kTurn) {
                        step_barrier<more ? kNewer : 0>(true);
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (more) load_scales(((first + i) >> 2) + 1);
                        read_scales(first + i + 1);
                    }
#pragma unroll
                    for (int t = (e - kTurn) * kReads; t < (e - kTurn + 1) * kReads && t < MT + kEarly; ++t) {
                        if (t < MT)
                            read_x(s == 0 ? x_at : x_next, s ^ 1, t);
                        else
                            read_w(s == 0 ? w_at : w_next, s ^ 1, t - MT);
                    }
                    if constexpr (more)
                        if (s == 1)
#pragma unroll
                            for (int c = (e - kTurn) * kEach; c < (e - kTurn + 1) * kEach && c < kLoads; ++c)
                                load(i + kRing, c, slot);
                }
                const int ni = e / MT, mi = e % MT;
                acc[mi][ni] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[ni], xf[s][mi], acc[mi][ni], 0, 0, 0,
                                                                             ws[ni], 0, xs[mi]);
                __builtin_amdgcn_sched_barrier(0);
            }
        slot = slot_next, x_at = x_next, w_at = w_next;
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    int i = 0;
    for (; i + kRing < n; ++i) step(i, yes);
    for (; i < n; ++i) step(i, no);

    if (TM == kTile && part >= 0) {
        float *sums = p.part + (static_cast<int64_t>(part) * p.rest + tile - p.whole) * (kTile * kTile);
#pragma unroll
        for (int mi = 0; mi < MT; ++mi)
#pragma unroll
            for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4 *>(sums + (wm + mi * 32 + l32) * kTile + wn + ni * 32 + 8 * q + 4 * half) =
                        f32x4{acc[mi][ni][4 * q], acc[mi][ni][4 * q + 1], acc[mi][ni][4 * q + 2], acc[mi][ni][4 * q + 3]};
        return;
    }
    // a bias past the last column reads the last ones; not stored
    if (p.bias)
#pragma unroll
        for (int ni = 0; ni < NT; ++ni)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint16_t *b = p.bias + min(n0 + wn + ni * 32 + 8 * q + 4 * half, p.n - 4);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int mi = 0; mi < MT; ++mi) acc[mi][ni][4 * q + e] += bf16_to_f32(b[e]);
            }
    if constexpr (!GELU) {
#pragma unroll
        for (int mi = 0; mi < MT; ++mi) {
            const int row = m0 + wm + mi * 32 + l32;
            if (row >= p.m) continue;
#pragma unroll
            for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int col = n0 + wn + ni * 32 + 8 * q + 4 * half;
                    if (col >= p.n) continue;
                    *reinterpret_cast<uint2 *>(p.y + static_cast<int64_t>(row) * p.n + col) =
                        make_uint2(pack_bf16x2(acc[mi][ni][4 * q], acc[mi][ni][4 * q + 1]),
                                   pack_bf16x2(acc[mi][ni][4 * q + 2], acc[mi][ni][4 * q + 3]));
                }
        }
        return;
    }
    // GELU, the largest magnitude of each row's 128 columns (those of two waves side
    // by side), the block
    uint32_t top[MT];
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) {
        top[mi] = 0;
#pragma unroll
        for (int ni = 0; ni < NT; ++ni)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool in = n0 + wn + ni * 32 + 8 * (r >> 2) + 4 * half < p.n;
                const float g = in ? gelu(acc[mi][ni][r]) : 0.f;
                acc[mi][ni][r] = g;
                top[mi] = max(top[mi], magnitude(g));
            }
        const auto both = __builtin_amdgcn_permlane32_swap(top[mi], top[mi], false, false);
        top[mi] = max(static_cast<uint32_t>(both[0]), static_cast<uint32_t>(both[1]));
    }
    uint32_t *tops = reinterpret_cast<uint32_t *>(smem);
    __syncthreads();  // all waves are done with the tiles
    if (half == 0)
#pragma unroll
        for (int mi = 0; mi < MT; ++mi) tops[wave * (MT * 32) + mi * 32 + l32] = top[mi];
    __syncthreads();
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) top[mi] = max(top[mi], tops[(wave ^ 1) * (MT * 32) + mi * 32 + l32]);
    const int block = (n0 + wn) / kFp8Block, last = p.np / kFp8Block - 1;
    if (block > last) return;
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) {
        const int row = m0 + wm + mi * 32 + l32;
        if (row >= p.m) continue;
        const uint32_t scale = fp8_scale(top[mi]);
        const float inv = fp8_inverse(scale == 255 ? 127 : scale);
#pragma unroll
        for (int ni = 0; ni < NT; ++ni)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t v = fp8_pack4(acc[mi][ni][4 * q], acc[mi][ni][4 * q + 1], acc[mi][ni][4 * q + 2],
                                             acc[mi][ni][4 * q + 3], inv);
                *reinterpret_cast<uint32_t *>(p.q + static_cast<int64_t>(row) * p.np + n0 + wn + ni * 32 + 8 * q + 4 * half) =
                    scale == 255 ? 0x7f7f7f7fu : v;
            }
        if (half || wn % kFp8Block) continue;
        // the last block's lane also fills its group
        for (int b = block; b == block || (block == last && b <= (last | 3)); ++b)
            p.qs[(static_cast<int64_t>(b >> 2) * p.m + row) * 4 + (b & 3)] = b == block ? static_cast<uint8_t>(scale) : 0;
    }
}

// ------------------------------------------------------------------ large tiles --
// 256 x 256 tiles, four waves of 128 x 128 (a third less read from LDS than by eight of
// 64 x 128, whose reads and the loads' writes took all of its cycles), one workgroup a compute
// unit that takes its tiles (and parts of tiles) one after another: the loads run two steps
// ahead of the products, into the next tile where this one ends, so that they go on during
// the epilogue.  24576 x 4096 x 4096, on one card: eight waves and a workgroup a tile 380 us, this 312.
// GELU's epilogue needs more than the registers hold (6 vector and 14 scalar ones are spilled); the same
// product with it takes 320-361 us.
constexpr int kBig = 256, kBigWaves = 4, kBigLoads = 2 * kBig / 8 / kBigWaves;
constexpr int kDeepLoads = 6;                                  // of a wave: 192 rows of x, three steps in LDS
constexpr int kNearLoads = kBigLoads - kDeepLoads;             // the other rows of x and w: two steps
constexpr int kDeepRows = kDeepLoads * kBigWaves * 8;
constexpr int kDeepBytes = kDeepRows * 128, kNearBytes = (2 * kBig - kDeepRows) * 128;
constexpr int kNearAt = 3 * kDeepBytes, kScalesAt = kNearAt + 2 * kNearBytes, kScaleBytes = 2 * kBig * 4;
constexpr int kBigLds = kScalesAt + 3 * kScaleBytes;
constexpr int kCus = 32;  // workgroups of an XCD at a time

struct Unit {
    int tile, part;   // part < 0: the whole of K
    int m0, n0, first, n;
};

__device__ __forceinline__ Unit unit_at(const Fp8Params &p, int xcd, int j)
{
    Unit u;
    const int whole_per = p.whole >> 3;
    u.part = -1;
    if (j < whole_per) {
        u.tile = xcd * whole_per + j;
    } else {
        const int i = xcd * p.per + j - whole_per;
        u.part = p.parts == 1 ? -1 : i / p.rest;
        u.tile = p.whole + i % p.rest;
    }
    tile_rows<kBig, kBig>(p.tiles_m, p.tiles_n, u.tile, u.m0, u.n0);
    // parts * blocks stays below 2^32: 256 parts at most of fewer than 2^24 blocks
    auto from = [&](int i) { return static_cast<int>(static_cast<uint32_t>(i) * p.blocks / static_cast<uint32_t>(p.parts)); };
    u.first = u.part < 0 ? 0 : from(u.part);
    u.n = (u.part < 0 ? p.blocks : from(u.part + 1)) - u.first;
    return u;
}

// Units of an XCD: its whole tiles, then its share of the cut ones.
__device__ __forceinline__ int units_of(const Fp8Params &p, int xcd)
{
    return (p.whole >> 3) + max(0, min(p.per, p.rest * p.parts - xcd * p.per));
}

// An accumulator's value where the epilogue uses it: in assembly because the compiler
// otherwise copies all 256 of them to vector registers at once, and spills.  It does not
// see that a product wrote them, so settle() comes first: 32 wait states, of which a product needs 19.
__device__ __forceinline__ float taken(float acc)
{
    float v;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(acc));
    return v;
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// The bias of four columns from `col`; past the last column the last ones' (not stored).
__device__ __forceinline__ uint2 bias4(const Fp8Params &p, int col)
{
    return p.bias ? *reinterpret_cast<const uint2 *>(p.bias + min(col, p.n - 4)) : make_uint2(0, 0);
}
__device__ __forceinline__ void widen(const uint2 &v, float f[4])
{
    f[0] = __uint_as_float(v.x << 16);
    f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16);
    f[3] = __uint_as_float(v.y & 0xffff0000u);
}

// rows16 of bytes.
__device__ __forceinline__ void rows16_bytes(const uint32_t v[4], uint2 &lo, uint2 &hi)
{
    const auto first = __builtin_amdgcn_permlane32_swap(v[0], v[1], false, false);
    const auto second = __builtin_amdgcn_permlane32_swap(v[2], v[3], false, false);
    const auto a = __builtin_amdgcn_permlane16_swap(first[0], second[0], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(first[1], second[1], false, false);
    lo = make_uint2(a[0], b[0]), hi = make_uint2(a[1], b[1]);
}

template <bool GELU>
__global__ void __launch_bounds__(kBigWaves * 64, 1) big_kernel(Fp8Params p)
{
    constexpr int MT = 4, NT = 4;
    __shared__ __attribute__((aligned(1024))) char smem[kBigLds];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int l32 = lane & 31, half = lane >> 5;
    const int wm = (wave >> 1) * 128, wn = (wave & 1) * 128;  // this wave's rows
    const int xcd = blockIdx.x & 7, units = units_of(p, xcd);
    int j = blockIdx.x >> 3;
    if (j >= units) return;

    const u32x4 xr = whole_memory(p.x), wr = whole_memory(p.w), xsr = whole_memory(p.xs), wsr = whole_memory(p.ws);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)smem));
    // Load c of a step: rows (4 c + wave) * 8 .. + 7 of the tile's x and w together, and rows
    // 64 wave .. of x's scales and of w's.  Rows past the last repeat it; their results
    // are not stored.
    uint32_t at[kBigLoads], at_s[2];
    const int first_row = wave * 8 + (lane >> 3);
    const uint32_t chunk = chunk_pos(first_row, lane & 7) * 16;  // the same 32 rows on
    auto address = [&](const Unit &u) {
#pragma unroll
        for (int c = 0; c < kBigLoads; ++c) {
            const int row = first_row + c * kBigWaves * 8;
            const int r = c * kBigWaves * 8 < kBig ? min(u.m0 + row, p.m - 1) : min(u.n0 + row - kBig, p.n - 1);
            at[c] = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.kp) + chunk;
        }
        at_s[0] = static_cast<uint32_t>(min(u.m0 + wave * 64 + lane, p.m - 1)) * 4;
        at_s[1] = static_cast<uint32_t>(min(u.n0 + wave * 64 + lane, p.n - 1)) * 4;
    };
    // of step `abs` of K, into places `deep` and `near` of the rings
    auto load = [&](int abs, int c, int deep, int near) {
        const int to = c < kDeepLoads ? deep * kDeepBytes + c * kBigWaves * 1024
                                      : kNearAt + near * kNearBytes + (c - kDeepLoads) * kBigWaves * 1024;
        load_lds16(c * kBigWaves * 8 < kBig ? xr : wr, __builtin_amdgcn_readfirstlane(lds0 + to + wave * 1024), at[c],
                   __builtin_amdgcn_readfirstlane(abs * kFp8Block));
    };
    auto load_scales = [&](int abs, int c, int deep) {
        load_lds4(c ? wsr : xsr,
                  __builtin_amdgcn_readfirstlane(lds0 + kScalesAt + deep * kScaleBytes + c * kBig * 4 + wave * 256), at_s[c],
                  __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(abs >> 2) * (c ? p.n : p.m) * 4));
    };

    int off[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) off[s] = l32 * 128 + chunk_pos(l32, 2 * s + half) * 16;
    // A row's place in LDS as deep * DEEP + near * NEAR + c: rows of this wave's first 64 of x are
    // deep (0 and 128), those of w near, the other 64 of x (64 and 192) one or the other.
    const bool x1_deep = wm + 64 < kDeepRows;
    const int x1_d = x1_deep ? kDeepBytes : 0, x1_n = x1_deep ? 0 : kNearBytes;
    const int x1_c = x1_deep ? (wm + 64) * 128 : kNearAt + (wm + 64 - kDeepRows) * 128;
    auto x0_at = [&](int deep) { return deep * kDeepBytes + wm * 128; };
    auto x1_at = [&](int deep, int near) { return deep * x1_d + near * x1_n + x1_c; };
    auto w_at = [&](int near) { return kNearAt + near * kNearBytes + (kBig + wn - kDeepRows) * 128; };
    // Fragments of a half step (64 values): x's in two sets, w's in one whose second half is
    // read while the first is multiplied.
    i32x8 xf[2][MT], wf[NT];
    int xs[MT], ws[NT], xs_next[MT], ws_next[NT];  // scales of this step and the next
    auto fragment = [&](int base, int s) {
        const i32x4 *lo = reinterpret_cast<const i32x4 *>(smem + base + off[2 * s]);
        const i32x4 *hi = reinterpret_cast<const i32x4 *>(smem + base + off[2 * s + 1]);
        return cat(*lo, *hi);
    };
    const int scale_row = kScalesAt + (wm + l32) * 4, scale_row_w = kScalesAt + (kBig + wn + l32) * 4;
    auto read_scale = [&](int t, int abs, int deep) {
        const char *s = smem + deep * kScaleBytes + (abs & 3);
        if (t < MT)
            xs_next[t] = *reinterpret_cast<const uint8_t *>(s + scale_row + t * 128);
        else
            ws_next[t - MT] = *reinterpret_cast<const uint8_t *>(s + scale_row_w + (t - MT) * 128);
    };

    Unit u = unit_at(p, xcd, j);
    address(u);
    for (int i = 0; i < 2; ++i) {  // a unit has two steps at least
#pragma unroll
        for (int c = 0; c < 2; ++c) load_scales(u.first + i, c, i);
#pragma unroll
        for (int c = 0; c < kBigLoads; ++c) load(u.first + i, c, i, i);
    }
    step_barrier<kBigLoads + 2>(true);
    int deep = 0, near = 0;
#pragma unroll
    for (int t = 0; t < MT + NT; ++t) read_scale(t, u.first, 0);
#pragma unroll
    for (int t = 0; t < MT; ++t) xf[0][t] = fragment((t < 2 ? x0_at(0) : x1_at(0, 0)) + (t & 1) * 4096, 0);
#pragma unroll
    for (int t = 0; t < 2; ++t) wf[t] = fragment(w_at(0) + t * 4096, 0);

    f32x16 acc[MT][NT];
    // One step: 32 products a wave.  Between them, of the step after it the scales (`next`
    // says which of their four bytes) and the first fragments are read, and step `ahead` of
    // the address is loaded, two further on.  No branch inside: the compiler would move the
    // products past it.
    auto step = [&](int next, int ahead) __attribute__((always_inline)) {
        const int deep1 = deep == 2 ? 0 : deep + 1, deep2 = deep1 == 2 ? 0 : deep1 + 1;
        const int x0 = x0_at(deep), x1 = x1_at(deep, near), w0 = w_at(near);
        const int x0n = x0_at(deep1), x1n = x1_at(deep1, near ^ 1), w0n = w_at(near ^ 1);
#pragma unroll
        for (int t = 0; t < MT; ++t) xs[t] = xs_next[t];
#pragma unroll
        for (int t = 0; t < NT; ++t) ws[t] = ws_next[t];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < MT * NT; ++e) {
                if (e < 2) wf[2 + e] = fragment(w0 + (2 + e) * 4096, s);
                if (s == 1 && e == 3) {
                    // the next step is there but for what this one's first half has issued, and all
                    // waves have read this one whole
                    step_barrier<kDeepLoads + 2>(true);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (e >= 4 && e < 16 && e % 2 == 0) {
                    const int t = (e - 4) / 2;
                    if (t < MT)
                        xf[s ^ 1][t] = fragment((s == 0 ? (t < 2 ? x0 : x1) : (t < 2 ? x0n : x1n)) + (t & 1) * 4096, s ^ 1);
                    else
                        wf[t - MT] = fragment((s == 0 ? w0 : w0n) + (t - MT) * 4096, s ^ 1);
                }
                if (s == 0 && e % 2 == 1) {
                    const int c = e / 2;
                    if (c < 2)
                        load_scales(ahead, c, deep2);
                    else
                        load(ahead, c - 2, deep2, near);
                }
                if (s == 1 && e >= 4 && e - 4 < kNearLoads) load(ahead, kDeepLoads + e - 4, deep2, near);
                if (s == 1 && e >= 5 && e - 5 < MT + NT) read_scale(e - 5, next, deep1);
                const int ni = e / MT, mi = e % MT;
                acc[mi][ni] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[ni], xf[s][mi], acc[mi][ni], 0, 0, 0,
                                                                             ws[ni], 0, xs[mi]);
                __builtin_amdgcn_sched_barrier(0);
            }
        deep = deep1, near ^= 1;
    };

    for (;;) {
#pragma unroll
        for (int mi = 0; mi < MT; ++mi)
#pragma unroll
            for (int ni = 0; ni < NT; ++ni) acc[mi][ni] = f32x16{};
        const Unit done = u;
        bool more = true;
        int ahead = u.first + 2, next = u.first + 1;
        for (int left = done.n; left > 0; --left) {
            if (left == 2) {  // the loads go on in the next unit; past the last one they repeat it unread
                j += kCus;
                more = j < units;
                if (more) u = unit_at(p, xcd, j);
                address(u);
                ahead = u.first;
            }
            if (left == 1) next = u.first;
            step(next, ahead);
            ++ahead, ++next;
        }

        // acc[i][j]: lane l holds row 32 i + l % 32 of x; register r row 32 j + 8 (r/4) + 4 half + r % 4 of w
        const int m0 = done.m0 + wm, n0 = done.n0 + wn;
        settle();
        if (done.part >= 0) {
            float *sums = p.part + (static_cast<int64_t>(done.part) * p.rest + done.tile - p.whole) * (kBig * kBig);
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = taken(acc[mi][ni][4 * q + e]);
                        *reinterpret_cast<f32x4 *>(sums + (wm + mi * 32 + l32) * kBig + wn + ni * 32 + 8 * q + 4 * half) = v;
                    }
        } else if constexpr (!GELU) {
            uint2 b[NT][4];
#pragma unroll
            for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                for (int q = 0; q < 4; ++q) b[ni][q] = bias4(p, n0 + ni * 32 + 8 * q + 4 * half);
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) {
#pragma unroll
                for (int ni = 0; ni < NT; ++ni) {
                    uint32_t v[4][2];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float f[4], c[4];
                        widen(b[ni][q], c);
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = taken(acc[mi][ni][4 * q + e]) + c[e];
                        v[q][0] = pack_bf16x2(f[0], f[1]);
                        v[q][1] = pack_bf16x2(f[2], f[3]);
                    }
                    u32x4 lo, hi;
                    rows16(v, lo, hi);
                    const int row = m0 + mi * 32 + (lane & 15), col = n0 + ni * 32 + 8 * half + (lane & 16);
                    if (row < p.m && col < p.n)
                        *reinterpret_cast<u32x4 *>(p.y + static_cast<int64_t>(row) * p.n + col) = lo;
                    if (row + 16 < p.m && col < p.n)
                        *reinterpret_cast<u32x4 *>(p.y + static_cast<int64_t>(row + 16) * p.n + col) = hi;
                }
            }
        } else {
            // GELU, and each row's 128 columns, a block
            const int block = n0 / kFp8Block, last = p.np / kFp8Block - 1;
            uint2 bias[NT][4];
#pragma unroll
            for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                for (int q = 0; q < 4; ++q) bias[ni][q] = bias4(p, n0 + ni * 32 + 8 * q + 4 * half);
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) {
                float g[NT][16], top = 0.f;
#pragma unroll
                for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float b[4];
                        widen(bias[ni][q], b);
#pragma unroll
                        for (int e = 0; e < 4; ++e) g[ni][4 * q + e] = gelu(taken(acc[mi][ni][4 * q + e]) + b[e]);
                    }
                if (n0 + 128 > p.n)  // past the last column zeros
#pragma unroll
                    for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (n0 + ni * 32 + 8 * (r >> 2) + 4 * half >= p.n) g[ni][r] = 0.f;
                // a NaN comes out of the maximum, so that its block is NaN as a whole
#pragma unroll
                for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                    for (int r = 0; r < 16; ++r) top = __builtin_elementwise_maximum(top, fabsf(g[ni][r]));
                const uint32_t t = magnitude(top);
                const auto both = __builtin_amdgcn_permlane32_swap(t, t, false, false);
                const uint32_t scale = fp8_scale(max(static_cast<uint32_t>(both[0]), static_cast<uint32_t>(both[1])));
                const float inv = fp8_inverse(scale == 255 ? 127 : scale);
#pragma unroll
                for (int ni = 0; ni < NT; ++ni) {
                    uint32_t v[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float *f = &g[ni][4 * q];
                        v[q] = scale == 255 ? 0x7f7f7f7fu : fp8_pack4(f[0], f[1], f[2], f[3], inv);
                    }
                    uint2 lo, hi;
                    rows16_bytes(v, lo, hi);
                    const int row = m0 + mi * 32 + (lane & 15), col = n0 + ni * 32 + 8 * half + (lane & 16);
                    if (row < p.m && block <= last) *reinterpret_cast<uint2 *>(p.q + static_cast<int64_t>(row) * p.np + col) = lo;
                    if (row + 16 < p.m && block <= last)
                        *reinterpret_cast<uint2 *>(p.q + static_cast<int64_t>(row + 16) * p.np + col) = hi;
                }
                const int row = m0 + mi * 32 + l32;
                const bool in = row < p.m && block <= last;
                // the last block's lane also fills its group
                if (in && half == 0)
                    for (int b = block; b == block || (block == last && b <= (last | 3)); ++b)
                        p.qs[(static_cast<int64_t>(b >> 2) * p.m + row) * 4 + (b & 3)] = b == block ? static_cast<uint8_t>(scale) : 0;
            }
        }
        if (!more) break;
    }
    step_barrier<0>(true);  // no load may write LDS that is no longer this workgroup's
}

// Adds the parts of the cut tiles in their order, then the bias, and rounds, or makes
// blocks: 8 columns a thread, 16 neighbouring lanes a block.
template <int TILE, bool GELU>
__global__ void __launch_bounds__(256) tile_sum_kernel(Fp8Params p)
{
    constexpr int kPer = TILE * TILE / 8 / 256;  // workgroups a tile
    const int t = blockIdx.x / kPer, i = (blockIdx.x % kPer * 256 + threadIdx.x) * 8;
    int m0, n0;
    tile_rows<TILE, TILE>(p.tiles_m, p.tiles_n, p.whole + t, m0, n0);
    const int row = m0 + i / TILE, col = n0 + i % TILE;
    if (row >= p.m || col >= (GELU ? p.np : p.n)) return;  // whole blocks of lanes
    float f[8] = {};
    if (col < p.n) {
        const float *s = p.part + static_cast<int64_t>(t) * (TILE * TILE) + i;
        f32x4 lo = {}, hi = {};
        for (int k = 0; k < p.parts; ++k, s += static_cast<int64_t>(p.rest) * (TILE * TILE)) {
            lo += *reinterpret_cast<const f32x4 *>(s);
            hi += *reinterpret_cast<const f32x4 *>(s + 4);
        }
        float b[8] = {};
        if (p.bias) unpack8v(*reinterpret_cast<const u32x4 *>(p.bias + col), b);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = lo[e] + b[e];
            f[4 + e] = hi[e] + b[4 + e];
        }
        if constexpr (GELU)
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = gelu(f[e]);
    }
    if constexpr (!GELU) {
        *reinterpret_cast<u32x4 *>(p.y + static_cast<int64_t>(row) * p.n + col) = pack8v(f);
    } else {
        uint32_t scale;
        *reinterpret_cast<uint2 *>(p.q + static_cast<int64_t>(row) * p.np + col) = fp8_quantize8(f, scale);
        const int block = col / kFp8Block, last = p.np / kFp8Block - 1;
        if (threadIdx.x & 15) return;
        for (int b = block; b == block || (block == last && b <= (last | 3)); ++b)
            p.qs[(static_cast<int64_t>(b >> 2) * p.m + row) * 4 + (b & 3)] = b == block ? static_cast<uint8_t>(scale) : 0;
    }
}

// ------------------------------------------------------------------ few rows --
// 32 * MT rows of x and 32 * NT of w a workgroup.  Each of its four waves takes every fourth
// block of K, through LDS of its own (so that the loads read whole rows of 128 bytes; straight
// to registers a load of 16 lanes touches 16 rows), RING blocks ahead and without a barrier;
// their sums are added in LDS at the end.  With GELU two waves take the 128 columns of a block side
// by side and every second block of K, so that the blocks of the result are made there, too.
constexpr int kFewWaves = 4;

// X16: x is bf16, and each workgroup quantises its rows of it into LDS while its first loads of w
// are on their way: for rows of at most kInline bytes there (a launch less).
constexpr int kInline = 17408;  // with the ring a third of LDS
// In LDS, 16 bytes of each lane, then a gap: 4 rows' 16 chunks of 8 columns cover the banks.
constexpr int kSumsRow = 68;

template <int MT_, int NT_, int RING_, bool X16_ = false, bool GELU_ = false>
struct Few {
    static constexpr int MT = MT_, NT = NT_, RING = RING_;
    static constexpr bool X16 = X16_, GELU = GELU_;
    static constexpr int over_n = GELU ? 2 : 1, over_k = kFewWaves / over_n;  // waves
    static constexpr int loads = X16 ? 4 * NT + 1 : 4 * (MT + NT) + 2;  // of a block: 8 rows each, and the scales
    static constexpr int w_at = X16 ? 0 : MT * 4096, scales_at = w_at + NT * 4096, bytes = scales_at + (X16 ? 256 : 512);
    static constexpr int ring = RING * bytes * kFewWaves, sums = kFewWaves * MT * NT * 4 * kSumsRow * 16;
    static constexpr int x_at = ring > sums ? ring : sums, lds = x_at + (X16 ? kInline : 0);
    static_assert(!GELU || (MT == 1 && NT == 2 && !X16), "32 rows of one block");
    static_assert(MT <= 2 && NT <= 2 && loads * (RING - 1) < 64, "a load takes 64 rows of scales, a wait counts to 63");
};

// x in LDS: rows of the values, 16 bytes apart from a multiple of 128 (so that 32 rows cover
// the banks), then rows of the scales.
__host__ __device__ inline int64_t inline_bytes(int64_t rows, int64_t kp) { return rows * (kp + 16 + kp / kFp8Block); }

// This wave's loads but the newest `n` have landed.
__device__ __forceinline__ void wait_loads(int n)
{
    asm volatile("" ::: "memory");
    switch (n) {
#define LTXK_WAIT(N) case N: __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4 << 14)); break;
    LTXK_WAIT(5)
    LTXK_WAIT(10)
    LTXK_WAIT(14)
    LTXK_WAIT(18)
    LTXK_WAIT(28)
#undef LTXK_WAIT
    default: __builtin_amdgcn_s_waitcnt(0x0f70);
    }
    asm volatile("" ::: "memory");
}

template <typename F, bool SUMS>
__global__ void __launch_bounds__(kFewWaves * 64) few_kernel(Fp8Params p)
{
    constexpr int MT = F::MT, NT = F::NT, R = F::RING;
    __shared__ __attribute__((aligned(1024))) char smem[F::lds];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int l32 = lane & 31, half = lane >> 5;
    // a tile of w goes to one XCD for all tiles of x, and all parts of a tile, too
    const int at_x = blockIdx.x >> 3;
    const int tn = at_x / p.tiles_m / p.parts * 8 + (blockIdx.x & 7), tm = at_x % p.tiles_m, part = at_x / p.tiles_m % p.parts;
    if (tn >= p.tiles_n) return;
    const int wn = wave % F::over_n, wk = wave / F::over_n;
    const int m0 = tm * 32 * MT, n0 = (tn * F::over_n + wn) * 32 * NT;
    // blocks of this part, then this wave's of them
    const int from = static_cast<int>(static_cast<uint32_t>(part) * p.blocks / p.parts);
    const int to = static_cast<int>(static_cast<uint32_t>(part + 1) * p.blocks / p.parts);
    const int first = from + wk, n = max(0, (to - first + F::over_k - 1) / F::over_k);

    const u32x4 xr = whole_memory(p.x), wr = whole_memory(p.w), xsr = whole_memory(p.xs), wsr = whole_memory(p.ws);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)smem)) + wave * R * F::bytes;
    // rows past the last repeat it; their results are not stored
    uint32_t xo[4 * MT], wo[4 * NT];
    const uint32_t chunk = chunk_pos(lane >> 3, lane & 7) * 16, chunk_odd = chunk_pos(8 + (lane >> 3), lane & 7) * 16;
#pragma unroll
    for (int c = 0; c < 4 * MT; ++c)
        xo[c] = static_cast<uint32_t>(min(m0 + c * 8 + (lane >> 3), p.m - 1)) * static_cast<uint32_t>(p.kp) + (c & 1 ? chunk_odd : chunk);
#pragma unroll
    for (int c = 0; c < 4 * NT; ++c)
        wo[c] = static_cast<uint32_t>(min(n0 + c * 8 + (lane >> 3), p.n - 1)) * static_cast<uint32_t>(p.kp) + (c & 1 ? chunk_odd : chunk);
    const uint32_t xso = static_cast<uint32_t>(min(m0 + lane, p.m - 1)) * 4, wso = static_cast<uint32_t>(min(n0 + lane, p.n - 1)) * 4;
    auto load = [&](int i, int slot) {
        const int b = first + i * F::over_k;
        const uint32_t at = lds0 + slot * F::bytes;
        const uint32_t k = __builtin_amdgcn_readfirstlane(b * kFp8Block), g = __builtin_amdgcn_readfirstlane(b >> 2);
#pragma unroll
        for (int c = 0; c < 4 * NT; ++c) load_lds16(wr, __builtin_amdgcn_readfirstlane(at + F::w_at + c * 1024), wo[c], k);
        load_lds4(wsr, __builtin_amdgcn_readfirstlane(at + F::scales_at), wso, __builtin_amdgcn_readfirstlane(g * p.n * 4));
        if constexpr (!F::X16) {
#pragma unroll
            for (int c = 0; c < 4 * MT; ++c) load_lds16(xr, __builtin_amdgcn_readfirstlane(at + c * 1024), xo[c], k);
            load_lds4(xsr, __builtin_amdgcn_readfirstlane(at + F::scales_at + 256), xso, __builtin_amdgcn_readfirstlane(g * p.m * 4));
        }
    };
    for (int i = 0; i < R && i < n; ++i) load(i, i);
    const int rows = min(32, p.m - m0);
    char *xl = smem + F::x_at, *xsl = xl + rows * (p.kp + 16);
    if constexpr (F::X16) {
        // a block 16 lanes, as quantize_fp8; the loads of kBatch blocks together
        constexpr int kBatch = 4, kStride = kFewWaves * 4;
        const int units = rows * p.blocks;
        for (int u0 = threadIdx.x >> 4; u0 < units; u0 += kBatch * kStride) {
            u32x4 raw[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {  // past the last: read again, not stored
                const int u = min(u0 + i * kStride, units - 1), row = u / p.blocks, col = u % p.blocks * kFp8Block + (lane & 15) * 8;
                raw[i] = *reinterpret_cast<const u32x4 *>(p.x16 + static_cast<int64_t>(m0 + row) * p.k + min(col, p.k - 8));
                if (col >= p.k) raw[i] = u32x4{};
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int u = u0 + i * kStride, row = u / p.blocks, b = u % p.blocks;
                float f[8];
                unpack8v(raw[i], f);
                uint32_t scale;
                const uint2 q = fp8_quantize8(f, scale);
                if (u >= units) continue;
                *reinterpret_cast<uint2 *>(xl + row * (p.kp + 16) + b * kFp8Block + (lane & 15) * 8) = q;
                if ((lane & 15) == 0) xsl[u] = static_cast<char>(scale);
            }
        }
        __syncthreads();
        xl += min(l32, rows - 1) * (p.kp + 16) + half * 16;
        xsl += min(l32, rows - 1) * p.blocks;
    }

    int off[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) off[s] = l32 * 128 + chunk_pos(l32, 2 * s + half) * 16;
    f32x16 acc[MT][NT] = {};
    int slot = 0;
    for (int i = 0; i < n; ++i) {
        wait_loads(min(R - 1, n - 1 - i) * F::loads);
        const char *at = smem + (wave * R + slot) * F::bytes;
        i32x8 f[2][MT + NT];
        int scale[MT + NT];
        const int b = first + i * F::over_k;
        if constexpr (F::X16) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
                f[s][0] = cat(*reinterpret_cast<const i32x4 *>(xl + b * kFp8Block + s * 64),
                              *reinterpret_cast<const i32x4 *>(xl + b * kFp8Block + s * 64 + 32));
            scale[0] = static_cast<uint8_t>(xsl[b]);
        }
#pragma unroll
        for (int t = F::X16 ? MT : 0; t < MT + NT; ++t) {
            const char *tile = t < MT ? at + t * 4096 : at + F::w_at + (t - MT) * 4096;
#pragma unroll
            for (int s = 0; s < 2; ++s)
                f[s][t] = cat(*reinterpret_cast<const i32x4 *>(tile + off[2 * s]),
                              *reinterpret_cast<const i32x4 *>(tile + off[2 * s + 1]));
            scale[t] = *reinterpret_cast<const uint8_t *>(at + F::scales_at + (t < MT ? 256 + t * 128 : (t - MT) * 128) + l32 * 4 + (b & 3));
        }
        // read whole: its place goes to block i + R
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        asm volatile("" ::: "memory");
        if (i + R < n) load(i + R, slot);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int ni = 0; ni < NT; ++ni)
#pragma unroll
                for (int mi = 0; mi < MT; ++mi)
                    acc[mi][ni] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(f[s][MT + ni], f[s][mi], acc[mi][ni], 0, 0, 0,
                                                                                 scale[MT + ni], 0, scale[mi]);
        slot = slot + 1 == R ? 0 : slot + 1;
    }

    // lane l: row l % 32 of x, rows 8 q + 4 (l / 32) .. + 3 of w in registers 4 q ..
    __syncthreads();  // all waves are done with their places
    f32x4 *sums = reinterpret_cast<f32x4 *>(smem);
#pragma unroll
    for (int t = 0; t < MT * NT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x16 &a = acc[t / NT][t % NT];
            sums[((wave * MT * NT + t) * 4 + q) * kSumsRow + lane] = f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
        }
    __syncthreads();
    if constexpr (F::GELU) {
        // 8 columns a lane, a row's block 16 lanes
        const int col = tn * kFp8Block + (lane & 15) * 8;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = i * 16 + wave * 4 + (lane >> 4), row = m0 + at;
            float v[8] = {};
            if (col < p.n) {
                f32x4 lo = {}, hi = {};
#pragma unroll
                for (int w = 0; w < F::over_k; ++w) {
                    // of the wave that holds these columns: its tile, and four times 8 columns there
                    const f32x4 *s = sums + (w * F::over_n * NT * 4 + (lane & 15)) * kSumsRow + at;
                    lo += s[0], hi += s[32];
                }
                float b[8] = {};
                if (p.bias) unpack8v(*reinterpret_cast<const u32x4 *>(p.bias + col), b);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = gelu((e < 4 ? lo[e] : hi[e - 4]) + b[e]);
            }
            uint32_t scale;
            const uint2 q = fp8_quantize8(v, scale);
            if (row >= p.m) continue;
            *reinterpret_cast<uint2 *>(p.q + static_cast<int64_t>(row) * p.np + col) = q;
            if (lane & 15) continue;
            for (int b = tn; b == tn || (tn == p.tiles_n - 1 && b <= (tn | 3)); ++b)  // the last block's lane fills its group
                p.qs[(static_cast<int64_t>(b >> 2) * p.m + row) * 4 + (b & 3)] = b == tn ? static_cast<uint8_t>(scale) : 0;
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < MT * NT; ++t) {  // this wave's q of each tile
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) v += sums[((w * MT * NT + t) * 4 + wave) * kSumsRow + lane];
        const int row = m0 + t / NT * 32 + l32, col = n0 + t % NT * 32 + 8 * wave + 4 * half;
        if (row >= p.m || col >= p.n) continue;
        if constexpr (SUMS) {
            *reinterpret_cast<f32x4 *>(p.part + (static_cast<int64_t>(part) * p.m + row) * p.np + col) = v;
        } else {
            if (p.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += bf16_to_f32(p.bias[col + e]);
            *reinterpret_cast<uint2 *>(p.y + static_cast<int64_t>(row) * p.n + col) =
                make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        }
    }
}

// Adds the parts of a cut K in their order, then the bias, and rounds, or makes blocks
// of the GELU: 8 columns a thread, 16 neighbouring lanes a block, as quantize_fp8.
template <bool GELU>
__global__ void __launch_bounds__(256) few_sum_kernel(Fp8Params p)
{
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, row = static_cast<int>(unit % p.m);
    const int group = static_cast<int>(unit / p.m), col = group * 512 + lane * 8;
    if (group * 512 >= p.np) return;
    float f[8] = {};
    if (col < p.n) {
        const float *s = p.part + static_cast<int64_t>(row) * p.np + col;
        f32x4 lo = {}, hi = {};
        for (int k = 0; k < p.parts; ++k, s += static_cast<int64_t>(p.m) * p.np) {
            lo += *reinterpret_cast<const f32x4 *>(s);
            hi += *reinterpret_cast<const f32x4 *>(s + 4);
        }
        float b[8] = {};
        if (p.bias) unpack8v(*reinterpret_cast<const u32x4 *>(p.bias + col), b);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = lo[e] + b[e];
            f[4 + e] = hi[e] + b[4 + e];
        }
        if constexpr (GELU)
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = gelu(f[e]);
        else
            *reinterpret_cast<u32x4 *>(p.y + static_cast<int64_t>(row) * p.n + col) = pack8v(f);
    }
    if constexpr (GELU) {
        uint32_t scale;
        const uint2 q = fp8_quantize8(f, scale);
        if (col < p.np) *reinterpret_cast<uint2 *>(p.q + static_cast<int64_t>(row) * p.np + col) = q;
        if ((lane & 15) == 0)
            p.qs[(static_cast<int64_t>(group) * p.m + row) * 4 + (lane >> 4)] = static_cast<uint8_t>(scale);
    }
}

template <typename F>
void few_rows(const Fp8Params &p, bool gelu, hipStream_t s)
{
    const unsigned grid = 8u * static_cast<unsigned>((p.tiles_n + 7) / 8) * static_cast<unsigned>(p.tiles_m) * static_cast<unsigned>(p.parts);
    if constexpr (F::GELU) {
        few_kernel<F, false><<<grid, kFewWaves * 64, 0, s>>>(p);
    } else if (gelu || p.parts > 1) {
        few_kernel<F, true><<<grid, kFewWaves * 64, 0, s>>>(p);
        const unsigned sums = static_cast<unsigned>((static_cast<int64_t>(p.m) * ((p.np + 511) / 512) + 3) / 4);
        if (gelu)
            few_sum_kernel<true><<<sums, 256, 0, s>>>(p);
        else
            few_sum_kernel<false><<<sums, 256, 0, s>>>(p);
    } else {
        few_kernel<F, false><<<grid, kFewWaves * 64, 0, s>>>(p);
    }
}

// The kernel that a product takes, and how it is cut over K.
//
// Few rows: up to 32, and outputs of at most 256 tiles of 64 x 64, one a compute unit; tiles of 64 x
// 32, or 32 x 32, where those are at most 256, too.  Cold operands, this kernel / 128 x 128 tiles, us,
// M x N x K: 126 x 2048 x 2048 6 / 15, 126 x 2048 x 8192 13 / 19, 126 x 8192 x 2048 11 / 19, 504 x
// 2048 x 8192 21 / 25, 256 x 4096 x 4096 15 / 22;  512 tiles, 512 x 4096 x 4096 25 / 25;  1024, 504 x
// 8192 x 2048 32 / 17.  32 x 32 / 64 x 32 / 64 x 64 tiles: 126 x 2048 x 2048 6 / 7 / 9, 252 x 2048 x
// 2048 - / 7 / 9.
// K is cut from 128 blocks on where the tiles leave units idle, into parts of at least 16; the
// second launch costs 5 us: 1 x 1024 x 16384 19 us whole, 12 in 8 parts; 126 x 1024 x 16384 28 and
// 17; 16 x 4096 x 16384 25 and 26.
//
// With GELU few rows take a second launch, which makes the blocks of sums in memory, or tiles of 32 x 128
// that make them themselves, where these are not too few for their K (blocks of it times 6) nor take
// longer than 32 blocks of K in turn.  Us, with the second launch / one: 126 x 8192 x 2048 13.3 / 10.9, 252 x
// 4096 x 4096 18.2 / 16.3, 504 x 4096 x 2048 22.3 / 18.3, 8 x 2048 x 256 5.0 / 3.9;  too few, 126 x 2048 x 2048 7.5 /
// 8.8, 126 x 4096 x 4096 14.2 / 16.3;  too long, 504 x 4096 x 4096 24.0 / 29.1, 504 x 8192 x 2048 19 / 35.
struct Cut {
    int tile, tile_n;  // rows of x and of w; few rows: 32, 48 (64 and 32) and 64
    bool fused;  // few rows with GELU: tiles of 32 x 128, the result's blocks made there
    int64_t tiles_m, tiles_n, whole, rest, parts;
};

Cut cut(int64_t m, int64_t n, int64_t k, bool gelu)
{
    Cut c{};
    const int64_t blocks = fp8_blocks(k), tiles64 = (m + 63) / 64 * ((n + 63) / 64);
    c.parts = 1;
    c.tiles_m = (m + 31) / 32;
    c.tiles_n = fp8_blocks(n);
    const int64_t tiles = c.tiles_m * c.tiles_n;
    if (gelu && tiles <= 512 && (tiles + 255) / 256 * blocks <= 32 && tiles >= 6 * blocks) {
        c.tile = 32;
        c.fused = true;
        return c;
    }
    if (m <= 32 || tiles64 <= 256) {
        const int mt = m <= 32 || tiles64 <= 64 ? 1 : 2, nt = m <= 32 || tiles64 <= 128 ? 1 : 2;
        c.tile = 16 * (mt + nt);
        c.tiles_m = (m + 32 * mt - 1) / (32 * mt);
        c.tiles_n = (n + 32 * nt - 1) / (32 * nt);
        if (blocks >= 128)
            while (c.tiles_m * c.tiles_n * c.parts * 2 <= 256 && blocks >= c.parts * 2 * 16) c.parts *= 2;
        return c;
    }
    // Tiles: the kind whose rounds of the chip take least, at 4, 6 and 7 for one of 128 x 128, 256 x
    // 128 and 256 x 256 (a round of K 4096: 24, 37 and 41 us).  128 x 128 / 256 x 128 / 256 x 256, us, M x N x K: 1024 x 4096 x
    // 4096 25 / 32 / -, 2048 x 4096 x 4096 44 / 38 / 49, 1500 x 4096 x 2048 32 / 24 / -, 2304 x 4096 x
    // 4096 59 / 54 / 42, 4290 x 2048 x 4096 53 / 51 / 40.  Those past the last full round are
    // dealt to its units in parts of K where that saves more than it takes.  Two parts / whole: 1024 x 2048 x 2048
    // 22.6 / 13.3, 6144 x 4096 x 2048 68 / 55, 6144 x 4096 x 4096 100 / 96, 777 x 2048 x 4096 22 / 23, 1024 x 1536 x
    // 8192 29 / 40;  four / whole: 4290 x 4096 x 4096 74 / 88.
    c.tile = c.tile_n = kTile;
    auto rounds = [&](int tm, int tn) { return ((m + tm - 1) / tm * ((n + tn - 1) / tn) + 255) / 256; };
    int64_t least = 4 * rounds(kTile, kTile);
    if (6 * rounds(kBig, kTile) < least) least = 6 * rounds(kBig, kTile), c.tile = kBig;
    if (blocks > 1 && 7 * rounds(kBig, kBig) < least) c.tile = c.tile_n = kBig;
    c.tiles_m = (m + c.tile - 1) / c.tile;
    c.tiles_n = (n + c.tile_n - 1) / c.tile_n;
    c.rest = c.tiles_m * c.tiles_n % 256;
    c.whole = c.tiles_m * c.tiles_n - c.rest;
    if (c.rest && c.tile == c.tile_n) {  // the least of 256 x 128, over 256 of 128 x 128, leave no unit two
        // what the parts save of a tile's steps (us), less what their sums take: a launch, written and read
        const double step = c.tile == kBig ? 1.3 : 0.75, sums = 2.0 * c.tile * c.tile * 4 * 1e-6 / 4;
        double most = 0;
        for (int64_t p = 2; p <= 256 / c.rest && p * 4 <= blocks; ++p) {
            const double saved = step * static_cast<double>(blocks) * (1.0 - 1.0 / static_cast<double>(p)) - 3.0 -
                                 sums * static_cast<double>(c.rest * p);
            if (saved > most) most = saved, c.parts = p;
        }
    }
    return c;
}

int64_t workspace_bytes(int64_t m, int64_t n, int64_t k, bool gelu)
{
    const Cut c = cut(m, n, k, gelu);
    if (c.tile >= kTile) return c.parts > 1 ? c.rest * c.parts * c.tile * c.tile * 4 : 0;
    return (gelu && !c.fused) || c.parts > 1 ? c.parts * m * fp8_blocks(n) * kFp8Block * 4 : 0;
}

template <bool GELU>
void tiles(const Fp8Params &p, const Cut &c, hipStream_t s)
{
    const unsigned per = static_cast<unsigned>(p.whole / 8 + p.per);  // of an XCD
    const unsigned sums = p.parts > 1 ? static_cast<unsigned>(p.rest * c.tile * c.tile / 8 / 256) : 0;
    if (c.tile_n == kBig) {
        big_kernel<GELU><<<8 * std::min<unsigned>(kCus, per), kBigWaves * 64, 0, s>>>(p);
        if (sums) tile_sum_kernel<kBig, GELU><<<sums, 256, 0, s>>>(p);
    } else if (c.tile == kBig) {
        tile_kernel<kBig, GELU><<<8 * per, kTileWaves * 64, 0, s>>>(p);
    } else {
        tile_kernel<kTile, GELU><<<8 * per, kTileWaves * 64, 0, s>>>(p);
        if (sums) tile_sum_kernel<kTile, GELU><<<sums, 256, 0, s>>>(p);
    }
}

bool takes_bf16(const Cut &c, int64_t m, int64_t kp) { return c.tile == 32 && !c.fused && inline_bytes(std::min<int64_t>(m, 32), kp) <= kInline; }

// x's blocks, where the call makes them: values (a multiple of 128 bytes), then scales.
int64_t blocks_bytes(int64_t m, int64_t n, int64_t k, bool gelu)
{
    return takes_bf16(cut(m, n, k, gelu), m, fp8_blocks(k) * kFp8Block) ? 0 : m * fp8_blocks(k) * kFp8Block + (m * fp8_groups(k) * kFp8Group + 15) / 16 * 16;
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
    if (!y || (gelu && !y_scale) || !x || !w || !w_scale) return fail(LTXK_E_ARG, "%s: null operand", what);
    for (const void *v : {static_cast<const void *>(y), static_cast<const void *>(y_scale), x, x_scale, w, w_scale, bias})
        if (!aligned16(v)) return fail(LTXK_E_ALIGN, "%s: operands must be 16-byte aligned", what);
    // operands are read through 32-bit offsets, outputs counted by 32-bit tiles
    const int64_t kMax = int64_t{1} << 31;
    if (k >= kMax / 2 || n >= kMax / 2) return fail(LTXK_E_ARG, "%s: n or k of 2^30 or more", what);
    const int64_t kp = fp8_blocks(k) * kFp8Block, np = fp8_blocks(n) * kFp8Block;
    if (m > (kMax - 1) / kp || n > (kMax - 1) / kp || m > (kMax - 1) / np)
        return fail(LTXK_E_ARG, "%s: x, w or y holds 2^31 values or more", what);
    const Cut c = cut(m, n, k, gelu);
    const int64_t blocks_at = x_scale ? 0 : blocks_bytes(m, n, k, gelu), need = blocks_at + workspace_bytes(m, n, k, gelu);
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
    p.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + blocks_at);
    if (!x_scale && takes_bf16(c, m, kp)) {
        p.x16 = static_cast<const uint16_t *>(x);
    } else if (!x_scale) {
        char *q = static_cast<char *>(workspace), *q_scale = q + m * kp;
        const int rc = ltxk_quantize_fp8(q, q_scale, x, m, k, stream);
        if (rc) return rc;
        p.x = reinterpret_cast<const uint8_t *>(q);
        p.xs = reinterpret_cast<const uint8_t *>(q_scale);
    }
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.k = static_cast<int>(k);
    p.kp = static_cast<int>(kp);
    p.blocks = static_cast<int>(kp / kFp8Block);
    p.np = static_cast<int>(np);
    p.tiles_m = static_cast<int>(c.tiles_m);
    p.tiles_n = static_cast<int>(c.tiles_n);
    p.whole = static_cast<int>(c.whole);
    p.rest = static_cast<int>(c.rest);
    p.parts = static_cast<int>(c.parts);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (c.tile >= kTile) {
        p.per = static_cast<int>((c.rest * c.parts + 7) / 8);
        gelu ? tiles<true>(p, c, s) : tiles<false>(p, c, s);
    } else if (c.fused) {
        few_rows<Few<1, 2, 3, false, true>>(p, gelu, s);
    } else if (c.tile == 64) {
        few_rows<Few<2, 2, 2>>(p, gelu, s);
    } else if (c.tile == 48) {
        few_rows<Few<2, 1, 3>>(p, gelu, s);
    } else if (p.x16) {
        few_rows<Few<1, 1, 2, true>>(p, gelu, s);
    } else {
        few_rows<Few<1, 1, 2>>(p, gelu, s);
    }
    return check_launch(what);
}

}  // namespace
}  // namespace ltxk

using namespace ltxk;

extern "C" int64_t ltxk_linear_fp8_workspace_bytes(int64_t m, int64_t n, int64_t k, int gelu, int quantize)
{
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const int64_t kMax = int64_t{1} << 31;  // sizes that the calls refuse
    if (m >= kMax || n >= kMax || k >= kMax) return 0;
    return (quantize ? blocks_bytes(m, n, k, gelu != 0) : 0) + workspace_bytes(m, n, k, gelu != 0);
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
