// Attention of chunks over a paged bf16 cache on the 5th-generation tensor cores: rows whose new tokens fill more than a warp-level tile.
// The mathematics is that of attention_paged.cu.  An item is up to 256 query rows, tokens x heads of one KV head's group, in two tiles of 128:
//
//   S_g[128 rows][80 keys] = Q_g . K^T          both K-major in shared memory
//   O_g[128 rows][dim]    += P_g . V            P in tensor memory, V N-major in shared memory
//
//   warp 0       TMA producer: pages to tiles of 80 keys, K and V in turn, in a ring
//   warps 1, 2   MMA issue for tile 0 and tile 1
//   warps 4-7    softmax of tile 0, a thread per row;   warps 8-11   of tile 1
// Tiles are of 80 keys because scores (80 columns) and weights (40) of two tiles of rows then fit beside their sums of 128 dimensions in the 512
// columns of tensor memory: the scores of the next tile are made while the weights of this one are.  An MMA of 80 keys reads shared memory as fast as
// it goes (419 clocks for 128 rows, 512 for 128 keys: 1.3 of the time a key; with the sums 716 a tile of 80, 1.12).
// The weights of chunks enter rounded to bf16, half a step (2^-8) each and independent, which the sum over the keys averages: 2.3e-3 of the norm, where the
// output's own rounding is 1.66e-3.  A second term of what rounding left would take a second product with V, and tiles of 64 keys, so that both terms fit
// tensor memory: 4096 tokens behind 12288 took 1140 to 1170 us so for 915, six mixed rows 156 for 130, with the sums' error gone.  Items of up to 16 query rows, which
// alone would go to the warp-level kernel and its two terms, have both here too, at no product more: their rows lie twice among the 128 of a tile, the second
// time with the second term, and the two rows of sums are added (the six mixed rows 133.5 us for 130.5).  So a token's precision does not hang on who shares its batch.  The sum of the weights is that of the f32
// weights.  Scores, maxima, sums and O are f32.  The weights are relative to a maximum per row that moves only when a score exceeds it by 2^8; then O is
// rescaled in tensor memory.
//
// 4096 tokens behind 12288, 32 / 8 heads of 128: 0.78 to 0.92 ms, by the card and for how long it runs (the power cap): 1.05 PFLOP/s and more, 0.63 of cuBLAS in a burst and 0.75 of it sustained; 2048 behind
// 2048 116 us; six rows of 1 to 512 tokens behind up to 5000 122 to 134 us; 4096 behind 12288, 16 / 4 heads of 64, 0.39 ms.  A tile of 80 keys takes some 2300 clocks, of which both tiles'
// exponentials (2 x 128 x 80, at 16 a clock) need 1280 and the products 1432; no pipe is full (1024 behind 3000 by counters: exponentials 42 %, tensor pipe 42 %, issue
// slots 36 %).  What bounds it is the chain of a softmax warp: scores from tensor memory, the maximum, the last tile's products, exponentials, weights back.
//
// Measured and not kept, each against the kernel of its day: the tiles' exponentials in turns by a barrier 0.98 ms for 0.91; polynomials for a quarter of
// them 0.96 for 0.91.  Forms before this one: tiles of 128 keys with the weights over the scores (a chain of scores, softmax and sums) 0.98 to 1.02;
// an MMA warp a tile there, weights handed over in two or four parts, 1.08 and 1.11; tiles of 64 with two places for weights 1.17, with registers spilled.
//
// Over codes (e4m3 pages, 512 threads; see PcUnit for the numbers):
//   warp 0       producer: values as codes by bulk copies to a ring of their own, keys by TMA as the operand of an e4m3 product, with queries in two terms
//   warps 4-11   softmax, with the scales of keys on the scores and of values on the weights (f16)
//   warps 12-15  values from codes to f16, in the ring's slots
// In one run, bf16 pages in brackets: 4096 behind 12288 1.00 to 1.04 ms (0.78 to 0.88), six mixed rows 151 us (122), 1024 behind 1024 60 (51), 4096 behind 12288 of 16 / 4 heads of 64 0.52 ms (0.39);
// through a window of 1024 8000 tokens of 16 / 4 heads behind 5000 174 us (135).
// What it costs more, by copies that leave a part out: making values f16 45 us of 4096 behind 12288, the scales in the softmax 30 or so; the rest is not taken apart.
// Measured and not kept there: queries in one term (no faster, 2^-4), keys and values both made f16 by warps (1465 us; 1153 with the scales beside the softmax's), values loaded to
// registers a tile ahead and converted by unrolled code (1150: its text drives the softmax's out of the instruction cache), the next tile's table and scales asked for ahead (no change).
//
// An MMA multiplies a hidden value by a weight of 0, so an Inf or a NaN there would reach rows that do not see it.  Rows of a page behind the
// sequence's end are cleared in shared memory; a row whose sums come out as Inf or NaN (a later token's value may hold them) is computed
// again on CUDA cores over the keys in its sight, behind all pieces of the CTA, so that no bounded wait lasts as long as that.  Every wait on an mbarrier is bounded; on a time-out the CTA records AB2_ERR_TIMEOUT and
// walks through the rest of its work without waiting.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "tcgen05_util.cuh"

using namespace ab2;
using namespace ab2::tc;

namespace ab2 {
namespace {

constexpr int PC_Q = 128, PC_KEYS = 80, PC_THREADS = 384, PC_LOAD = 128;   // threads; those that make codes values
constexpr int PC_QBOX = PC_Q * 128, PC_BOX = PC_KEYS * 128;   // boxes of queries, and of keys or values: rows of 64 elements
constexpr int PC_ROWS = 16;   // that one copy brings: the least that a page holds
constexpr int PC_TWICE = 16;  // query rows of an item up to which it has each of them twice, for both terms of its weights
constexpr int PC_FEW_REGS = 80, PC_LOAD_REGS = 48, PC_MANY_REGS = 192;   // over codes, of a thread of copies and issue, of those that make values, and of softmax: 128 of either of the first, and 256, are the 512 of 128 of the launch
constexpr float PC_SLACK = 8.f;  // powers of two a score may exceed the row's maximum by
constexpr float PC_NONE = -1e30f;

template <int HD, bool E8 = false> struct PcShape {
    static constexpr int THREADS = PC_THREADS + (E8 ? PC_LOAD : 0);
    static constexpr int BOXES = HD / 64, QTILE = BOXES * PC_QBOX, VTILE = BOXES * PC_BOX, KTILE = E8 ? PC_KEYS * HD : VTILE;   // bytes of a tile: queries (over codes two terms of 8 bits), values, keys
    static constexpr int SLOTS = HD == 128 ? 4 : 8, SLOT = KTILE + VTILE;   // a slot holds a tile's keys and its values
    static constexpr int RAWS = E8 ? 2 : 0, RAW = E8 ? PC_KEYS * HD : 0;             // codes of values as they come
    static constexpr int SMEM = 1024 + 2 * QTILE + SLOTS * SLOT + RAWS * RAW;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two f32 at a time.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float low(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float high(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) { return pair(ex2(low(x)), ex2(high(x))); }
// What all roles know of a piece.
struct PcPiece {
    PagedPiece w;
    PagedSpan s;
    int first, second;   // tiles of keys that either tile of rows looks at
    __device__ __forceinline__ int most() const { return max(first, second); }
};
template <bool WIN> __device__ __forceinline__ bool pc_next(const PagedPlan &a, PagedRun &run, PcPiece &x) {
    if (!paged_next<WIN>(a, run, x.w)) return false;
    x.s = paged_span<WIN>(a, x.w);
    const int rows = x.s.ntok * a.group;
    const int gap = paged_hole<WIN>(a, x.s.base, x.w.q_tile).gap;
    auto tiles = [&](int first, int end) {   // of rows [first, end) of the item: keys up to those of the last token
        const int last = min(x.s.hi, x.s.base + x.s.t0 + paged_token(a, end - 1) + 1 - gap);
        return end > first ? max(0, (last - x.s.lo + PC_KEYS - 1) / PC_KEYS) : 0;
    };
    x.first = tiles(0, min(rows, PC_Q));
    x.second = tiles(PC_Q, rows);
    return true;
}

struct PcTile {   // of codes
    float k[PC_KEYS / PC_ROWS], v;    // scales of the blocks of keys, and the unit of the values
    __half2 f[PC_KEYS / PC_ROWS];     // scales of the blocks of values in that unit; those far below it times -PC_FAR
    int rows;                         // that the piece has of it; negative: there is no more tile
    uint32_t blocks;                  // a bit for each that a token sees
};
template <int SLOTS, int RAWS, int THREADS> struct PcShared {
    static constexpr int TILES = RAWS ? SLOTS + RAWS : 1;   // on their way or in use
    uint64_t full[SLOTS], empty[SLOTS], qfull[2], sfull[2], sfree[2], pfull[2], odone[2], rfull[RAWS ? RAWS : 1], rempty[RAWS ? RAWS : 1];
    uint32_t tmem_base;
    int failed;
    float lost;   // of codes: how far a value may be off at most, of blocks far below their tile's unit
    union {
        struct {                                // while the CTA looks for its run
            long long warp_sums[THREADS / 32];
            int2 found[2];
        };
        struct {
            PagedRun start;                     // that run, over the sums alone: other threads may still read what was found
            PcTile tiles[TILES];                // behind a barrier of all
        };
    };
    // of every softmax warp: its run, the piece that it is at and the next one (kept from its registers, which the scores fill)
    PagedRun run[8];
    PcPiece piece[8][2];
};

// Of a tile's scores v(0) .. v(PC_KEYS - 1), those out of sight become -inf: past `lim` and, WIN, from `sinks` up to `since`.
template <bool WIN, class Scores> __device__ __forceinline__ void pc_hide(Scores v, int lim, int sinks, int since) {
    if constexpr (WIN) {
        // a bit for each key in sight, 32 at a time
        auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };   // bits of the keys below n
#pragma unroll
        for (int w = 0; w < PC_KEYS; w += 32) {
            const uint32_t seen = below(lim + 1 - w) & (below(sinks - w) | ~below(since - w));
#pragma unroll
            for (int k = w; k < w + 32 && k < PC_KEYS; ++k)
                if (!((seen >> (k - w)) & 1)) v(k) = 0xff800000u;
        }
    } else {
#pragma unroll
        for (int k = 0; k < PC_KEYS; ++k)
            if (k > lim) v(k) = 0xff800000u;
    }
}

// One tile of keys for the warp's 32 rows, a lane each: scores to weights.  With `edge` some may be out of sight (pc_hide); with `twice` a lane that is `second` hands on
// what rounding left of each weight.  `before` waits until the products with the tile before are done: its weights' place is free then, and the sums stand still.
// KIND: 0 of a tile with neither, 1 of one with an edge, 2 of either.  Over codes and through windows one text serves all tiles, with branches around what some need: two
// drove each other, and all that runs between pieces, out of the instruction cache (six mixed rows over codes 179 us, in one text 150; 8000 tokens through a window of 1024 149 and 134).  Else
// tiles with an edge have their own: a prompt has few of them, and its long runs of others go by 3.5 % faster (4096 behind 4096 370 for 383).
template <int HD, bool WIN, int KIND, class Before>
__device__ __forceinline__ void pc_softmax(uint32_t s_addr, uint32_t o_addr, float sl, bool flip, bool edge, int lim, int sinks, int since, bool twice, bool second, bool has_o, float &top, float &sum, uint64_t *taken, uint64_t *ready, Before before) {
    uint32_t va[32], vb[32], vc[16];
    tmem_ld32_start(va, s_addr);
    tmem_ld32_start(vb, s_addr + 32);
    tmem_ld16_start(vc, s_addr + 64);
    tmem_ld16_wait(vc);
    tmem_ld32_wait(va);
    tmem_ld32_wait(vb);
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(taken);
    auto v = [&](int k) -> uint32_t & { return k < 32 ? va[k] : k < 64 ? vb[k - 32] : vc[k - 64]; };
    if (flip)   // a negative scale
#pragma unroll
        for (int k = 0; k < PC_KEYS; ++k) v(k) ^= 0x80000000u;
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    edge = KIND == 2 ? edge : KIND == 1;
    twice &= KIND != 0;
    if (edge) pc_hide<WIN>(v, lim, sinks, since);
#pragma unroll
    for (int k = 0; k < PC_KEYS; k += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(v(k + e)), __uint_as_float(v(k + 4 + e)));
    const float best = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * sl;  // the scale is not negative
    const float now = best > top + PC_SLACK ? best : top;
    before();
    if (__any_sync(0xffffffffu, now != top)) {
        const float corr = ex2(top - now);
        sum *= corr;
        top = now;
        if (has_o) {
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(o, o_addr + 32 * c);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                tmem_st32(o_addr + 32 * c, o);
            }
        }
    }
    const uint64_t sl2 = pair(sl, sl), top2 = pair(-top, -top);
    uint64_t total[2] = {0ull, 0ull};
    auto weights = [&](int k) {   // of keys k and k + 1
        const uint64_t e = ex2_pair(fma2(pair(__uint_as_float(v(k)), __uint_as_float(v(k + 1))), sl2, top2));
        total[(k >> 1) & 1] = add2(total[(k >> 1) & 1], e);
        const __nv_bfloat162 b = __floats2bfloat162_rn(low(e), high(e));
        return *reinterpret_cast<const uint32_t *>(&b);
    };
    auto rest = [&](int k, uint32_t word) {
        const uint64_t e = ex2_pair(fma2(pair(__uint_as_float(v(k)), __uint_as_float(v(k + 1))), sl2, top2));
        const __nv_bfloat162 left = __floats2bfloat162_rn(low(e) - __uint_as_float(word << 16), high(e) - __uint_as_float(word & 0xffff0000u));
        return second ? *reinterpret_cast<const uint32_t *>(&left) : word;
    };
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = weights(32 * c + 2 * k);
        if (twice)
#pragma unroll
            for (int k = 0; k < 16; ++k) p[k] = rest(32 * c + 2 * k, p[k]);
        tmem_st16(s_addr + PC_KEYS + 16 * c, p);
    }
    {
        uint32_t p[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = weights(64 + 2 * k);
        if (twice)
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = rest(64 + 2 * k, p[k]);
        tmem_st8(s_addr + PC_KEYS + 32, p);
    }
    total[0] = add2(total[0], total[1]);
    sum += low(total[0]) + high(total[0]);
    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(ready);
}

// Four lanes with four pieces each: piece k of lane i for piece i of lane k.
__device__ __forceinline__ void exchange4(uint4 (&o)[4], int lane) {
    auto swap = [](uint4 &a, uint4 &b, bool odd, int d) {   // the even lane's b for the odd lane's a
        uint4 s = odd ? a : b;
        s.x = __shfl_xor_sync(0xffffffffu, s.x, d); s.y = __shfl_xor_sync(0xffffffffu, s.y, d); s.z = __shfl_xor_sync(0xffffffffu, s.z, d); s.w = __shfl_xor_sync(0xffffffffu, s.w, d);
        if (odd) a = s;
        else b = s;
    };
    swap(o[0], o[1], lane & 1, 1);
    swap(o[2], o[3], lane & 1, 1);
    swap(o[0], o[2], lane & 2, 2);
    swap(o[1], o[3], lane & 2, 2);
}

// Over codes keys are multiplied as they are, with queries in two e4m3 terms: a bf16 number has 8 significant bits, and is the sum of two of 4 (in units of a power of two of
// its row's that puts the largest at 224 to 448; below 2^-2 the second term has fewer: 2^-18 of the row's largest element off at most).  A block's scale multiplies its scores beside the
// softmax's factor.  Values are f16, in units of the tile's largest scale (a block's other scale is a power of two below it, and exact down to 2^-15); their weights are f16 in units of `vref`, a
// scale of values that moves as the maximum does: up to one over 4 times it (2^8 of a weight, 4 and PC_UP make 2^15), down where f16 would lose bits of them.  Values of a block further
// below its tile's largest than 2^-15 are rounded to 2^-24 of the unit, and the producer notes by how much they may be off: rows whose largest output is not 2^20 times that, as of those that see hardly anything else, are computed
// again in f32 like those that meet NaN.  (With all rows of such a tile computed again one block of 2^-20 among 1000 took 4096 behind 12288 from 1.0 ms to 475; with bf16 for both operands of such a tile
// all others took 2 to 8 % longer.  This takes 1.12 ms of it, and of 4096 behind 12288 without such blocks nothing, with heads of 64 4 %.)
constexpr float PC_UP = 32.f, PC_MORE = 4.f, PC_LESS = 9.765625e-4f, PC_APART = 3.0517578e-5f, PC_NOTHING = 8.6736174e-19f, PC_ZEROS = 7.8886091e-31f, PC_FAR = 4096.f, PC_ENOUGH = 1048576.f;   // 2^-10, 2^-15, 2^-60, 2^-100, 2^20
// What a row's warp keeps of the values' scales: the unit of the sums, and of the tile before its scale, what that adds to a weight's exponent, and its inverse as a factor.
struct PcUnit {
    float vref, last, more, less;
};
template <int HD, bool WIN, class Before>
__device__ __forceinline__ void pc_softmax_codes(uint32_t s_addr, uint32_t o_addr, float sl, bool edge, int lim, int sinks, int since, const PcTile &of, bool has_o, float &top, float &sum, PcUnit &unit,
                                                 uint64_t *taken, uint64_t *ready, Before before) {
    constexpr int BLOCKS = PC_KEYS / PC_ROWS;
    uint32_t va[32], vb[32], vc[16];
    tmem_ld32_start(va, s_addr);
    tmem_ld32_start(vb, s_addr + 32);
    tmem_ld16_start(vc, s_addr + 64);
    float scale[BLOCKS], vref = unit.vref;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) scale[b] = fmaxf(sl * of.k[b], 1.17549435e-38f);   // above 0, so that hidden scores stay -inf
    const float values = of.v;
    if (values > vref * PC_MORE || (values < vref * PC_LESS && values > vref * PC_NOTHING)) vref = fmaxf(values, 3.0092655e-36f);
    tmem_ld16_wait(vc);
    tmem_ld32_wait(va);
    tmem_ld32_wait(vb);
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(taken);
    auto v = [&](int k) -> uint32_t & { return k < 32 ? va[k] : k < 64 ? vb[k - 32] : vc[k - 64]; };
    if (edge) pc_hide<WIN>(v, lim, sinks, since);
    float best = -INFINITY;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        auto s = [&](int k) { return __uint_as_float(v(16 * b + k)); };
        float m0 = max3(s(0), s(1), s(2)), m1 = max3(s(3), s(4), s(5));
#pragma unroll
        for (int k = 6; k < 14; k += 4) {
            m0 = max3(m0, s(k), s(k + 1));
            m1 = max3(m1, s(k + 2), s(k + 3));
        }
        best = max3(best, max3(m0, s(14), s(15)) * scale[b], m1 * scale[b]);
    }
    const float now = best > top + PC_SLACK ? best : top;
    before();
    if (__any_sync(0xffffffffu, now != top || vref != unit.vref)) {
        const float keep = ex2(top - now), corr = vref == unit.vref ? keep : keep * (unit.vref / vref);
        sum *= keep;
        top = now;
        if (has_o) {
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(o, o_addr + 32 * c);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                tmem_st32(o_addr + 32 * c, o);
            }
        }
    }
    // The tile's values in units of vref, PC_UP times as large; 2^-40 and less makes weights of nothing (and their sum is still theirs).
    if (values != unit.last || vref != unit.vref) {   // the same for all lanes
        const float f = vref > 0.f ? fmaxf(values / vref * PC_UP, 9.0949470e-13f) : PC_UP;
        unit.last = values;
        unit.vref = vref;
        unit.more = __log2f(f);
        unit.less = 1.f / f;
    }
    const float shifted = unit.more - top;
    const uint64_t top2 = pair(shifted, shifted);
    uint64_t total[2] = {0ull, 0ull};
    auto weights = [&](int k) {   // of keys k and k + 1
        const uint64_t e = ex2_pair(fma2(pair(__uint_as_float(v(k)), __uint_as_float(v(k + 1))), pair(scale[k >> 4], scale[k >> 4]), top2));
        total[(k >> 1) & 1] = add2(total[(k >> 1) & 1], e);
        const __half2 h = __floats2half2_rn(low(e), high(e));
        return *reinterpret_cast<const uint32_t *>(&h);
    };
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = weights(32 * c + 2 * k);
        tmem_st16(s_addr + PC_KEYS + 16 * c, p);
    }
    {
        uint32_t p[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = weights(64 + 2 * k);
        tmem_st8(s_addr + PC_KEYS + 32, p);
    }
    total[0] = add2(total[0], total[1]);
    sum = fmaf(low(total[0]) + high(total[0]), unit.less, sum);
    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(ready);
}

// E8: pages of e4m3.  Keys come by the same copies; four more warps make values, which come as codes, f16 in the ring's slots.
// WIN: a window.
template <int HD, bool E8, bool WIN>
__global__ void __launch_bounds__(PcShape<HD, E8>::THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedAttnArgs a) {
    using S = PcShape<HD, E8>;
    using Page = std::conditional_t<E8, uint8_t, __nv_bfloat16>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PcShared<S::SLOTS, S::RAWS, S::THREADS> sh;
    constexpr int RAWS = S::RAWS ? S::RAWS : 1, TILES = sh.TILES;
    static_assert(S::SMEM + sizeof(sh) <= 227 * 1024, "shared memory of a CTA");
    static_assert(sizeof(PagedRun) <= S::THREADS / 32 * sizeof(long long), "the run lies over the sums");
    uint8_t *qbuf = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023), *ring = qbuf + 2 * S::QTILE, *codes = ring + S::SLOTS * S::SLOT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *failed = &sh.failed;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::SLOTS; ++i) { bar_init(&sh.full[i], 1 + (E8 ? PC_LOAD / 32 : 0)); bar_init(&sh.empty[i], 2); }
        for (int i = 0; i < S::RAWS; ++i) { bar_init(&sh.rfull[i], 1); bar_init(&sh.rempty[i], PC_LOAD / 32); }
        for (int i = 0; i < 2; ++i) { bar_init(&sh.qfull[i], 4); bar_init(&sh.sfull[i], 1); bar_init(&sh.sfree[i], 4); bar_init(&sh.pfull[i], 4); bar_init(&sh.odone[i], 1); }
        sh.failed = 0;
        sh.lost = 0.f;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    pdl_wait();   // ahead of tensor memory too, which the launch before may hold
    PagedRun run = paged_run<S::THREADS, WIN>(a.plan, blockIdx.x, a.ctas, sh.warp_sums, sh.found, a.status);
    if (threadIdx.x == PC_THREADS - 1) paged_uncut(a, blockIdx.x);
    if (run.u >= run.u1) return;   // the whole CTA
    if (threadIdx.x == 0) sh.start = run;
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(sptr(&sh.tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem = sh.tmem_base, tmem_o = tmem + 256;   // a tile of rows has 128 columns for scores and weights
    const PagedView &p = a.plan.p;
    PcPiece x;
    // the block's registers: 128 threads of 72 and 256 of 216 are the 384 of 168 that it was launched with (over codes PC_FEW_REGS and the others of 128)
    if (E8 && warp >= PC_THREADS / 32) {
        // ---------------------------------------------------------- values from codes
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(PC_LOAD_REGS));
        // A short loop: unrolled, its text drives that of the softmax out of the instruction cache (4096 behind 12288, values by registers a tile ahead, 1150 us).
        // A thread has 16 codes of every ROWS-th row: two chunks of the row in its box of 64 elements; those of the second box go in the other order, so that eight lanes
        // meet in no bank.
        constexpr int CH = HD / 16, ROWS = PC_LOAD / CH;
        const int me = threadIdx.x - PC_THREADS, row0 = me / CH, ch = me % CH, odd = (ch >> 2) & 1, c0 = 2 * (ch & 3) + odd;
        const uint8_t *from = codes + row0 * HD + ch * 16;
        uint8_t *to0 = ring + S::KTILE + (ch >> 2) * PC_BOX + row0 * 128 + ((c0 ^ (row0 & 7)) << 4), *to1 = to0 + ((((c0 ^ 1) ^ (row0 & 7)) << 4) - ((c0 ^ (row0 & 7)) << 4));
        for (int n = 0;; ++n) {
            const int slot = n % S::SLOTS, raw = n % RAWS;
            warp_wait(&sh.rfull[raw], (n / RAWS) & 1, failed);
            const PcTile &tile = sh.tiles[n % TILES];
            const int rows = tile.rows;
            if (rows < 0 || *failed) break;
            const uint32_t blocks = tile.blocks;
            warp_wait(&sh.empty[slot], ((n / S::SLOTS) & 1) ^ 1, failed);
#pragma unroll 1
            for (int r = row0; r < PC_KEYS; r += ROWS) {
                const __half2 f = tile.f[r / PC_ROWS];
                const bool far = *reinterpret_cast<const int *>(&f) < 0;   // the same for all lanes
                uint4 c = make_uint4(0u, 0u, 0u, 0u);   // behind the piece's keys, and where no token sees a block
                if (r < rows && ((blocks >> (r / PC_ROWS)) & 1)) c = *reinterpret_cast<const uint4 *>(from + raw * S::RAW + (r - row0) * HD);
                auto two = [&](uint32_t codes) {
                    const uint32_t h = f16x2_of_codes(codes);
                    __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&h), f);
                    if (far) y = __hmul2(y, __float2half2_rn(-1.f / PC_FAR));
                    return *reinterpret_cast<const uint32_t *>(&y);
                };
                const uint4 low8 = make_uint4(two(c.x), two(c.x >> 16), two(c.y), two(c.y >> 16)), high8 = make_uint4(two(c.z), two(c.z >> 16), two(c.w), two(c.w >> 16));
                *reinterpret_cast<uint4 *>(to0 + slot * S::SLOT + (r - row0) * 128) = odd ? high8 : low8;
                *reinterpret_cast<uint4 *>(to1 + slot * S::SLOT + (r - row0) * 128) = odd ? low8 : high8;
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();   // every lane's codes have been read, as what it stored is made of them
            if (lane == 0) {
                bar_arrive(&sh.full[slot]);
                bar_arrive(&sh.rempty[raw]);
            }
        }
    } else if (warp < 4) {
        if (E8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(PC_FEW_REGS));
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        if (E8 && warp == 0) {
            // ---------------------------------------------------------- producer over codes: V, as codes, then K
            int n = 0;
            float lost = 0.f;
            while (pc_next<WIN>(a.plan, run, x)) {
                const PagedHole hole = paged_hole<WIN>(a.plan, x.s.base, x.w.q_tile);
                for (int j = 0; j < x.most(); ++j, ++n) {
                    const int v = x.s.lo + j * PC_KEYS + lane * PC_ROWS, key = WIN ? paged_key(hole, v) : v, raw = n % RAWS, slot = n % S::SLOTS;
                    const bool mine = lane < PC_KEYS / PC_ROWS && v < x.s.hi && !(WIN && paged_hidden(a.plan, x.s, key, PC_ROWS));
                    const int page = mine ? paged_page(p, x.w.row, key, a.status) : 0, at = key & ((1 << p.page_shift) - 1);
                    const size_t row = mine ? (((size_t)page * p.kv_heads + x.w.head) << p.page_shift) + at : 0;
                    const float ks = mine ? __ldg(a.k_scales + row / PAGED_BLOCK) : 0.f, vs = mine ? __ldg(a.v_scales + row / PAGED_BLOCK) : 0.f;
                    const uint32_t blocks = __ballot_sync(0xffffffffu, mine);
                    const int bytes = __popc(blocks) * PC_ROWS * HD;
                    float unit = vs;
#pragma unroll
                    for (int m = 1; m < 8; m <<= 1) unit = fmaxf(unit, __shfl_xor_sync(0xffffffffu, unit, m));
                    const float part = unit > 0.f ? vs / unit : 0.f;
                    const bool far = part < PC_APART && vs > PC_ZEROS;
                    const __half2 f = __float2half2_rn(far ? part * -PC_FAR : part);
                    warp_wait(&sh.rempty[raw], ((n / RAWS) & 1) ^ 1, failed);
                    PcTile &tile = sh.tiles[n % TILES];
                    if (lane < PC_KEYS / PC_ROWS) { tile.k[lane] = ks; tile.f[lane] = f; }
                    if (lane == 0) { tile.v = unit; tile.rows = x.s.hi - (x.s.lo + j * PC_KEYS); tile.blocks = blocks; }
                    __syncwarp();
                    if (lane == 0) bar_expect_tx(&sh.rfull[raw], (uint32_t)bytes);
                    __syncwarp();
                    if (mine && !*failed) bulk_copy(codes + raw * S::RAW + lane * PC_ROWS * HD, (const uint8_t *)a.v + row * HD, PC_ROWS * HD, &sh.rfull[raw]);
                    if (__any_sync(0xffffffffu, far)) {   // behind the values' copies; the keys' barrier hands it on to those that read it
                        float off = far ? unit * fminf(2.9802322e-8f, 448.f * part) : 0.f;   // half of f16's least step, or all of the value
#pragma unroll
                        for (int m = 1; m < 8; m <<= 1) off = fmaxf(off, __shfl_xor_sync(0xffffffffu, off, m));
                        if (lane == 0 && off > lost) sh.lost = lost = off;
                    }
                    warp_wait(&sh.empty[slot], ((n / S::SLOTS) & 1) ^ 1, failed);
                    if (lane == 0) bar_expect_tx(&sh.full[slot], (uint32_t)bytes);
                    __syncwarp();
                    // (of blocks that are not copied the slot holds what it held: their scores are hidden, whatever they are)
                    if (mine && !*failed) tma_load_3d(ring + slot * S::SLOT + lane * PC_ROWS * HD, &kmap, 0, at, page * p.kv_heads + x.w.head, &sh.full[slot]);
                }
            }
            warp_wait(&sh.rempty[n % RAWS], ((n / RAWS) & 1) ^ 1, failed);
            if (lane == 0) {
                sh.tiles[n % TILES].rows = -1;
                bar_arrive(&sh.rfull[n % RAWS]);
            }
        } else if (warp == 0) {
            // ---------------------------------------------------------- TMA producer: K, V, K, V, ...
            int n = 0;
            while (pc_next<WIN>(a.plan, run, x)) {
                const PagedHole hole = paged_hole<WIN>(a.plan, x.s.base, x.w.q_tile);
                for (int j = 0; j < x.most(); ++j) {
                    const int v = x.s.lo + j * PC_KEYS + lane * PC_ROWS, key = WIN ? paged_key(hole, v) : v;
                    const bool mine = lane < PC_KEYS / PC_ROWS && v < x.s.hi;
                    // a block that no token sees comes from behind the pool, as zeros
                    const int page = !mine ? 0 : WIN && paged_hidden(a.plan, x.s, key, PC_ROWS) ? p.pages : paged_page(p, x.w.row, key, a.status);
                    const int bytes = __popc(__ballot_sync(0xffffffffu, mine)) * PC_ROWS * HD * 4;
                    const int slot = n % S::SLOTS;
                    warp_wait(&sh.empty[slot], ((n++ / S::SLOTS) & 1) ^ 1, failed);
                    // The first queries come before what is fetched ahead.  Only at the second slot of the run's first piece with keys, and only where the first
                    // tile of rows looks at it: its warps cannot announce their next queries without that slot, so the barrier is in its first phase or just
                    // behind it.  A later phase would have this parity again, and might wait for what is not yet fetched.
                    if (n == 2 && j == 1 && x.first > 1) warp_wait(&sh.qfull[0], 0, failed);
                    if (lane == 0) bar_expect_tx(&sh.full[slot], (uint32_t)bytes);
                    __syncwarp();
                    if (mine && !*failed)
#pragma unroll
                        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                            for (int b = 0; b < S::BOXES; ++b)
                                tma_load_3d(ring + slot * S::SLOT + kv * S::KTILE + b * PC_BOX + lane * PC_ROWS * 128, kv ? &vmap : &kmap, b * 64, key & ((1 << p.page_shift) - 1), page * p.kv_heads + x.w.head, &sh.full[slot]);
                }
            }
        } else if (warp < 3) {
            // ---------------------------------------------------------- MMA issue for a tile of rows
            constexpr uint32_t IDESC = (1u << 4) | (E8 ? 0u : (1u << 7) | (1u << 10)) | ((128u >> 4) << 24);   // both operands e4m3 (of scores) or f16, or bf16
            constexpr uint32_t S_DESC = IDESC | ((uint32_t)(PC_KEYS >> 3) << 17), O_DESC = IDESC | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
            const int g = warp - 1;
            const uint32_t s_at = tmem + (uint32_t)(g * 128), p_at = s_at + PC_KEYS, o_at = tmem_o + (uint32_t)(g * HD);
            int n = 0, scored = 0, done = 0, asked = 0;   // slots of the ring passed; scores, sums and pieces of this tile of rows
            auto scores = [&](int n) {
                const int slot = n % S::SLOTS;
                warp_wait(&sh.full[slot], (n / S::SLOTS) & 1, failed);
                if (scored > 0) warp_wait(&sh.sfree[g], (scored - 1) & 1, failed);
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                if (elect_one()) {
                    if constexpr (E8) {   // both terms of the queries: of 128 dimensions two boxes, of 64 the halves of a row
                        const uint64_t kd = HD == 128 ? umma_desc(sptr(ring + slot * S::SLOT)) : umma_desc_64(sptr(ring + slot * S::SLOT));
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const uint64_t qd = umma_desc(sptr(qbuf + g * S::QTILE + (HD == 128 ? b * PC_QBOX : 0))) + (uint64_t)(HD == 128 ? 0 : 4 * b);
#pragma unroll
                            for (int k = 0; k < HD / 32; ++k) umma_f8(s_at, qd + (uint64_t)(2 * k), kd + (uint64_t)(2 * k), S_DESC, (b | k) != 0);
                        }
                    } else {
#pragma unroll
                        for (int b = 0; b < S::BOXES; ++b) {
                            const uint64_t qd = umma_desc(sptr(qbuf + g * S::QTILE + b * PC_QBOX)), kd = umma_desc(sptr(ring + slot * S::SLOT + b * PC_BOX));
#pragma unroll
                            for (int k = 0; k < 4; ++k)  // descriptors count in 16 bytes
                                umma_bf16(s_at, qd + (uint64_t)(2 * k), kd + (uint64_t)(2 * k), S_DESC, (b | k) != 0);
                        }
                    }
                    umma_commit(&sh.sfull[g]);
                }
                __syncwarp();
                ++scored;
            };
            while (pc_next<WIN>(a.plan, run, x)) {
                const int tiles = g ? x.second : x.first;
                if (tiles > 0) {
                    warp_wait(&sh.qfull[g], asked++ & 1, failed);
                    scores(n);
                }
                for (int j = 0; j < x.most(); ++j, ++n) {
                    const int slot = n % S::SLOTS;
                    if (j + 1 < tiles) scores(n + 1);
                    if (j >= tiles) {   // only the other tile of rows looks at this one
                        warp_wait(&sh.full[slot], (n / S::SLOTS) & 1, failed);
                        if (lane == 0) bar_arrive(&sh.empty[slot]);
                        continue;
                    }
                    warp_wait(&sh.pfull[g], done++ & 1, failed);
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    if (elect_one()) {
                        const uint64_t vd = umma_desc_mn(sptr(ring + slot * S::SLOT + S::KTILE), PC_BOX);
#pragma unroll
                        for (int k = 0; k < PC_KEYS / 16; ++k)
                            umma_bf16_ts(o_at, p_at + (uint32_t)(8 * k), vd + (uint64_t)(k * (2048 >> 4)), O_DESC, j > 0 || k > 0);
                        umma_commit(&sh.odone[g]);
                        umma_commit(&sh.empty[slot]);
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        // ---------------------------------------------------------- softmax
        if (E8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(PC_MANY_REGS));
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        const int g = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane, group = a.plan.group;
        const uint32_t quad_addr = (uint32_t)(quad * 32) << 16, s_addr = tmem + quad_addr + (uint32_t)(g * 128), o_addr = tmem_o + quad_addr + (uint32_t)(g * HD);
        const float sl = fmaxf(fabsf(a.sl), 1.17549435e-38f);   // above 0, so that hidden scores stay -inf
        const bool flip = a.sl < 0.f;
        int n = 0, scored = 0;
        int n0 = 0, here = 0;   // the first of the ring's slots of the next piece; where that is kept
        if (lane == 0) sh.run[warp - 4] = run;
        // the next piece in which this tile of rows has any
        auto next = [&]() {
            __syncwarp();
            PagedRun run = sh.run[warp - 4];
            PcPiece x;
            bool more;
            while ((more = pc_next<WIN>(a.plan, run, x))) {
                n0 = n;
                n += x.most();
                if (threadIdx.x == PC_THREADS - 1) paged_cut(a, run, x.w, x.s, blockIdx.x);
                if (x.s.ntok * group > g * PC_Q) break;
            }
            here ^= 1;
            __syncwarp();
            if (lane == 0) { sh.run[warp - 4] = run; sh.piece[warp - 4][here] = x; }
            __syncwarp();
            return more;
        };
        // its queries, on their way to shared memory
        float back = 1.f;   // E8: what the row's queries are to be multiplied by
        PcUnit unit;
        auto fetch_q = [&]() {
            const PcPiece &x = sh.piece[warp - 4][here];
            if ((g ? x.second : x.first) == 0) return;   // nothing to ask
            const PagedSpan s = x.s;
            const long long first = x.w.r.first + s.t0, head0 = x.w.head * group;
            if constexpr (E8) {   // every warp its own rows, which it makes codes where they come to lie
#pragma unroll 2   // short text: the instruction cache has all of a piece to hold (through a window of 128 unrolled 81 us, by 4 73, so 71)
                for (int u = 0; u < HD / 8; ++u) {
                    const int i = lane + 32 * u, d = i % (HD / 8), row = quad * 32 + i / (HD / 8), rr = g * PC_Q + row, in = rr < s.ntok * group ? 16 : 0, tok = paged_token(a.plan, in ? rr : 0);
                    const __nv_bfloat16 *src = (const __nv_bfloat16 *)a.q + (first + tok) * a.q_stride + (head0 + (in ? rr - tok * group : 0)) * HD + d * 8;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(sptr(qbuf + g * S::QTILE + (d >> 3) * PC_QBOX + row * 128 + (((d & 7) ^ (row & 7)) << 4))), "l"(src), "r"(in) : "memory");
                }
                asm volatile("cp.async.commit_group;\n" ::: "memory");
                return;
            }
            const int i0 = threadIdx.x & 127, rows = s.ntok * group;
            const bool twice = rows <= PC_TWICE;
#pragma unroll 2   // short text: the instruction cache has all of a piece to hold (through a window of 128 unrolled 81 us, by 4 73, so 71)
            for (int u = 0; u < PC_Q * HD / 8 / 128; ++u) {
                const int i = i0 + 128 * u, d = i % (HD / 8), row = i / (HD / 8), rr = twice && row < 2 * PC_TWICE ? row % PC_TWICE : g * PC_Q + row, in = rr < rows ? 16 : 0, tok = paged_token(a.plan, in ? rr : 0);
                const __nv_bfloat16 *src = (const __nv_bfloat16 *)a.q + (first + tok) * a.q_stride + (head0 + (in ? rr - tok * group : 0)) * HD + d * 8;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(sptr(qbuf + g * S::QTILE + (d >> 3) * PC_QBOX + row * 128 + (((d & 7) ^ (row & 7)) << 4))), "l"(src), "r"(in) : "memory");
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
        // E8: a thread's row of queries, from bf16 to two terms of codes in its place
        auto terms_of_q = [&]() {
            auto at = [&](int c) { return reinterpret_cast<uint4 *>(qbuf + g * S::QTILE + (c >> 3) * PC_QBOX + r * 128 + (((c & 7) ^ (r & 7)) << 4)); };   // 16 bytes c of it
            uint4 q[HD / 8];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) q[i] = *at(i);
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
                for (uint32_t w : {q[i].x, q[i].y, q[i].z, q[i].w}) most = max3(most, fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u)));
            // times 2^(127 - down) the largest is between 224 and 448 = 1.75 2^8
            const uint32_t bits = __float_as_uint(most);
            const int down = min(max((int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u), 1), 253);
            const float f = most < INFINITY ? __uint_as_float((uint32_t)(254 - down) << 23 | (flip ? 0x80000000u : 0u)) : __uint_as_float(0x7fc00000u);   // Inf has no code
            back = __uint_as_float((uint32_t)down << 23);
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                uint32_t high[4], rest[4];
                const uint32_t words[8] = {q[2 * i].x, q[2 * i].y, q[2 * i].z, q[2 * i].w, q[2 * i + 1].x, q[2 * i + 1].y, q[2 * i + 1].z, q[2 * i + 1].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t h[2], l[2];
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const uint32_t w = words[2 * e + d];
                        const __half2 x = __floats2half2_rn(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xffff0000u) * f);   // exact down to 2^-14
                        h[d] = codes_of(x);
                        const uint32_t y = f16x2_of_codes(h[d]);
                        l[d] = codes_of(__hsub2(x, *reinterpret_cast<const __half2 *>(&y)));
                    }
                    high[e] = h[0] | h[1] << 16;
                    rest[e] = l[0] | l[1] << 16;
                }
                *at(i) = make_uint4(high[0], high[1], high[2], high[3]);
                *at(HD / 16 + i) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
            }
        };
        bool more = next(), again = false;   // again: a row's sums came out as Inf or NaN
        if (more) fetch_q();
        while (more) {
            const PcPiece &x = sh.piece[warp - 4][here];
            const int rows = x.s.ntok * group, tiles = g ? x.second : x.first, lo = x.s.lo, hi = x.s.hi, slot0 = n0;
            if (tiles > 0) {
                asm volatile("cp.async.wait_group 0;\n" ::: "memory");
                if constexpr (E8) {
                    __syncwarp();   // the warp's rows have come
                    terms_of_q();
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.qfull[g]);
            }
            const bool twice = !E8 && rows <= PC_TWICE;   // and this the first tile of rows
            const float row_sl = E8 ? sl * back : sl;
            unit = {0.f, -1.f, 0.f, 1.f};
            const bool second = twice && (lane & PC_TWICE);
            const int rr = g * PC_Q + r, asks = twice && r < 2 * PC_TWICE ? r % PC_TWICE : rr;
            const int gap = paged_hole<WIN>(a.plan, x.s.base, x.w.q_tile).gap, first = x.s.base + x.s.t0 - gap;   // all in virtual keys
            const int pos = asks < rows ? first + paged_token(a.plan, asks) : -1;
            const int least = first + paged_token(a.plan, g * PC_Q);   // the first row sees up to here
            const int late = WIN ? first + paged_token(a.plan, min(rows, (g + 1) * PC_Q) - 1) + 1 - a.plan.window : 0;   // the last row sees from here on, and the sinks
            float top = PC_NONE, sum = 0.f;
            for (int j = 0; j < tiles; ++j, ++scored) {
                const int at = lo + j * PC_KEYS;
                warp_wait(&sh.sfull[g], scored & 1, failed);
                if (!E8 && at + PC_KEYS > hi) {   // what lies behind the piece's keys may be anything
                    // Behind the wait for the scores, never ahead of it: these warps pass over pieces without rows of theirs, and the slot's barrier may still be phases
                    // away from the one meant, with the same parity.
                    const int slot = (slot0 + j) % S::SLOTS;
                    warp_wait(&sh.full[slot], ((slot0 + j) / S::SLOTS) & 1, failed);
                    if (at + r >= hi && r < PC_KEYS)
#pragma unroll
                        for (int b = 0; b < S::BOXES; ++b)
#pragma unroll
                            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4 *>(ring + slot * S::SLOT + S::KTILE + b * PC_BOX + r * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();   // and the products wait for all four warps
                }
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const int lim = min(pos, hi - 1) - at, low = WIN ? pos + 1 - a.plan.window - at : 0;
                auto before = [&] { if (j > 0) warp_wait(&sh.odone[g], (scored - 1) & 1, failed); };
                const bool edge = at + PC_KEYS - 1 > least || at + PC_KEYS > hi || (g + 1) * PC_Q > rows || (WIN && at < late && at + PC_KEYS > a.plan.sinks);
                const int sinks = WIN ? a.plan.sinks - at : 0;
                if constexpr (E8) pc_softmax_codes<HD, WIN>(s_addr, o_addr, row_sl, edge, lim, sinks, low, sh.tiles[(slot0 + j) % TILES], j > 0, top, sum, unit, &sh.sfree[g], &sh.pfull[g], before);
                else if constexpr (WIN) pc_softmax<HD, true, 2>(s_addr, o_addr, sl, flip, edge, lim, sinks, low, twice, second, j > 0, top, sum, &sh.sfree[g], &sh.pfull[g], before);
                else if (edge) pc_softmax<HD, false, 1>(s_addr, o_addr, sl, flip, true, lim, 0, 0, twice, second, j > 0, top, sum, &sh.sfree[g], &sh.pfull[g], before);
                else pc_softmax<HD, false, 0>(s_addr, o_addr, sl, flip, false, lim, 0, 0, false, false, j > 0, top, sum, &sh.sfree[g], &sh.pfull[g], before);
            }
            const float of_sums = E8 ? unit.vref * (1.f / PC_UP) : 1.f;
            // the scores are all made: the next piece's queries may take the place of these, while the sums go out
            more = next();
            if (more) fetch_q();
            const PagedPiece w = x.w;
            const PagedSpan s = x.s;
            if (tiles > 0) warp_wait(&sh.odone[g], (scored - 1) & 1, failed);
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const bool all = w.k0 == 0 && w.k1 == w.k_tiles;
            const size_t slot = (2 * (size_t)blockIdx.x + (w.k0 == 0)) * a.tile_rows;
            const float f = !all ? of_sums : sum == 0.f ? 0.f : of_sums / sum;
            float poison = 0.f;  // stays 0 unless an output is Inf or NaN
            // A lane has a row, 16 bytes of which at a time would go to 32 places: four lanes exchange pieces and store 64 bytes of a row each time.
            __nv_bfloat16 *dst[4];
            bool have[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int row = g * PC_Q + quad * 32 + (lane & ~3) + k, t = paged_token(a.plan, row);
                have[k] = row < rows;
                dst[k] = (__nv_bfloat16 *)a.out + (size_t)(w.r.first + s.t0 + t) * a.o_stride + (size_t)(w.head * group + row - t * group) * HD + 8 * (lane & 3);
            }
            float *part = a.acc + (slot + g * PC_Q + quad * 32 + (lane & ~3)) * HD + 4 * (lane & 3);
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t v[32];
                __syncwarp();
                tmem_ld32(v, o_addr + 32 * c);
                if (tiles == 0)
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = 0u;
                if (twice)   // both terms' sums
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) + __shfl_xor_sync(0xffffffffu, __uint_as_float(v[k]), PC_TWICE));
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    const float y = __uint_as_float(v[k]) * f;
                    poison = fmaf(y, 0.f, poison);
                    v[k] = __float_as_uint(y);
                }
                if (all) {
                    uint4 o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[8 * k + 2 * e]), __uint_as_float(v[8 * k + 2 * e + 1]));
                            w[e] = *reinterpret_cast<const uint32_t *>(&b);
                        }
                        o[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    exchange4(o, lane);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (have[k]) *reinterpret_cast<uint4 *>(dst[k] + 32 * c) = o[k];
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint4 o[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[k] = make_uint4(v[16 * h + 4 * k], v[16 * h + 4 * k + 1], v[16 * h + 4 * k + 2], v[16 * h + 4 * k + 3]);
                        exchange4(o, lane);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (have[k]) *reinterpret_cast<uint4 *>(part + k * HD + 32 * c + 16 * h) = o[k];
                    }
                }
            }
            if (!all && rr < rows) *reinterpret_cast<float2 *>(a.ml + (slot + rr) * 2) = make_float2(top, sum);
            again |= __any_sync(0xffffffffu, rr < rows && poison != 0.f);   // NaN is not 0
            // the next piece's products may go over what has been read
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        }
        // Rows to compute again, found by what has been stored of them.  Behind the last piece: it may take long, and until then other roles would wait for these
        // warps at barriers whose waits are bounded.
        const float lost = E8 ? __shfl_sync(0xffffffffu, *(const volatile float *)&sh.lost, 0) : 0.f;   // of the tiles that these warps' rows have seen, and it may be others
        if (again || lost > 0.f) {
            PagedRun walk = sh.start;
            PcPiece x;
            while (pc_next<WIN>(a.plan, walk, x)) {
                const int rr = g * PC_Q + r, rows = x.s.ntok * group;
                if (rows <= g * PC_Q) continue;
                const bool all = x.w.k0 == 0 && x.w.k1 == x.w.k_tiles;
                const size_t slot = (2 * (size_t)blockIdx.x + (x.w.k0 == 0)) * a.tile_rows;
                uint32_t worst = 0;   // of the exponents
                float least = 0.f;    // that the largest element has to reach
                if (rr < rows) {
                    if (E8) least = lost * PC_ENOUGH * (all ? 1.f : a.ml[(slot + rr) * 2 + 1]);
                    const int tok = paged_token(a.plan, rr);
                    const uint32_t *o = all ? (const uint32_t *)((const __nv_bfloat16 *)a.out + (size_t)(x.w.r.first + x.s.t0 + tok) * a.o_stride + (size_t)(x.w.head * group + rr - tok * group) * HD)
                                            : (const uint32_t *)(a.acc + (slot + rr) * HD);
                    for (int i = 0; i < (all ? HD / 2 : HD); ++i) {
                        worst = max(worst, o[i] & 0x7f800000u);
                        if (all) worst = max(worst, (o[i] & 0x7f80u) << 16);
                    }
                }
                for (uint32_t left = __ballot_sync(0xffffffffu, worst == 0x7f800000u || (E8 && __uint_as_float(worst) < least)); left; left &= left - 1)
                    paged_again<HD, Page, WIN>(a, x.w, x.s, g * PC_Q + quad * 32 + __ffs(left) - 1, lane, all, slot);
                __syncwarp();
            }
        }
    }
    // ---- teardown: every warp arrives here (all waits are bounded)
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && sh.failed) atomicExch(a.status, (int)AB2_ERR_TIMEOUT);
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

// The pages of a layer: [pages kv_heads][page_size][dim], in boxes of 64 elements of 16 rows.
int pages_map(CUtensorMap *map, const void *pages, const PagedView &p, int hd) {
    const int page = 1 << p.page_shift;
    return make_mats_map(map, pages, p.pages * p.kv_heads, page, hd, hd, (long long)page * hd, PC_ROWS);
}

template <int HD, bool E8, bool WIN>
int launch_tc(PagedAttnArgs a, void *workspace, size_t bytes, cudaStream_t s) {
    using S = PcShape<HD, E8>;
    static bool configured[64] = {false};  // the attribute is per device
    int dev = 0;
    AB2_CUDA(cudaGetDevice(&dev));
    AB2_REQUIRE(dev >= 0 && dev < 64, AB2_ERR_BAD_ARG, "device index %d out of range", dev);
    if (!configured[dev]) {
        AB2_CUDA(cudaFuncSetAttribute(paged_tc_kernel<HD, E8, WIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        configured[dev] = true;
    }
    CUtensorMap kmap = {}, vmap = {};
    if (E8) {
        const int rc = make_byte_mats_map(&kmap, a.k, a.plan.p.pages * a.plan.p.kv_heads, 1 << a.plan.p.page_shift, HD, PC_ROWS);
        if (rc != AB2_OK) return rc;
    } else {
        int rc = pages_map(&kmap, a.k, a.plan.p, HD);
        if (rc == AB2_OK) rc = pages_map(&vmap, a.v, a.plan.p, HD);
        if (rc != AB2_OK) return rc;
    }
    paged_deal(a, device_sm_count(), 2 * PC_Q, 7, 4, HD, workspace, bytes);
    // Set up while the launch before it ends, up to 65536 query rows: all that were tried gain there, and beyond it none does and the longest loses.  32 heads of 128, us
    // not set up early and early: 300 tokens behind 300 35.0 and 32.6, behind 16000 103 and 101.4, 1024 behind 1024 53.7 and 51.9, 2048 alone 82.0 and 80.9, behind
    // 12288 383.8 and 382.6; 3000 behind 3000 231 to 240 and 233 to 237, 4096 alone 207 and 207 to 210, behind 4096 372 and 371, behind 12288 860 to 872 and 876 to 884, 8192 alone 617 and 613 to 621.
    ChainedLaunches chained((long long)a.plan.p.tokens * a.plan.group * a.plan.p.kv_heads <= 65536);
    AB2_CUDA(launch_kernel(paged_tc_kernel<HD, E8, WIN>, dim3(a.ctas), dim3(S::THREADS), S::SMEM, s, kmap, vmap, a));
    return a.plan.whole ? AB2_OK : paged_merge(a, HD, AB2_BF16, s);
}

template <int HD>
int launch_tc(const PagedAttnArgs &a, void *workspace, size_t bytes, cudaStream_t s) {
    if (a.plan.window) return a.k_scales ? launch_tc<HD, true, true>(a, workspace, bytes, s) : launch_tc<HD, false, true>(a, workspace, bytes, s);
    return a.k_scales ? launch_tc<HD, true, false>(a, workspace, bytes, s) : launch_tc<HD, false, false>(a, workspace, bytes, s);
}

}  // namespace

size_t paged_tc_bytes(int hd) { return paged_piece_bytes(device_sm_count(), 2 * PC_Q, hd); }
int paged_tc_attention(const PagedAttnArgs &a, int hd, void *workspace, size_t bytes, cudaStream_t s) {
    return hd == 128 ? launch_tc<128>(a, workspace, bytes, s) : launch_tc<64>(a, workspace, bytes, s);
}

}  // namespace ab2
