// Attention of single tokens and short runs of them over a paged bf16 cache: rows whose new tokens times the query heads of a KV head are at
// most 16.  The mathematics is that of attention_paged.cu.
//
// Bound by HBM: every key and value is read once for up to 16 query rows.  Each warp has an equal run of all keys to itself (paged.cuh) and
// a ring of 16-key blocks, filled by cp.async as far ahead as shared memory goes, across the ends of pieces, rows and heads; no warp waits
// for another.  Products are warp-level MMAs with the keys as rows, so that 8 query rows a tile are enough:
//
//   S^T[16 keys][8 rows] = K . Q^T        K by ldmatrix, Q^T in registers
//   O^T[dim][8 rows]    += V^T . P^T      V^T by ldmatrix.trans, P^T from S^T's registers by movmatrix
//
// Weights enter as two bf16 terms, the rounded weight and what rounding left: the tensor pipe has time for both, and no rounding but the
// output's is left.  A row's maximum moves only when a score exceeds it by 2^8.
//
// 48 rows of up to 8192 tokens, 32 / 8 heads of 128 (1.02 GB): 170 us with the merge, 0.92 of a copy's rate (on CUDA cores 672); 2 x 100000 128 to 138 us
// (0.89 to 0.83 by the card).  1 x 700: 10.3 to 10.9 us (12.3 to 12.7 before a launch was set up while the one before it ended), a kernel of 8 and a merge of 4.3 by themselves:
// latency.  Through a window of 2048 with 4 first tokens, 32 rows of 30000: 55 us, 0.75 of a copy's rate.
//
// Over codes (e4m3) a code is an f16 number as it is, and products are of f16: queries times a power of two of their row's that brings the largest to 2^14 to 2^15 (exact but for
// elements below 2^-28 of it), a block's scale of keys on its scores, its scale of values on its weights, relative to `vref`, a scale that moves as the maximum does.
// Weights have one f16 term (2^-11): the output's rounding is 2^-8, and the conversions leave the pipes no time for a second.  48 rows of up to 8192: 94 us,
// 0.83 of a copy's rate for half the bytes (bf16 pages 164); 2 x 100000 73; 64 rows of 12000 through a window of 1024, 16 / 4 heads, 26.5; 1 x 700: 10.7.
// A merge by fewer CTAs, each for the cuts of several runs, took 80 us for 41 at 1 x 32000: cuts lie evenly apart, and met in the same CTAs.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

using namespace ab2;

namespace ab2 {
namespace {

constexpr int PM_WARPS = 4, PM_KEYS = 16;
constexpr float PM_SLACK = 8.f, PM_NONE = -1e30f;
constexpr float PM_UP = 128.f, PM_LESS = 9.765625e-4f, PM_NOTHING = 8.6736174e-19f;   // E8: weights as f16 are this much larger, at most 2^15; 2^-10 and 2^-60

template <int HD, bool E8> struct PmShape {
    static constexpr int ROW = HD * (E8 ? 1 : 2), BLOCK = 2 * PM_KEYS * ROW;          // bytes of a row, and of a block's keys and values
    static constexpr int STAGES = (HD == 128 ? 3 : 6) * (E8 ? 2 : 1), SMEM = PM_WARPS * STAGES * BLOCK;   // 96 KB: two CTAs an SM
    // where chunk ch (16 bytes) of row r lies: eight rows' chunks meet in no bank
    static __device__ __forceinline__ int at(int r, int ch) { return r * ROW + ((ch ^ (ROW == 64 ? (r >> 1) & 3 : r & 7)) << 4); }
};

__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float pm_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 b = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}

template <int HD, int NT, bool E8, bool WIN>  // NT tiles of 8 query rows; pages of e4m3; a window
__global__ void __launch_bounds__(32 * PM_WARPS, 2) paged_mma_kernel(const __grid_constant__ PagedAttnArgs a) {
    using S = PmShape<HD, E8>;
    using Page = std::conditional_t<E8, uint8_t, __nv_bfloat16>;
    constexpr int KS = HD / 16, ROW = S::ROW, CH = ROW / 16, STAGES = S::STAGES, LOADS = PM_KEYS * CH / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int2 found[PM_WARPS][2];
    __shared__ float2 scales[E8 ? PM_WARPS : 1][E8 ? STAGES : 1];   // of the keys and the values of a stage
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, group = a.plan.group;
    const PagedView &p = a.plan.p;
    uint8_t *ring = smem + warp * STAGES * S::BLOCK;
    const int me = warp * gridDim.x + blockIdx.x;   // a little work spreads over all SMs
    PagedRun run = paged_run<32, WIN>(a.plan, me, a.ctas, nullptr, found[warp], a.status);
    if (lane == 0) paged_uncut(a, me);

    // ---- the copies run ahead of the products, over the same pieces
    PagedRun ahead = run;
    PagedPiece aw = {};
    PagedSpan as = {};
    PagedHole ah = {};
    int akey = 0, apage = 0;   // the next block's first key, and its page (-1: a block that no token sees, of zeros)
    bool more = true;
    auto look = [&]() {
        const int key = WIN ? paged_key(ah, akey) : akey;
        apage = WIN && paged_hidden(a.plan, as, key, PM_KEYS) ? -1 : paged_page(p, aw.row, key, a.status);
    };
    auto seek = [&]() {        // the first block of the next piece that has keys
        for (;;) {
            if (!paged_next<WIN>(a.plan, ahead, aw)) { more = false; return; }
            as = paged_span<WIN>(a.plan, aw);
            if (WIN) ah = paged_hole(a.plan, as.base, aw.q_tile);
            akey = as.lo;
            if (akey < as.hi) break;
        }
        look();
    };
    auto fetch = [&](int stage) {
        if (more) {
            const int key = WIN ? paged_key(ah, akey) : akey;
            const bool hidden = WIN && apage < 0;
            const size_t row = (((size_t)(hidden ? 0 : apage) * p.kv_heads + aw.head) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
            const uint8_t *k = (const uint8_t *)a.k + row * ROW, *v = (const uint8_t *)a.v + row * ROW;
            const uint32_t at = smem_at(ring + stage * S::BLOCK);
            const int left = hidden ? 0 : as.hi - akey;   // rows past the last key are zeros
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = (lane + 32 * i) / CH, ch = (lane + 32 * i) % CH, in = r < left ? 16 : 0, from = r < left ? r : 0;
                const uint32_t dst = at + S::at(r, ch);
                asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(k + from * ROW + ch * 16), "r"(in) : "memory");
                asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;\n" ::"r"(dst + PM_KEYS * ROW), "l"(v + from * ROW + ch * 16), "r"(in) : "memory");
            }
            if (E8 && lane < 2)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(smem_at(&scales[warp][stage]) + 4 * lane), "l"((lane ? a.v_scales : a.k_scales) + row / PAGED_BLOCK), "r"(hidden ? 0 : 4) : "memory");
            akey += PM_KEYS;
            if (akey < as.hi) look();
            else seek();
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    if (run.u < run.u1) seek();
    else more = false;
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);

    int stage = 0;
    PagedPiece w;
    while (paged_next<WIN>(a.plan, run, w)) {
        const PagedSpan sp = paged_span<WIN>(a.plan, w);
        const int gap = paged_hole<WIN>(a.plan, sp.base, w.q_tile).gap;
        if (lane == 0) paged_cut(a, run, w, sp, me);
        const int rows = sp.ntok * group;
        // rows of the tile: 8 t + g as columns of Q^T, 8 t + 2 c and 8 t + 2 c + 1 as columns of scores and sums
        uint32_t q[NT][KS][2];
        int lim[NT][2];
        float top[NT][2], sum[NT][2], o[KS][NT][4];
        float qsl[NT][2];      // E8: what a column's products are multiplied by, but for the block's scale
        float vref = 0.f, vinv = 0.f;   // E8: the sums are in units of this scale of values; PM_UP by it
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = 8 * t + g, tok = paged_token(a.plan, r);
            const uint32_t *src = (const uint32_t *)((const __nv_bfloat16 *)a.q + (size_t)(w.r.first + sp.t0 + tok) * a.q_stride + (size_t)(w.head * group + r - tok * group) * HD);
            if constexpr (E8) {
                // Elements 4 c .. 4 c + 3 of each 16 stand for 2 c, 2 c + 1, 2 c + 8 and 2 c + 9, as those of the keys do.  As f16, the row's largest between 2^14 and
                // 2^15: exact for all that are not 2^-28 of it or less.
                uint2 x[KS];
                float most = 0.f;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    x[s] = r < rows ? *reinterpret_cast<const uint2 *>(src + 8 * s + 2 * c) : make_uint2(0u, 0u);
                    most = fmaxf(fmaxf(most, fmaxf(fabsf(__uint_as_float(x[s].x << 16)), fabsf(__uint_as_float(x[s].x & 0xffff0000u)))),
                                 fmaxf(fabsf(__uint_as_float(x[s].y << 16)), fabsf(__uint_as_float(x[s].y & 0xffff0000u))));
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const int up = min(max(268 - (int)(__float_as_uint(most) >> 23), 1), 253);
                const float f = __uint_as_float((uint32_t)up << 23), back = __uint_as_float((uint32_t)(254 - up) << 23) * a.sl;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    q[t][s][0] = pack_f16(__uint_as_float(x[s].x << 16) * f, __uint_as_float(x[s].x & 0xffff0000u) * f);
                    q[t][s][1] = pack_f16(__uint_as_float(x[s].y << 16) * f, __uint_as_float(x[s].y & 0xffff0000u) * f);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) qsl[t][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * c + e));
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    q[t][s][0] = r < rows ? src[8 * s + c] : 0u;
                    q[t][s][1] = r < rows ? src[8 * s + c + 4] : 0u;
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = 8 * t + 2 * c + e;
                lim[t][e] = col < rows ? sp.base + sp.t0 + paged_token(a.plan, col) - gap : 0x7fffffff;   // a column without a row is not looked at
                top[t][e] = PM_NONE;
                sum[t][e] = 0.f;
            }
#pragma unroll
            for (int m = 0; m < KS; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][t][e] = 0.f;
        }
        const int sure = min(sp.hi, sp.base + sp.t0 + 1 - gap);   // keys that every column sees, but for those that a window hides: ahead of `late`, behind the sinks
        const int late = WIN ? sp.base + sp.t0 + sp.ntok - a.plan.window - gap : 0;
#pragma unroll 1
        for (int key = sp.lo; key < sp.hi; key += PM_KEYS) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
            __syncwarp();   // the block has come for all lanes, and all have left the one before, which is filled anew
            fetch(stage == 0 ? STAGES - 1 : stage - 1);
            const uint32_t at = smem_at(ring + stage * S::BLOCK);
            const float2 bs = E8 ? scales[warp][stage] : make_float2(1.f, 1.f);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            // ---- scores: rows of K are keys
            float s[NT][4], s2[NT][4];   // two sums, so that a product waits for every other one only
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] = s2[t][e] = 0.f;
            if constexpr (E8) {
#pragma unroll
                for (int k = 0; k < KS; k += 2) {
                    uint32_t f[4];
                    ldsm4(f, at + S::at(lane & 15, k + (lane >> 4)));   // rows g and g + 8, four codes each, of chunks k and k + 1
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x[4] = {f16x2_of_codes(f[2 * h]), f16x2_of_codes(f[2 * h + 1]), f16x2_of_codes(f[2 * h] >> 16), f16x2_of_codes(f[2 * h + 1] >> 16)};
#pragma unroll
                        for (int t = 0; t < NT; ++t) mma_f16(h ? s2[t] : s[t], x, q[t][k + h][0], q[t][k + h][1]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t f[4];
                    ldsm4(f, at + S::at(lane & 15, 2 * k + (lane >> 4)));
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_bf16(k & 1 ? s2[t] : s[t], f, q[t][k][0], q[t][k][1]);
                }
            }
            // ---- weights
            uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] = (s[t][e] + s2[t][e]) * (E8 ? qsl[t][e & 1] * bs.x : a.sl);
                if (key + PM_KEYS > sure)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (key + g + 8 * (e >> 1) > min(lim[t][e & 1], sp.hi - 1)) s[t][e] = -INFINITY;
                if (WIN && key < late && key + PM_KEYS > a.plan.sinks)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int k = key + g + 8 * (e >> 1);
                        if (k >= a.plan.sinks && k <= lim[t][e & 1] - a.plan.window) s[t][e] = -INFINITY;
                    }
            }
            bool moves = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) moves |= s[t][e] > top[t][e & 1] + PM_SLACK;
            if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float corr[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float best = fmaxf(s[t][e], s[t][e + 2]);
#pragma unroll
                        for (int m = 4; m < 32; m <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, m));
                        best = fmaxf(top[t][e], best);
                        corr[e] = pm_ex2(top[t][e] - best);
                        top[t][e] = best;
                        sum[t][e] *= corr[e];
                    }
#pragma unroll
                    for (int m = 0; m < KS; ++m) { o[m][t][0] *= corr[0]; o[m][t][1] *= corr[1]; o[m][t][2] *= corr[0]; o[m][t][3] *= corr[1]; }
                }
            }
            float vs = 0.f;
            if constexpr (E8) {
                // The unit moves to a block's scale that is larger, or so much smaller that f16 would lose bits of its weights (but not to one whose values are
                // nothing beside the others, as of a block of zeros).  The same for all lanes.
                if (bs.y > vref || (bs.y < vref * PM_LESS && bs.y > vref * PM_NOTHING)) {
                    const float to = fmaxf(bs.y, 3.0092655e-36f), f = vref / to;   // 2^-118 at least, and the sums move by what the unit does
                    vref = to;
                    vinv = PM_UP / vref;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int m = 0; m < KS; ++m)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[m][t][e] *= f;
                }
                vs = bs.y * vinv;
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] = pm_ex2(s[t][e] - top[t][e & 1]);
                    sum[t][e & 1] += s[t][e];
                    if (E8) s[t][e] *= vs;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // keys 0 to 7 and 8 to 15
                    if constexpr (E8) {
                        hi[t][h] = transposed(pack_f16(s[t][2 * h], s[t][2 * h + 1]));
                        continue;
                    }
                    const uint32_t x = pack_bf16(s[t][2 * h], s[t][2 * h + 1]);
                    const uint32_t y = pack_bf16(s[t][2 * h] - __uint_as_float(x << 16), s[t][2 * h + 1] - __uint_as_float(x & 0xffff0000u));
                    hi[t][h] = transposed(x);
                    lo[t][h] = transposed(y);
                }
            }
            // ---- sums: rows of V^T are dimensions
            if constexpr (E8) {
#pragma unroll
                for (int m = 0; m < KS; m += 2) {
                    uint32_t f[4];
                    ldsm4_t(f, at + PM_KEYS * ROW + S::at(lane & 15, m + (lane >> 4)));   // dimensions 2 g and 2 g + 1 of keys 2 c and 2 c + 1, + 8, of chunks m and m + 1
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x0 = __byte_perm(f[2 * h], 0u, 0x3120), x1 = __byte_perm(f[2 * h + 1], 0u, 0x3120);   // a dimension's two keys side by side
                        const uint32_t x[4] = {f16x2_of_codes(x0), f16x2_of_codes(x0 >> 16), f16x2_of_codes(x1), f16x2_of_codes(x1 >> 16)};
#pragma unroll
                        for (int t = 0; t < NT; ++t) mma_f16(o[m + h][t], x, hi[t][0], hi[t][1]);
                    }
                }
            } else {
#pragma unroll
                for (int m = 0; m < KS; ++m) {
                    uint32_t f[4];
                    ldsm4_t(f, at + PM_KEYS * ROW + S::at((lane & 7) + ((lane >> 4) << 3), 2 * m + ((lane >> 3) & 1)));
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_bf16(o[m][t], f, hi[t][0], hi[t][1]);
                        mma_bf16(o[m][t], f, lo[t][0], lo[t][1]);
                    }
                }
            }
        }
        // ---- the piece's end
        const bool all = w.k0 == 0 && w.k1 == w.k_tiles;
        const size_t slot = (2 * (size_t)me + (w.k0 == 0)) * a.tile_rows;
        uint32_t poisoned = 0;   // rows whose sums are Inf or NaN
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int m = 4; m < 32; m <<= 1) sum[t][e] += __shfl_xor_sync(0xffffffffu, sum[t][e], m);
                f[e] = !all ? 1.f : sum[t][e] == 0.f ? 0.f : 1.f / sum[t][e];
                if (E8) f[e] *= vref / PM_UP;
            }
            float poison[2] = {0.f, 0.f};
#pragma unroll
            for (int m = 0; m < KS; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[m][t][e] *= f[e & 1];
                    poison[e & 1] = fmaf(o[m][t][e], 0.f, poison[e & 1]);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t b = __ballot_sync(0xffffffffu, poison[e] != 0.f);   // NaN is not 0
                b |= b >> 16; b |= b >> 8; b |= b >> 4;                     // by c
#pragma unroll
                for (int i = 0; i < 4; ++i) poisoned |= ((b >> i) & 1) << (8 * t + 2 * i + e);
            }
            if (all && E8) {
                const int r = 8 * t + g, tok = paged_token(a.plan, r);
                __nv_bfloat16 *dst = (__nv_bfloat16 *)a.out + (size_t)(w.r.first + sp.t0 + tok) * a.o_stride + (size_t)(w.head * group + r - tok * group) * HD + 4 * c;
#pragma unroll
                for (int m = 0; m < KS; ++m) {   // rows 2 c and 2 c + 1 are dimensions 4 c and 4 c + 2, with 8 more 4 c + 1 and 4 c + 3
                    const uint32_t x = transposed(pack_bf16(o[m][t][0], o[m][t][1])), y = transposed(pack_bf16(o[m][t][2], o[m][t][3]));
                    if (r < rows) *reinterpret_cast<uint2 *>(dst + 16 * m) = make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
                }
            } else if (all) {
#pragma unroll
                for (int m = 0; m < KS; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x = transposed(pack_bf16(o[m][t][2 * h], o[m][t][2 * h + 1]));   // row 8 t + g, dimensions 2 c and 2 c + 1 of the 8
                        const int r = 8 * t + g, tok = paged_token(a.plan, r);
                        if (r < rows) *reinterpret_cast<uint32_t *>((__nv_bfloat16 *)a.out + (size_t)(w.r.first + sp.t0 + tok) * a.o_stride + (size_t)(w.head * group + r - tok * group) * HD + 16 * m + 8 * h + 2 * c) = x;
                    }
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * t + 2 * c + e;
                    if (r >= rows) continue;
#pragma unroll
                    for (int m = 0; m < KS; ++m) {
                        if (E8) {
                            *reinterpret_cast<float2 *>(a.acc + (slot + r) * HD + 16 * m + 2 * g) = make_float2(o[m][t][e], o[m][t][e + 2]);
                            continue;
                        }
                        a.acc[(slot + r) * HD + 16 * m + g] = o[m][t][e];
                        a.acc[(slot + r) * HD + 16 * m + 8 + g] = o[m][t][e + 2];
                    }
                    if (g == 0) *reinterpret_cast<float2 *>(a.ml + (slot + r) * 2) = make_float2(top[t][e], sum[t][e]);
                }
            }
        }
        __syncwarp();
        for (poisoned &= rows >= 32 ? 0xffffffffu : (1u << rows) - 1; poisoned; poisoned &= poisoned - 1) paged_again<HD, Page, WIN>(a, w, sp, __ffs(poisoned) - 1, lane, all, slot);
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
}

int mma_runs() { return 2 * PM_WARPS * device_sm_count(); }

template <int HD, int NT, bool E8, bool WIN>
int launch_mma(PagedAttnArgs a, void *workspace, size_t bytes, cudaStream_t s) {
    using S = PmShape<HD, E8>;
    static bool configured[64] = {false};  // the attribute is per device
    int dev = 0;
    AB2_CUDA(cudaGetDevice(&dev));
    AB2_REQUIRE(dev >= 0 && dev < 64, AB2_ERR_BAD_ARG, "device index %d out of range", dev);
    if (!configured[dev]) {
        AB2_CUDA(cudaFuncSetAttribute(paged_mma_kernel<HD, NT, E8, WIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        configured[dev] = true;
    }
    paged_deal(a, mma_runs(), 8 * NT, 6, 1, HD, workspace, bytes);
    ChainedLaunches chained(true);   // set up while the launch before it ends
    AB2_CUDA(launch_kernel(paged_mma_kernel<HD, NT, E8, WIN>, dim3(a.ctas / PM_WARPS), dim3(32 * PM_WARPS), S::SMEM, s, a));
    return a.plan.whole ? AB2_OK : paged_merge(a, HD, AB2_BF16, s);
}
template <int HD, int NT>
int launch_mma(const PagedAttnArgs &a, void *workspace, size_t bytes, cudaStream_t s) {
    if (a.plan.window) return a.k_scales ? launch_mma<HD, NT, true, true>(a, workspace, bytes, s) : launch_mma<HD, NT, false, true>(a, workspace, bytes, s);
    return a.k_scales ? launch_mma<HD, NT, true, false>(a, workspace, bytes, s) : launch_mma<HD, NT, false, false>(a, workspace, bytes, s);
}

}  // namespace

size_t paged_mma_bytes(int hd) { return paged_piece_bytes(mma_runs(), 16, hd); }
int paged_mma_attention(const PagedAttnArgs &a, int hd, int max_new, void *workspace, size_t bytes, cudaStream_t s) {
    const bool one = (long long)max_new * a.plan.group <= 8;
    if (hd == 128) return one ? launch_mma<128, 1>(a, workspace, bytes, s) : launch_mma<128, 2>(a, workspace, bytes, s);
    return one ? launch_mma<64, 1>(a, workspace, bytes, s) : launch_mma<64, 2>(a, workspace, bytes, s);
}

}  // namespace ab2
