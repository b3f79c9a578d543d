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
// 4096 tokens behind 12288, 32 / 8 heads of 128: 0.92 ms, 1.05 PFLOP/s, 0.63 of cuBLAS in a burst and 0.75 of it sustained; 2048 behind 2048 120 us;
// six rows of 1 to 512 tokens behind up to 5000 134 us; 4096 behind 12288, 16 / 4 heads of 64, 0.41 ms.  A tile of 80 keys takes some 2300 clocks, of which both tiles'
// exponentials (2 x 128 x 80, at 16 a clock) need 1280 and the products 1432; no pipe is full (1024 behind 3000 by counters: exponentials 42 %, tensor pipe 42 %, issue
// slots 36 %).  What bounds it is the chain of a softmax warp: scores from tensor memory, the maximum, the last tile's products, exponentials, weights back.
//
// Measured and not kept, each against the kernel of its day: the tiles' exponentials in turns by a barrier 0.98 ms for 0.91; polynomials for a quarter of
// them 0.96 for 0.91.  Forms before this one: tiles of 128 keys with the weights over the scores (a chain of scores, softmax and sums) 0.98 to 1.02;
// an MMA warp a tile there, weights handed over in two or four parts, 1.08 and 1.11; tiles of 64 with two places for weights 1.17, with registers spilled.
//
// An MMA multiplies a hidden value by a weight of 0, so an Inf or a NaN there would reach rows that do not see it.  Rows of a page behind the
// sequence's end are cleared in shared memory; a row whose sums come out as Inf or NaN (a later token's value may hold them) is computed
// again on CUDA cores over the keys in its sight, behind all pieces of the CTA, so that no bounded wait lasts as long as that.  Every wait on an mbarrier is bounded; on a time-out the CTA records AB2_ERR_TIMEOUT and
// walks through the rest of its work without waiting.
#include <algorithm>

#include "paged.cuh"
#include "tcgen05_util.cuh"

using namespace ab2;
using namespace ab2::tc;

namespace ab2 {
namespace {

constexpr int PC_Q = 128, PC_KEYS = 80, PC_THREADS = 384;
constexpr int PC_QBOX = PC_Q * 128, PC_BOX = PC_KEYS * 128;   // boxes of queries, and of keys or values: rows of 64 elements
constexpr int PC_ROWS = 16;   // that one copy brings: the least that a page holds
constexpr int PC_TWICE = 16;  // query rows of an item up to which it has each of them twice, for both terms of its weights
constexpr float PC_SLACK = 8.f;  // powers of two a score may exceed the row's maximum by
constexpr float PC_NONE = -1e30f;

template <int HD> struct PcShape {
    static constexpr int BOXES = HD / 64, QTILE = BOXES * PC_QBOX, TILE = BOXES * PC_BOX, SLOTS = HD == 128 ? 4 : 8;   // a slot holds a tile's keys and its values
    static constexpr int SMEM = 1024 + 2 * QTILE + SLOTS * 2 * TILE;
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
    int most;
};
__device__ __forceinline__ bool pc_next(const PagedPlan &a, PagedRun &run, PcPiece &x) {
    if (!paged_next(a, run, x.w)) return false;
    x.s = paged_span(a, x.w);
    const int rows = x.s.ntok * a.group;
    auto tiles = [&](int first, int end) {   // of rows [first, end) of the item: keys up to those of the last token
        const int last = min(x.s.hi, x.s.base + x.s.t0 + paged_token(a, end - 1) + 1);
        return end > first ? max(0, (last - x.s.lo + PC_KEYS - 1) / PC_KEYS) : 0;
    };
    x.first = tiles(0, min(rows, PC_Q));
    x.second = tiles(PC_Q, rows);
    x.most = max(x.first, x.second);
    return true;
}

struct PcShared {
    uint64_t full[8], empty[8], qfull[2], sfull[2], sfree[2], pfull[2], odone[2];
    uint32_t tmem_base;
    int failed;
    int2 found[2];
    union {
        long long warp_sums[PC_THREADS / 32];   // while the CTA looks for its run
        PagedRun start;                         // that run, from then on
    };
    // of every softmax warp: its run, the piece that it is at and the next one (kept from its registers, which the scores fill)
    PagedRun run[8];
    PcPiece piece[8][2];
};

// One tile of keys for the warp's 32 rows, a lane each: scores to weights.  With EDGE keys past `lim` are out of sight, and a lane that is `second` hands on what
// rounding left of each weight (a kind of its own for that cost the loops around it 5 %).  `before` waits until the
// products with the tile before are done: its weights' place is free then, and the sums stand still.
template <int HD, bool EDGE, class Before>
__device__ __forceinline__ void pc_softmax(uint32_t s_addr, uint32_t o_addr, float sl, bool flip, int lim, bool second, bool has_o, float &top, float &sum, uint64_t *taken, uint64_t *ready, Before before) {
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
#pragma unroll
    for (int k = 0; k < PC_KEYS; ++k)
        if (EDGE && k > lim) v(k) = 0xff800000u;
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
        uint32_t word = *reinterpret_cast<const uint32_t *>(&b);
        if (EDGE) {
            const __nv_bfloat162 left = __floats2bfloat162_rn(low(e) - __uint_as_float(word << 16), high(e) - __uint_as_float(word & 0xffff0000u));
            if (second) word = *reinterpret_cast<const uint32_t *>(&left);
        }
        return word;
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

template <int HD>
__global__ void __launch_bounds__(PC_THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedAttnArgs a) {
    using S = PcShape<HD>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PcShared sh;
    static_assert(S::SMEM + sizeof(PcShared) <= 227 * 1024, "shared memory of a CTA");
    uint8_t *qbuf = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023), *ring = qbuf + 2 * S::QTILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *failed = &sh.failed;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::SLOTS; ++i) { bar_init(&sh.full[i], 1); bar_init(&sh.empty[i], 2); }
        for (int i = 0; i < 2; ++i) { bar_init(&sh.qfull[i], 4); bar_init(&sh.sfull[i], 1); bar_init(&sh.sfree[i], 4); bar_init(&sh.pfull[i], 4); bar_init(&sh.odone[i], 1); }
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    pdl_wait();   // ahead of tensor memory too, which the launch before may hold
    PagedRun run = paged_run<PC_THREADS>(a.plan, blockIdx.x, a.ctas, sh.warp_sums, sh.found, a.status);
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
    // the block's registers: 128 threads of 72 and 256 of 216 are the 384 of 168 that it was launched with
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        if (warp == 0) {
            // ---------------------------------------------------------- TMA producer: K, V, K, V, ...
            int n = 0;
            while (pc_next(a.plan, run, x)) {
                for (int j = 0; j < x.most; ++j) {
                    const int key = x.s.lo + j * PC_KEYS + lane * PC_ROWS;
                    const bool mine = lane < PC_KEYS / PC_ROWS && key < x.s.hi;
                    const int page = mine ? paged_page(p, x.w.row, key, a.status) : 0;
                    const int bytes = __popc(__ballot_sync(0xffffffffu, mine)) * PC_ROWS * HD * 2;
                    const int slot = n % S::SLOTS;
                    warp_wait(&sh.empty[slot], ((n++ / S::SLOTS) & 1) ^ 1, failed);
                    // The first queries come before what is fetched ahead.  Only at the second slot of the run's first piece with keys, and only where the first
                    // tile of rows looks at it: its warps cannot announce their next queries without that slot, so the barrier is in its first phase or just
                    // behind it.  A later phase would have this parity again, and might wait for what is not yet fetched.
                    if (n == 2 && j == 1 && x.first > 1) warp_wait(&sh.qfull[0], 0, failed);
                    if (lane == 0) bar_expect_tx(&sh.full[slot], (uint32_t)(2 * bytes));
                    __syncwarp();
                    if (mine && !*failed)
#pragma unroll
                        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                            for (int b = 0; b < S::BOXES; ++b)
                                tma_load_3d(ring + (2 * slot + kv) * S::TILE + b * PC_BOX + lane * PC_ROWS * 128, kv ? &vmap : &kmap, b * 64, key & ((1 << p.page_shift) - 1), page * p.kv_heads + x.w.head, &sh.full[slot]);
                }
            }
        } else if (warp < 3) {
            // ---------------------------------------------------------- MMA issue for a tile of rows
            constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
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
#pragma unroll
                    for (int b = 0; b < S::BOXES; ++b) {
                        const uint64_t qd = umma_desc(sptr(qbuf + g * S::QTILE + b * PC_QBOX)), kd = umma_desc(sptr(ring + 2 * slot * S::TILE + b * PC_BOX));
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // descriptors count in 16 bytes
                            umma_bf16(s_at, qd + (uint64_t)(2 * k), kd + (uint64_t)(2 * k), S_DESC, (b | k) != 0);
                    }
                    umma_commit(&sh.sfull[g]);
                }
                __syncwarp();
                ++scored;
            };
            while (pc_next(a.plan, run, x)) {
                const int tiles = g ? x.second : x.first;
                if (tiles > 0) {
                    warp_wait(&sh.qfull[g], asked++ & 1, failed);
                    scores(n);
                }
                for (int j = 0; j < x.most; ++j, ++n) {
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
                        const uint64_t vd = umma_desc_mn(sptr(ring + (2 * slot + 1) * S::TILE), PC_BOX);
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
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
            while ((more = pc_next(a.plan, run, x))) {
                n0 = n;
                n += x.most;
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
        auto fetch_q = [&]() {
            const PcPiece &x = sh.piece[warp - 4][here];
            if ((g ? x.second : x.first) == 0) return;   // nothing to ask
            const PagedSpan s = x.s;
            const long long first = x.w.r.first + s.t0, head0 = x.w.head * group;
            const int i0 = threadIdx.x & 127, rows = s.ntok * group;
            const bool twice = rows <= PC_TWICE;
#pragma unroll
            for (int u = 0; u < PC_Q * HD / 8 / 128; ++u) {
                const int i = i0 + 128 * u, d = i % (HD / 8), row = i / (HD / 8), rr = twice && row < 2 * PC_TWICE ? row % PC_TWICE : g * PC_Q + row, in = rr < rows ? 16 : 0, tok = paged_token(a.plan, in ? rr : 0);
                const __nv_bfloat16 *src = (const __nv_bfloat16 *)a.q + (first + tok) * a.q_stride + (head0 + (in ? rr - tok * group : 0)) * HD + d * 8;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(sptr(qbuf + g * S::QTILE + (d >> 3) * PC_QBOX + row * 128 + (((d & 7) ^ (row & 7)) << 4))), "l"(src), "r"(in) : "memory");
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
        bool more = next(), again = false;   // again: a row's sums came out as Inf or NaN
        if (more) fetch_q();
        while (more) {
            const PcPiece &x = sh.piece[warp - 4][here];
            const int rows = x.s.ntok * group, tiles = g ? x.second : x.first, lo = x.s.lo, hi = x.s.hi, slot0 = n0;
            if (tiles > 0) {
                asm volatile("cp.async.wait_group 0;\n" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.qfull[g]);
            }
            const bool twice = rows <= PC_TWICE;   // and this the first tile of rows
            const bool second = twice && (lane & PC_TWICE);
            const int rr = g * PC_Q + r, asks = twice && r < 2 * PC_TWICE ? r % PC_TWICE : rr, pos = asks < rows ? x.s.base + x.s.t0 + paged_token(a.plan, asks) : -1;
            const int least = x.s.base + x.s.t0 + paged_token(a.plan, g * PC_Q);   // the first row sees up to here
            float top = PC_NONE, sum = 0.f;
            for (int j = 0; j < tiles; ++j, ++scored) {
                const int at = lo + j * PC_KEYS;
                warp_wait(&sh.sfull[g], scored & 1, failed);
                if (at + PC_KEYS > hi) {   // what lies behind the piece's keys may be anything
                    // Behind the wait for the scores, never ahead of it: these warps pass over pieces without rows of theirs, and the slot's barrier may still be phases
                    // away from the one meant, with the same parity.
                    const int slot = (slot0 + j) % S::SLOTS;
                    warp_wait(&sh.full[slot], ((slot0 + j) / S::SLOTS) & 1, failed);
                    if (at + r >= hi && r < PC_KEYS)
#pragma unroll
                        for (int b = 0; b < S::BOXES; ++b)
#pragma unroll
                            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4 *>(ring + (2 * slot + 1) * S::TILE + b * PC_BOX + r * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();   // and the products wait for all four warps
                }
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const int lim = min(pos, hi - 1) - at;
                auto before = [&] { if (j > 0) warp_wait(&sh.odone[g], (scored - 1) & 1, failed); };
                if (at + PC_KEYS - 1 > least || at + PC_KEYS > hi || (g + 1) * PC_Q > rows) pc_softmax<HD, true>(s_addr, o_addr, sl, flip, lim, second, j > 0, top, sum, &sh.sfree[g], &sh.pfull[g], before);
                else pc_softmax<HD, false>(s_addr, o_addr, sl, flip, lim, false, j > 0, top, sum, &sh.sfree[g], &sh.pfull[g], before);
            }
            // the scores are all made: the next piece's queries may take the place of these, while the sums go out
            more = next();
            if (more) fetch_q();
            const PagedPiece w = x.w;
            const PagedSpan s = x.s;
            if (tiles > 0) warp_wait(&sh.odone[g], (scored - 1) & 1, failed);
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const bool all = w.k0 == 0 && w.k1 == w.k_tiles;
            const size_t slot = (2 * (size_t)blockIdx.x + (w.k0 == 0)) * a.tile_rows;
            const float f = !all ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
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
        if (again) {
            PagedRun walk = sh.start;
            PcPiece x;
            while (pc_next(a.plan, walk, x)) {
                const int rr = g * PC_Q + r, rows = x.s.ntok * group;
                if (rows <= g * PC_Q) continue;
                const bool all = x.w.k0 == 0 && x.w.k1 == x.w.k_tiles;
                const size_t slot = (2 * (size_t)blockIdx.x + (x.w.k0 == 0)) * a.tile_rows;
                uint32_t worst = 0;   // of the exponents
                if (rr < rows) {
                    const int tok = paged_token(a.plan, rr);
                    const uint32_t *o = all ? (const uint32_t *)((const __nv_bfloat16 *)a.out + (size_t)(x.w.r.first + x.s.t0 + tok) * a.o_stride + (size_t)(x.w.head * group + rr - tok * group) * HD)
                                            : (const uint32_t *)(a.acc + (slot + rr) * HD);
                    for (int i = 0; i < (all ? HD / 2 : HD); ++i) {
                        worst = max(worst, o[i] & 0x7f800000u);
                        if (all) worst = max(worst, (o[i] & 0x7f80u) << 16);
                    }
                }
                for (uint32_t left = __ballot_sync(0xffffffffu, worst == 0x7f800000u); left; left &= left - 1)
                    paged_again<HD>(a, x.w, x.s, g * PC_Q + quad * 32 + __ffs(left) - 1, lane, all, slot);
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

template <int HD>
int launch_tc(PagedAttnArgs a, void *workspace, size_t bytes, cudaStream_t s) {
    using S = PcShape<HD>;
    static bool configured[64] = {false};  // the attribute is per device
    int dev = 0;
    AB2_CUDA(cudaGetDevice(&dev));
    AB2_REQUIRE(dev >= 0 && dev < 64, AB2_ERR_BAD_ARG, "device index %d out of range", dev);
    if (!configured[dev]) {
        AB2_CUDA(cudaFuncSetAttribute(paged_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        configured[dev] = true;
    }
    CUtensorMap kmap, vmap;
    int rc = pages_map(&kmap, a.k, a.plan.p, HD);
    if (rc == AB2_OK) rc = pages_map(&vmap, a.v, a.plan.p, HD);
    if (rc != AB2_OK) return rc;
    paged_deal(a, device_sm_count(), 2 * PC_Q, 7, 4, HD, workspace, bytes);
    // Set up while the launch before it ends, up to 65536 query rows: all that were tried gain there, and beyond it none does and the longest loses.  32 heads of 128, us
    // not set up early and early: 300 tokens behind 300 35.0 and 32.6, behind 16000 103 and 101.4, 1024 behind 1024 53.7 and 51.9, 2048 alone 82.0 and 80.9, behind
    // 12288 383.8 and 382.6; 3000 behind 3000 231 to 240 and 233 to 237, 4096 alone 207 and 207 to 210, behind 4096 372 and 371, behind 12288 860 to 872 and 876 to 884, 8192 alone 617 and 613 to 621.
    ChainedLaunches chained((long long)a.plan.p.tokens * a.plan.group * a.plan.p.kv_heads <= 65536);
    AB2_CUDA(launch_kernel(paged_tc_kernel<HD>, dim3(a.ctas), dim3(PC_THREADS), S::SMEM, s, kmap, vmap, a));
    return a.plan.whole ? AB2_OK : paged_merge(a, HD, AB2_BF16, s);
}

}  // namespace

size_t paged_tc_bytes(int hd) { return paged_piece_bytes(device_sm_count(), 2 * PC_Q, hd); }
int paged_tc_attention(const PagedAttnArgs &a, int hd, void *workspace, size_t bytes, cudaStream_t s) {
    return hd == 128 ? launch_tc<128>(a, workspace, bytes, s) : launch_tc<64>(a, workspace, bytes, s);
}

}  // namespace ab2
