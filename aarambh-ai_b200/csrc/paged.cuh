// Paged caches as kernels receive them, and the turning of a pair by a position (internal header).
#pragma once

#include "common.cuh"

namespace ab2 {

int device_status_word(int **out);
int device_sm_count();
int paged_check(const ab2_paged *c, ab2_dtype dtype);
int append_check(const ab2_paged *cache, long long page_es, const void *k_dev, long long k_stride, const void *v_dev, long long v_stride, const void *q_dev, long long q_stride, int heads, void *q_out_dev,
                 long long q_out_stride, const double *frequencies_dev, int rot_dims, int layout, ab2_dtype dtype);

// What deals work out is compiled for the host too, where tests/test_paged_plan.py runs it over batches of all kinds.

// What a ragged batch of new tokens says of a row, with everything that device memory could hold brought within bounds: row b's new tokens
// are [first, first + count) of q, k and v, and its last one is at position len - 1.
struct PagedRow {
    int first, count, len;
};
struct PagedView {
    const int *table, *lens, *starts;
    long long table_stride;
    int rows, tokens, width, pages, page_shift, kv_heads;
};
PagedView paged_view(const ab2_paged *c);
__host__ __device__ __forceinline__ void paged_bad(int *status) {
#ifdef __CUDA_ARCH__
    atomicCAS(status, 0, (int)AB2_ERR_BAD_ARG);
#else
    *status = (int)AB2_ERR_BAD_ARG;
#endif
}
__host__ __device__ __forceinline__ PagedRow paged_row(const PagedView &p, int b, int *status) {
    PagedRow r;
    const int s0 = p.starts ? p.starts[b] : b, s1 = p.starts ? p.starts[b + 1] : b + 1, len = p.lens[b];
    r.first = min(max(s0, 0), p.tokens);
    r.count = min(max(s1, r.first), p.tokens) - r.first;
    r.len = (int)min((long long)max(len, 0), (long long)p.width << p.page_shift);
    if (status && (r.first != s0 || r.first + r.count != s1 || r.len != len)) paged_bad(status);
    return r;
}
// The page that holds position pos (less than the row's bounded length) of row b.  An entry outside the pool is recorded and read as page 0.
__device__ __forceinline__ int paged_page(const PagedView &p, int b, int pos, int *status) {
    const int id = __ldg(p.table + b * p.table_stride + (pos >> p.page_shift));
    if ((unsigned)id < (unsigned)p.pages) return id;
    paged_bad(status);
    return 0;
}

// ---- pages of 8 bits: e4m3 codes, and a scale for every PAGED_BLOCK tokens of a head ([pages][kv_heads][page_size / PAGED_BLOCK] f32); a value is its code times
// its scale.
constexpr int PAGED_BLOCK = 16;
__device__ __forceinline__ uint32_t f16x2_of_codes(uint32_t two) {   // of the lower 16 bits, exactly
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(d) : "h"((uint16_t)two));
    return d;
}
__device__ __forceinline__ float2 floats_of_codes(uint32_t two) {
    const uint32_t h = f16x2_of_codes(two);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
__device__ __forceinline__ uint32_t codes_of(float lo, float hi) {   // the nearest, up to 448
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t codes_of(__half2 x) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;\n" : "=h"(d) : "r"(*reinterpret_cast<const uint32_t *>(&x)));
    return d;
}
// 16 bytes of a row of keys or values as floats, to be scaled where they are codes.
template <typename P> struct PagedChunk {   // bf16: 8 elements
    static constexpr int N = 8;
    static __device__ __forceinline__ void floats(uint4 x, float (&y)[N]) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { y[2 * i] = __uint_as_float(w[i] << 16); y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ float one(P x) { return to_f32(x); }
};
template <> struct PagedChunk<uint8_t> {
    static constexpr int N = 16;
    static __device__ __forceinline__ void floats(uint4 x, float (&y)[N]) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) { const float2 f = floats_of_codes(w[i >> 1] >> (16 * (i & 1))); y[2 * i] = f.x; y[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ float one(uint8_t x) { return floats_of_codes(x).x; }
};

// ---- rotary positions
// A pair (x, y) at position p turns by the angle p f: (x cos - y sin, x sin + y cos), times a magnitude.  Only the fraction of a turn
// matters, so f becomes turns per position as a 64-bit fraction of a turn, and p times it wraps by itself: the angle of position
// 2^20 is as exact as that of position 1 (an error of p 2^-54 turns from f, in f64, is all there is), where an f32 product would be off by
// 2^20 2^-24 radians.
__device__ __forceinline__ unsigned long long turns_per_position(double f) {
    const double t = f * 0.15915494309189535;  // 1 / (2 pi)
    return __double2ull_rn((t - floor(t)) * 18446744073709551616.0);
}
// cos and sin of `a` 2^-64 turns, times m.  The nearest quarter turn goes by the top bits; what is left, an eighth of a turn at most either way,
// is a whole number of up to 2^29 units of 2^-31 half turns, and keeps 24 bits as a float: off by 2^4 units at most there, 2^-25.3 radians (cutting the bits below a
// unit off takes 2^-29.3 more).
__device__ __forceinline__ void turn_cos_sin(unsigned long long a, float m, float &c, float &s) {
    const unsigned q = (unsigned)((a + (1ull << 61)) >> 62);
    const int left = (int)((long long)(a - ((unsigned long long)q << 62)) >> 32);
    float s0, c0;
    sincospif((float)left * 4.656612873077393e-10f, &s0, &c0);  // 2^-31: halves of a turn
    const float cq = (q & 1) ? s0 : c0, sq = (q & 1) ? c0 : s0;
    c = m * (((q + 1) & 2) ? -cq : cq);
    s = m * ((q & 2) ? -sq : sq);
}

// ---- attention over a paged cache: how the work is dealt out
// An item is a tile of 2^tq_shift of a row's new tokens, with all query heads of one KV head, against the keys that they see; a unit is 2^key_shift
// of those keys.  Every CTA of a launch takes an equal run of the units of all rows, whose lengths only the device knows (so a recorded
// launch serves other lengths when it runs again).  An item that one CTA has to itself is finished there; the pieces of one that is cut meet in
// the merge kernel.  A piece that does not begin its item is its CTA's first: slot 2 c; one that begins it and does not end it is its last: slot 2 c + 1.
// Without room for pieces items are not cut.  A launch serves the rows whose new tokens times query heads a KV head are above `above` and
// at most `most`.
struct PagedPlan {
    PagedView p;
    int tq_shift, key_shift, whole, group, above, most;
    int least;                  // units that are worth a CTA
    int per_group;              // 2^16 / group, rounded up: r / group is r per_group / 2^16 for rows r of a tile (at most 256) and groups up to 32
    int window, sinks;          // a token sees its row's last `window` keys (0: all) and the first `sinks`
};
__host__ __device__ __forceinline__ int paged_token(const PagedPlan &a, int r) { return (r * a.per_group) >> 16; }
struct PagedShape {
    int q_tiles, base;          // of the row; keys before its new tokens, negative where those are more than its keys
    long long per;              // units of a head
    long long units;
};
// The sum over x < y of floor(x / 2^s).
__host__ __device__ __forceinline__ long long paged_floors(long long y, int s) {
    const long long q = y >> s;
    return (q * (q - 1) / 2 << s) + q * (y & ((1ll << s) - 1));
}
// WIN: for kernels that are compiled without windows.  Through a window a tile of queries sees two runs of units: those of the sinks, and those from its first token's window on.  The units between are left
// out, and the tile's units are numbered as if there were none ("virtual" keys: those behind the sinks' units, less what is left out).
__host__ __device__ __forceinline__ long long paged_sink_units(const PagedPlan &a) { return ((long long)a.sinks + (1 << a.key_shift) - 1) >> a.key_shift; }
template <bool WIN = true> __host__ __device__ __forceinline__ int paged_gap(const PagedPlan &a, int base, int q_tile) {   // units between
    if (!WIN || !a.window) return 0;
    const long long y = (long long)base + ((long long)q_tile << a.tq_shift) - a.window + 1, gap = (y >> a.key_shift) - paged_sink_units(a);
    return gap > 0 ? (int)gap : 0;
}
template <bool WIN = true> __host__ __device__ __forceinline__ long long paged_gaps(const PagedPlan &a, int base, long long n) {   // their sum over the first n tiles
    if (!WIN || !a.window) return 0;
    const long long sinks = paged_sink_units(a), y = (long long)base - a.window + 1, from = ((sinks + 1) << a.key_shift) - y;   // tile i has some where i tq >= from
    const long long first = from > 0 ? (from + (1 << a.tq_shift) - 1) >> a.tq_shift : 0, m = n - first, y0 = y + (first << a.tq_shift);
    if (m <= 0) return 0;
    const int s = a.key_shift - a.tq_shift;
    if (s <= 0) return m * ((y0 >> a.key_shift) - sinks) + ((m * (m - 1) / 2) << -s);
    const long long c = y0 >> a.tq_shift;
    return paged_floors(c + m, s) - paged_floors(c, s) - m * sinks;
}
template <bool WIN = true> __host__ __device__ __forceinline__ int paged_keys(const PagedPlan &a, int base, int q_tile) {   // units of a tile of queries
    return a.whole ? 1 : (int)((max(base, 0) + ((long long)(q_tile + 1) << a.tq_shift) + (1 << a.key_shift) - 1) >> a.key_shift) - paged_gap<WIN>(a, base, q_tile);
}
// Units of the first n tiles of a row's queries: the sum over i < n of ceil((base + (i + 1) tq) / keys), both powers of two, less what a window leaves out.  A base
// below none counts as none there; only the window knows where such a row's tokens stand, so that its gap is the one that their keys are read by.
// ONE: with a short way for rows of one tile, which takes 1 to 2 % off steps of single tokens; the f32 kernel of chunks goes without it (its registers: 22.3 us for 21.8, three rows
// of up to 130 tokens).
template <bool WIN = true, bool ONE = true> __host__ __device__ __forceinline__ long long paged_units(const PagedPlan &a, int base, long long n) {
    if (a.whole) return n;
    if (ONE && n <= 1) return n == 1 ? paged_keys<WIN>(a, base, 0) : 0;   // single tokens
    const int s = a.key_shift - a.tq_shift;
    const long long ahead = max(base, 0);
    if (s <= 0) return n * ((ahead + (1 << a.key_shift) - 1) >> a.key_shift) + ((n * (n + 1) / 2) << -s) - paged_gaps<WIN>(a, base, n);
    // ceil((b + i + 1) / 2^s) with b = ceil(base / tq): floors of c + i over 2^s, summed up to c + n and without those up to c
    const long long c = ((ahead + (1 << a.tq_shift) - 1) >> a.tq_shift) + (1ll << s);
    return paged_floors(c + n, s) - paged_floors(c, s) - paged_gaps<WIN>(a, base, n);
}
template <bool WIN = true, bool ONE = true> __host__ __device__ __forceinline__ PagedShape paged_shape(const PagedPlan &a, const PagedRow &r) {
    PagedShape s = {0, 0, 0, 0};
    const long long rows = (long long)r.count * a.group;
    if (rows <= a.above || rows > a.most) return s;
    s.q_tiles = (int)(((long long)r.count + (1 << a.tq_shift) - 1) >> a.tq_shift);
    s.base = r.len - r.count;
    s.per = paged_units<WIN, ONE>(a, s.base, s.q_tiles);
    s.units = s.per * a.p.kv_heads;
    return s;
}
// Sums over a CTA of THREADS threads: returns the thread's exclusive prefix of v, `total` gets the sum.  Every thread calls it.
// A warp by itself (THREADS 32) needs no shared memory and no other warp.
template <int THREADS> __device__ __forceinline__ long long cta_prefix(long long v, long long &total, long long *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (THREADS == 32) {
        total = __shfl_sync(0xffffffffu, x, 31);
        return x - v;
    }
    __syncthreads();  // the last call's sums have been read
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    return before + x - v;
}
struct PagedRun {
    long long u, u1;       // units left to the CTA, the first and the one behind them
    long long total;       // units of the launch
    int ctas;              // that have any
    int row, head, q_tile, k, k_tiles;   // where the run stands: the next unit, and the units of its item
    PagedRow r;            // that row
    int q_tiles, base;
};
// a / b of numbers that are not negative: in 32 bits, a fifth of the time, where they fit.
__host__ __device__ __forceinline__ long long paged_div(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// Where the run of CTA c begins.
__host__ __device__ __forceinline__ long long paged_begin(const PagedRun &run, int c) { return paged_div(run.total * min(c, run.ctas), run.ctas); }
// Unit `in` of a row: its head, the tile of queries it is of, and which of that tile's.
struct PagedUnit {
    int head, q_tile, k;
};
template <bool WIN = true, bool ONE = true> __host__ __device__ __forceinline__ PagedUnit paged_find(const PagedPlan &a, const PagedShape &s, long long in) {
    const int head = (int)paged_div(in, s.per);
    const long long y = in - head * s.per;
    int lo = 0, hi = s.q_tiles - 1;   // the tile that unit y of the head is of
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (paged_units<WIN, ONE>(a, s.base, mid) <= y) lo = mid;
        else hi = mid - 1;
    }
    return {head, lo, (int)(y - paged_units<WIN, ONE>(a, s.base, lo))};
}
// Puts the run at that unit.
template <bool WIN = true> __host__ __device__ __forceinline__ void paged_at(const PagedPlan &a, PagedRun &run, int row, const PagedUnit &u) {
    run.row = row; run.head = u.head; run.q_tile = u.q_tile; run.k = u.k;
    run.r = paged_row(a.p, row, nullptr);
    const PagedShape s = paged_shape<WIN>(a, run.r);
    run.q_tiles = s.q_tiles;
    run.base = s.base;
    run.k_tiles = paged_keys<WIN>(a, run.base, run.q_tile);
}
__host__ __device__ __forceinline__ int paged_ctas(const PagedPlan &a, long long total, int ctas) {   // that have any of `total` units
    const long long n = paged_div(total, a.least);
    return n < 1 ? 1 : n < ctas ? (int)n : ctas;
}
// The run of CTA (or, with THREADS 32, warp) `c` of `ctas`, found by all its threads.  `found` is shared.
template <int THREADS, bool WIN = true, bool ONE = true> __device__ __forceinline__ PagedRun paged_run(const PagedPlan &a, int c, int ctas, long long *warp_sums, int2 *found, int *status) {
    PagedRun run = {};
    long long n, prefix = 0, units = 0, row_first = 0;
    for (int r0 = 0; r0 < a.p.rows; r0 += THREADS) {
        const int r = r0 + (int)(threadIdx.x % THREADS);
        const long long here = r < a.p.rows ? paged_shape<WIN, ONE>(a, paged_row(a.p, r, c == 0 ? status : nullptr)).units : 0;
        const long long at = cta_prefix<THREADS>(here, n, warp_sums);
        if (r0 == 0) { prefix = at; units = here; }
        run.total += n;
    }
    run.ctas = paged_ctas(a, run.total, ctas);
    run.u = paged_begin(run, c);
    run.u1 = paged_begin(run, c + 1);
    if (run.u >= run.u1) return run;
    // the row whose units the run's first is among; found by one thread
    for (int r0 = 0;; r0 += THREADS) {
        if (r0 > 0) {
            const int r = r0 + (int)(threadIdx.x % THREADS);
            units = r < a.p.rows ? paged_shape<WIN, ONE>(a, paged_row(a.p, r, nullptr)).units : 0;
            prefix = row_first + cta_prefix<THREADS>(units, n, warp_sums);
        } else if (a.p.rows > THREADS) {
            (void)cta_prefix<THREADS>(units, n, warp_sums);
        } else {
            n = run.total;
        }
        if (units > 0 && run.u >= prefix && run.u < prefix + units) {
            const int row = r0 + (int)(threadIdx.x % THREADS);
            const PagedUnit u = paged_find<WIN, ONE>(a, paged_shape<WIN, ONE>(a, paged_row(a.p, row, nullptr)), run.u - prefix);
            found[0] = make_int2(row, u.head);
            found[1] = make_int2(u.q_tile, u.k);
        }
        if (run.u < row_first + n) break;
        row_first += n;
    }
    if (THREADS == 32) __syncwarp();
    else __syncthreads();
    paged_at<WIN>(a, run, found[0].x, {found[0].y, found[1].x, found[1].y});
    return run;
}
// A piece of work: units [k0, k1) of the item (row, head, q_tile), which has k_tiles of them.
struct PagedPiece {
    int row, head, q_tile, k0, k1, k_tiles;
    PagedRow r;
};
// The next piece of the run; false at its end.  The same for all threads that call it with the same run.
template <bool WIN = true> __host__ __device__ __forceinline__ bool paged_next(const PagedPlan &a, PagedRun &run, PagedPiece &w) {
    if (run.u >= run.u1) return false;
    if (run.k == run.k_tiles) {   // the next item: of the head, of the row, of the next row that has any
        run.k = 0;
        if (++run.q_tile == run.q_tiles) {
            run.q_tile = 0;
            if (++run.head == a.p.kv_heads) {
                run.head = 0;
                do {
                    if (++run.row >= a.p.rows) return false;
                    run.r = paged_row(a.p, run.row, nullptr);
                    const PagedShape s = paged_shape<WIN>(a, run.r);
                    run.q_tiles = s.q_tiles;
                    run.base = s.base;
                } while (run.q_tiles == 0);
            }
        }
        run.k_tiles = paged_keys<WIN>(a, run.base, run.q_tile);
    }
    w.row = run.row; w.head = run.head; w.q_tile = run.q_tile; w.r = run.r; w.k_tiles = run.k_tiles;
    w.k0 = run.k;
    w.k1 = (int)min((long long)w.k_tiles, w.k0 + (run.u1 - run.u));
    run.k = w.k1;
    run.u += w.k1 - w.k0;
    return true;
}
// What a piece covers: its tokens [t0, t0 + ntok) of the row's new ones, and the (virtual) keys [lo, hi) of it that any of them sees, or may see: hidden ones lie
// at the ends of the units of the sinks and of the window.
struct PagedSpan {
    int t0, ntok, base, lo, hi;
};
// What a window leaves out of a tile of queries: `gap` keys ahead of virtual key `jump`.
struct PagedHole {
    int gap, jump;
};
template <bool WIN = true> __host__ __device__ __forceinline__ PagedHole paged_hole(const PagedPlan &a, int base, int q_tile) {
    PagedHole h;
    h.gap = paged_gap<WIN>(a, base, q_tile) << a.key_shift;
    h.jump = h.gap ? (int)(paged_sink_units(a) << a.key_shift) : 0;
    return h;
}
template <bool WIN = true> __host__ __device__ __forceinline__ PagedSpan paged_span(const PagedPlan &a, const PagedPiece &w) {
    PagedSpan s;
    s.t0 = w.q_tile << a.tq_shift;
    s.ntok = min(1 << a.tq_shift, w.r.count - s.t0);
    s.base = w.r.len - w.r.count;
    const int last = s.base + s.t0 + s.ntok - paged_hole<WIN>(a, s.base, w.q_tile).gap;   // behind the last key that a token of the item sees
    s.lo = a.whole ? 0 : (int)min((long long)w.k0 << a.key_shift, 0x7fffffffll);
    s.hi = a.whole ? last : (int)min((long long)last, (long long)w.k1 << a.key_shift);
    return s;
}
__host__ __device__ __forceinline__ int paged_key(const PagedHole &h, int key) { return key >= h.jump ? key + h.gap : key; }
// Whether no token of the item sees any of the n keys from `key` (of the row) on: their page may be gone.
__host__ __device__ __forceinline__ bool paged_hidden(const PagedPlan &a, const PagedSpan &s, int key, int n) {
    return a.window && key >= a.sinks && key + n <= s.base + s.t0 - a.window + 1;
}

// `ctas` counts runs: CTAs, or warps where each has a run of its own.
struct PagedAttnArgs {
    PagedPlan plan;
    const void *q, *k, *v;
    void *out;
    long long q_stride, o_stride;
    float sl;          // scale in powers of two
    float *acc, *ml;   // pieces: [2 ctas][rows of a tile][dim] sums, [2 ctas][rows of a tile][2] maximum and sum of weights
    int4 *cut;         // [ctas] the item that a run began and did not end: its first token, its tokens (0: there is none), its head, the run that ends it
    int ctas, tile_rows;
    int *status;
    const float *k_scales, *v_scales;   // of e4m3 pages: one for PAGED_BLOCK tokens of a head
};
// Bytes that the pieces of a launch take.
static inline size_t paged_piece_bytes(int ctas, int tile_rows, int hd) { return (size_t)2 * ctas * tile_rows * (hd + 2) * 4 + (size_t)ctas * 16; }
static inline int paged_log2(int n) { return 31 - __builtin_clz(n); }
// Sets how a launch of `ctas` CTAs, tiles of `tile_rows` query rows and 2^key_shift keys deals its work out, cutting items where the workspace has room.
static inline void paged_deal(PagedAttnArgs &a, int ctas, int tile_rows, int key_shift, int least, int hd, void *workspace, size_t bytes) {
    a.ctas = ctas; a.tile_rows = tile_rows;
    a.plan.tq_shift = paged_log2(tile_rows / a.plan.group);
    a.plan.key_shift = key_shift;
    a.plan.per_group = (65536 + a.plan.group - 1) / a.plan.group;
    a.plan.whole = !workspace || bytes < paged_piece_bytes(ctas, tile_rows, hd);
    a.plan.least = a.plan.whole ? 1 : least;
    a.acc = (float *)workspace;
    a.ml = a.acc + (size_t)2 * ctas * tile_rows * hd;
    a.cut = (int4 *)(a.ml + (size_t)4 * ctas * tile_rows);
}
// What run c leaves to the merge, written by one thread: nothing, to begin with, and its last piece if that begins an item and does not end it.
__device__ __forceinline__ void paged_uncut(const PagedAttnArgs &a, int c) { if (!a.plan.whole) a.cut[c] = make_int4(0, 0, 0, 0); }
__host__ __device__ __forceinline__ void paged_cut(const PagedAttnArgs &a, const PagedRun &run, const PagedPiece &w, const PagedSpan &sp, int c) {
    if (w.k0 > 0 || w.k1 == w.k_tiles) return;
    const long long end = run.u + (w.k_tiles - w.k1);   // the unit behind the item: the last run that begins before it ends it
    a.cut[c] = make_int4(w.r.first + sp.t0, sp.ntok, w.head, (int)min((long long)run.ctas - 1, paged_div(end * run.ctas - 1, run.total)));
}

// Row r of a piece (queries of bf16, pages of P: bf16, or e4m3 codes) over the keys of it that it sees, by one warp: where a product with hidden values has left Inf or
// NaN (a weight of 0 times either), this gives what the keys in sight alone give.  32 keys at a time: a lane has one for the scores, and every 32nd dimension for the
// sums, so that loads of 32 keys are in flight where one key after the other waited for its page, its shuffles and its exponential.
template <int HD, typename P, bool WIN>
__device__ __forceinline__ void paged_again(const PagedAttnArgs &a, const PagedPiece &w, const PagedSpan &sp, int r, int lane, bool all, size_t slot) {
    constexpr int N = HD / 32;
    constexpr bool CODES = sizeof(P) == 1;
    using Chunk = PagedChunk<P>;
    const int tok = paged_token(a.plan, r), head = w.head * a.plan.group + r - tok * a.plan.group;
    const PagedHole hole = paged_hole<WIN>(a.plan, sp.base, w.q_tile);
    const int pos = sp.base + sp.t0 + tok, to = min(sp.hi - 1, pos - hole.gap);
    const __nv_bfloat16 *q = (const __nv_bfloat16 *)a.q + (size_t)(w.r.first + sp.t0 + tok) * a.q_stride + (size_t)head * HD;
    float acc[N] = {}, top = -INFINITY, sum = 0.f;
    for (int key0 = sp.lo; key0 <= to; key0 += 32) {
        const int key = paged_key(hole, key0 + lane), n = min(32, to - key0 + 1);
        long long row = -1;   // of a key out of sight
        float s = -INFINITY, vs = 1.f;
        if (lane < n && (!WIN || key < a.plan.sinks || key > pos - a.plan.window)) {
            row = (((long long)paged_page(a.plan.p, w.row, key, a.status) * a.plan.p.kv_heads + w.head) << a.plan.p.page_shift) + (key & ((1 << a.plan.p.page_shift) - 1));
            const P *k = (const P *)a.k + row * HD;
            s = 0.f;
#pragma unroll 4
            for (int d = 0; d < HD; d += Chunk::N) {
                float x[Chunk::N], y[Chunk::N];
                Chunk::floats(*reinterpret_cast<const uint4 *>(k + d), y);
#pragma unroll
                for (int i = 0; i < Chunk::N; i += 8) PagedChunk<__nv_bfloat16>::floats(*reinterpret_cast<const uint4 *>(q + d + i), *reinterpret_cast<float (*)[8]>(x + i));
#pragma unroll
                for (int i = 0; i < Chunk::N; ++i) s = fmaf(x[i], y[i], s);
            }
            s *= a.sl;
            if (CODES) {
                s *= a.k_scales[row / PAGED_BLOCK];
                vs = a.v_scales[row / PAGED_BLOCK];
            }
        }
        float best = fmaxf(top, s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        const float m = best == -INFINITY ? 0.f : best, keep = exp2f(top - m), e = row >= 0 ? exp2f(s - m) : 0.f;
        float here = e;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) here += __shfl_xor_sync(0xffffffffu, here, o);
        sum = sum * keep + here;
        top = best;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] *= keep;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const float f = __shfl_sync(0xffffffffu, CODES ? e * vs : e, j);
            const long long from = __shfl_sync(0xffffffffu, row, j);
            if (from < 0) continue;
            const P *v = (const P *)a.v + from * HD + lane;
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] = fmaf(f, Chunk::one(v[32 * i]), acc[i]);
        }
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (all) ((__nv_bfloat16 *)a.out)[(size_t)(w.r.first + sp.t0 + tok) * a.o_stride + (size_t)head * HD + lane + 32 * i] = __float2bfloat16_rn(acc[i] * f);
        else a.acc[(slot + r) * HD + lane + 32 * i] = acc[i];
    }
    if (!all && lane == 0) *reinterpret_cast<float2 *>(a.ml + (slot + r) * 2) = make_float2(top, sum);
}

// Finishes the items that the launch before it cut.
int paged_merge(const PagedAttnArgs &a, int hd, ab2_dtype dtype, cudaStream_t s);

}  // namespace ab2
