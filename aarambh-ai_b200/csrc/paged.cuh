// Paged caches as kernels receive them, and the turning of a pair by a position (internal header).
#pragma once

#include "common.cuh"

namespace ab2 {

int device_status_word(int **out);
int device_sm_count();

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
__device__ __forceinline__ void paged_bad(int *status) { atomicCAS(status, 0, (int)AB2_ERR_BAD_ARG); }
__device__ __forceinline__ PagedRow paged_row(const PagedView &p, int b, int *status) {
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
// keeps 29 bits as a float.
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
// An item is a tile of a row's queries (tq of its new tokens, all heads of one KV head's group) against that row's keys; a unit is `1 << key_shift`
// of an item's keys.  Every CTA of a launch takes an equal run of the units of all rows, whose lengths only the device knows (so a recorded
// launch serves other lengths when it runs again).  An item that one CTA has to itself is finished there; the pieces of one that is cut meet in
// the merge kernel.  A piece that does not begin its item is its CTA's first: slot 2 c; one that begins it and does not end it is its last: slot 2 c + 1.
// Without room for pieces items are not cut.  Keys that no query of an item sees are counted in, but skipped.
struct PagedPlan {
    PagedView p;
    int tq, key_shift, whole;
};
struct PagedShape {
    int q_tiles, k_tiles;       // of the row
    long long units;
};
__device__ __forceinline__ PagedShape paged_shape(const PagedPlan &a, const PagedRow &r) {
    PagedShape s;
    s.q_tiles = (r.count + a.tq - 1) / a.tq;
    s.k_tiles = a.whole ? 1 : max(1, (int)(((long long)r.len + (1 << a.key_shift) - 1) >> a.key_shift));
    s.units = (long long)s.q_tiles * s.k_tiles * a.p.kv_heads;
    return s;
}
// Sums over a CTA of THREADS threads: returns the thread's exclusive prefix of v, `total` gets the sum.  Every thread calls it.
template <int THREADS> __device__ __forceinline__ long long cta_prefix(long long v, long long &total, long long *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
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
    long long u, u1;       // units left to the CTA
    int row;               // that u lies in
    long long row_first;   // the row's first unit
};
// The run of CTA `c` of `ctas`, found by the whole CTA.  `found` is shared.
template <int THREADS> __device__ __forceinline__ PagedRun paged_run(const PagedPlan &a, int c, int ctas, long long *warp_sums, PagedRun *found, int *status) {
    long long total = 0, n, first_prefix = 0, first_units = 0;
    for (int r0 = 0; r0 < a.p.rows; r0 += THREADS) {
        const int r = r0 + threadIdx.x;
        const long long units = r < a.p.rows ? paged_shape(a, paged_row(a.p, r, c == 0 ? status : nullptr)).units : 0;
        const long long at = cta_prefix<THREADS>(units, n, warp_sums);
        if (r0 == 0) { first_prefix = at; first_units = units; }
        total += n;
    }
    const long long u = total * c / ctas, u1 = total * (c + 1) / ctas;
    if (threadIdx.x == 0) *found = {u, u, 0, 0};  // nothing to do
    long long before = 0;
    for (int r0 = 0; r0 < a.p.rows && before <= u; r0 += THREADS) {
        const int r = r0 + threadIdx.x;
        long long units = first_units, at = first_prefix;
        if (r0 > 0) {
            units = r < a.p.rows ? paged_shape(a, paged_row(a.p, r, nullptr)).units : 0;
            at = cta_prefix<THREADS>(units, n, warp_sums);
        } else {
            __syncthreads();
            n = THREADS < a.p.rows ? 0 : total;
            if (THREADS < a.p.rows) (void)cta_prefix<THREADS>(units, n, warp_sums);
        }
        at += before;
        if (u < u1 && units > 0 && u >= at && u < at + units) *found = {u, u1, r, at};
        before += n;
    }
    __syncthreads();
    return *found;
}
// A piece of work: tiles [k0, k1) of the item (row, head, q_tile), which has k_tiles of them.
struct PagedPiece {
    int row, head, q_tile, k0, k1, k_tiles;
    PagedRow r;
};
// The next piece of the run; false at its end.  The same for all threads that call it with the same run.
__device__ __forceinline__ bool paged_next(const PagedPlan &a, PagedRun &run, PagedPiece &w) {
    if (run.u >= run.u1) return false;
    PagedShape s;
    for (;;) {
        w.r = paged_row(a.p, run.row, nullptr);
        s = paged_shape(a, w.r);
        if (run.u < run.row_first + s.units) break;
        run.row_first += s.units;
        if (++run.row >= a.p.rows) return false;
    }
    const long long in = run.u - run.row_first;
    const int item = (int)(in / s.k_tiles);
    w.row = run.row;
    w.k_tiles = s.k_tiles;
    w.k0 = (int)(in - (long long)item * s.k_tiles);
    w.k1 = (int)min((long long)s.k_tiles, w.k0 + (run.u1 - run.u));
    w.head = item / s.q_tiles;
    w.q_tile = item - w.head * s.q_tiles;
    run.u += w.k1 - w.k0;
    return true;
}

}  // namespace ab2
