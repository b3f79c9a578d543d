// How paged attention through a window deals its work out, run on the host: the functions are those of csrc/paged.cuh that the kernels call.
#include "paged.cuh"

using namespace ab2;

// Pieces of every run: run, row, head, first new token of the row, tokens, first virtual key, the one behind the last, gap, jump, k0, k1, k_tiles.  Returns how many.
extern "C" __attribute__((visibility("default"))) int plan(const int *lens, const int *starts, int rows, int tokens, int width, int page_shift, int kv_heads, int group, int ctas, int tile_rows,
                                                           int key_shift, int least, int cutting, int window, int sinks, int *pieces, int room, int *status) {
    PagedAttnArgs a = {};
    a.plan.p.lens = lens; a.plan.p.starts = starts; a.plan.p.rows = rows; a.plan.p.tokens = tokens; a.plan.p.width = width;
    a.plan.p.page_shift = page_shift; a.plan.p.kv_heads = kv_heads; a.plan.p.pages = 1;
    a.plan.group = group; a.plan.most = 0x7fffffff;
    a.plan.window = window; a.plan.sinks = sinks;
    static char workspace[16];
    paged_deal(a, ctas, tile_rows, key_shift, least, 64, cutting ? workspace : nullptr, cutting ? paged_piece_bytes(ctas, tile_rows, 64) : 0);
    long long total = 0;
    for (int r = 0; r < rows; ++r) total += paged_shape(a.plan, paged_row(a.plan.p, r, status)).units;
    int n = 0;
    for (int c = 0; c < ctas; ++c) {
        PagedRun run = {};
        run.total = total;
        run.ctas = paged_ctas(a.plan, total, ctas);
        run.u = paged_begin(run, c);
        run.u1 = paged_begin(run, c + 1);
        if (run.u >= run.u1) continue;
        int row = 0;
        for (long long before = 0;; ++row) {
            const PagedShape s = paged_shape(a.plan, paged_row(a.plan.p, row, nullptr));
            if (run.u < before + s.units) {
                paged_at(a.plan, run, row, paged_find(a.plan, s, run.u - before));
                break;
            }
            before += s.units;
        }
        PagedPiece w;
        while (paged_next(a.plan, run, w)) {
            const PagedSpan sp = paged_span(a.plan, w);
            const PagedHole h = paged_hole(a.plan, sp.base, w.q_tile);
            if (n == room) return -1;
            const int one[12] = {c, w.row, w.head, sp.t0, sp.ntok, sp.lo, sp.hi, h.gap, h.jump, w.k0, w.k1, w.k_tiles};
            for (int i = 0; i < 12; ++i) pieces[12 * n + i] = one[i];
            ++n;
        }
    }
    return n;
}

extern "C" __attribute__((visibility("default"))) int hidden(int base, int t0, int window, int sinks, int key, int n) {
    PagedPlan p = {};
    p.window = window; p.sinks = sinks;
    PagedSpan s = {};
    s.base = base; s.t0 = t0;
    return paged_hidden(p, s, key, n);
}

extern "C" __attribute__((visibility("default"))) long long units(int base, long long n, int tile_shift, int key_shift, int window, int sinks, long long *by_tile) {
    PagedPlan p = {};
    p.tq_shift = tile_shift; p.key_shift = key_shift; p.window = window; p.sinks = sinks;
    *by_tile = 0;
    for (int i = 0; i < n; ++i) *by_tile += paged_keys(p, base, i);
    return paged_units(p, base, n);
}
