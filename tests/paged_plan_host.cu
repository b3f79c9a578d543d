// How paged attention deals its work out, run on the host: the functions are those of csrc/paged.cuh that the kernels call.
#include "paged.cuh"

using namespace ab2;

static PagedAttnArgs args(const int *lens, const int *starts, int rows, int tokens, int width, int page_shift, int kv_heads, int group, int above, int most, int ctas, int tile_rows, int key_shift, int least,
                          int cutting, int *cut) {
    PagedAttnArgs a = {};
    a.plan.p.lens = lens; a.plan.p.starts = starts; a.plan.p.rows = rows; a.plan.p.tokens = tokens; a.plan.p.width = width;
    a.plan.p.page_shift = page_shift; a.plan.p.kv_heads = kv_heads; a.plan.p.pages = 1;
    a.plan.group = group; a.plan.above = above; a.plan.most = most;
    static char workspace[16];   // only its being there and its size are looked at
    paged_deal(a, ctas, tile_rows, key_shift, least, 64, cutting ? workspace : nullptr, cutting ? paged_piece_bytes(ctas, tile_rows, 64) : 0);
    a.cut = (int4 *)cut;
    return a;
}

// Pieces of every run: run, row, head, q_tile, k0, k1, k_tiles, first token, tokens, first key, key behind the last, slot.  cut: [ctas][4], none: zeros.  Returns how many.
extern "C" __attribute__((visibility("default"))) int plan(const int *lens, const int *starts, int rows, int tokens, int width, int page_shift, int kv_heads, int group, int above, int most, int ctas,
                                                           int tile_rows, int key_shift, int least, int cutting, int *cut, int *pieces, int room, int *status) {
    const PagedAttnArgs a = args(lens, starts, rows, tokens, width, page_shift, kv_heads, group, above, most, ctas, tile_rows, key_shift, least, cutting, cut);
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
            if (cutting) paged_cut(a, run, w, sp, c);
            if (n == room) return -1;
            const int one[12] = {c, w.row, w.head, w.q_tile, w.k0, w.k1, w.k_tiles, w.r.first + sp.t0, sp.ntok, sp.lo, sp.hi, 2 * c + (w.k0 == 0)};
            for (int i = 0; i < 12; ++i) pieces[12 * n + i] = one[i];
            ++n;
        }
    }
    return n;
}

extern "C" __attribute__((visibility("default"))) long long units(int base, long long n, int tile_shift, int key_shift, int whole) {
    PagedPlan p = {};
    p.tq_shift = tile_shift; p.key_shift = key_shift; p.whole = whole;
    return paged_units(p, base, n);
}

extern "C" __attribute__((visibility("default"))) int token(int group, int row) {
    PagedPlan p = {};
    p.per_group = (65536 + group - 1) / group;
    return paged_token(p, row);
}
