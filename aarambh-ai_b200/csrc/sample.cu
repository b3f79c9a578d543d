// A token of every row of logits, drawn with a given number u in [0, 1):
//
//   p_v = 2^(-x_v),  x_v = (max z - z_v) log2(e) / temperature;  tokens in order of falling z, of equal ones the lower index first
//   top-k: the first k stay;  top-p: of these the shortest prefix whose mass is p of theirs or more;  min-p: of these the ones with p_v >= min_p
//   the token: the first one that stayed, in order of index, whose cumulative mass exceeds u times all of theirs
//
// Weights are whole numbers, round(2^F p_v) with F up to 44, from f64: their sums are exact whatever the order, so that every run and every way of dealing the
// row out draws the same token, and a border between two tokens lies within 2^-45 a token of where real numbers have it (f32 sums would move it by more than a
// token's width in large vocabularies).
//
// A cluster of CTAs has a row, each a slice of it, which it keeps in shared memory.  Nothing is sorted: tokens are counted by x in bins of 1/32; the bin in which
// the k-th token lies, or a bracket of bins around the border of top-p, follows from the counts (a bin's weights differ by 2^(1/32) at most), and the few tokens
// up to there go to the first CTA's list, which finds both borders by halving keys, exactly.  Where a list does not hold them (a nucleus of thousands of tokens,
// thousands of equal logits), or all tokens stay, the CTAs work on their slices instead, and join their sums.
#include <algorithm>
#include <cooperative_groups.h>

#include "common.cuh"

using namespace ab2;
namespace cg = cooperative_groups;

namespace ab2 {
int device_sm_count();
namespace {

typedef unsigned long long u64;
constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_BINS = 2048, SP_PER = 32, SP_LIST = 4096, SP_MINE = SP_LIST / SP_THREADS, SP_CTAS = 8;

struct SampleArgs {
    const void *logits, *uniforms;
    long long stride;
    int uniforms_64, vocab, slice, shift;   // tokens of a CTA; F
    const float *temperature, *top_p, *min_p;
    const int *top_k;
    int *out;
};

struct alignas(16) SampleShared {
    int counts[SP_BINS];          // of the slice; read by the cluster's others
    int cum[SP_BINS];             // of the row, cumulative
    float least[SP_BINS], most[SP_BINS];   // bounds of the cumulative mass
    float list_z[SP_LIST];
    int list_i[SP_LIST];
    u64 red[2][SP_WARPS], slot[2], part[SP_WARPS];
    float scan[3][SP_WARPS];
    int top_bits, listed, found[4];
    uint32_t cut_key;
    int cut_index;
};

__device__ __forceinline__ uint32_t key_of(float z) {   // larger for larger logits; 0 for those that are never drawn (NaN and -inf)
    if (!(z > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(z + 0.f);   // -0 is 0
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) { return key == 0u ? -INFINITY : __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

template <typename T, bool CACHED>
__global__ void __launch_bounds__(SP_THREADS) sample_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared &sh = *(SampleShared *)smem;
    T *cache = (T *)(smem + sizeof(SampleShared));
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int first = rank * a.slice, n = max(0, min(a.slice, a.vocab - first));
    const T *in = (const T *)a.logits + row * a.stride + first;
    const float temperature = a.temperature ? a.temperature[row] : 1.f;
    const bool warm = temperature > 0.f;   // else the likeliest token
    const double c = warm ? 1.4426950408889634 / (double)temperature : INFINITY;
    float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
    int k = a.top_k ? a.top_k[row] : 0;
    if (!warm || min_p > 1.f) k = 1;
    min_p = fminf(min_p, 1.f);   // NaN: 1, the likeliest and what is as likely

    // ---- the slice, and the row's largest logit
    for (int b = tid; b < SP_BINS; b += SP_THREADS) sh.counts[b] = 0;
    if (tid == 0) sh.listed = 0;
    float top = -INFINITY;
    constexpr int V = 16 / sizeof(T);
    if (((uintptr_t)in & 15) == 0) {
        for (int i = tid * V; i < n; i += SP_THREADS * V) {
            alignas(16) T e[V];
            if (i + V <= n) {
                *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(in + i);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) e[j] = i + j < n ? in[i + j] : from_f32<T>(-INFINITY);
            }
            if (CACHED) *reinterpret_cast<uint4 *>(cache + i) = *reinterpret_cast<const uint4 *>(e);   // the slice is a multiple of V
#pragma unroll
            for (int j = 0; j < V; ++j) top = fmaxf(top, to_f32(e[j]));
        }
    } else {
        for (int i = tid; i < n; i += SP_THREADS) {
            if (CACHED) cache[i] = in[i];
            top = fmaxf(top, to_f32(in[i]));
        }
    }
    auto logit = [&](int i) { return to_f32(CACHED ? cache[i] : in[i]); };
    int phase = 0;
    auto block_sum = [&](u64 v) {   // of all threads, for all threads
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) sh.red[phase][warp] = v;
        __syncthreads();
        u64 s = 0;
#pragma unroll
        for (int w = 0; w < SP_WARPS; ++w) s += sh.red[phase][w];
        phase ^= 1;   // the next sum goes elsewhere: some may still read this one
        return s;
    };
    int cphase = 0;
    auto cluster_sum = [&](u64 v) {   // of all threads of the cluster, for all
        const u64 mine = block_sum(v);
        if (C == 1) return mine;
        if (tid == 0) sh.slot[cphase] = mine;
        cluster.sync();
        u64 s = 0;
        for (int r = 0; r < C; ++r) s += *cluster.map_shared_rank(&sh.slot[cphase], r);
        cphase ^= 1;
        return s;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) sh.scan[0][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SP_WARPS; ++w) top = fmaxf(top, sh.scan[0][w]);
    if (C > 1) {
        if (tid == 0) sh.top_bits = __float_as_int(top);
        cluster.sync();
        for (int r = 0; r < C; ++r) top = fmaxf(top, __int_as_float(*cluster.map_shared_rank(&sh.top_bits, r)));
    }
    if (!(top > -INFINITY)) {   // no token can be drawn
        if (rank == 0 && tid == 0) a.out[row] = -1;
        if (C > 1) cluster.sync();   // the others may still read this CTA's maximum
        return;
    }
    const double F = (double)a.shift, full = (double)(1ull << a.shift);
    auto weight = [&](float z) -> u64 {
        if (z == top) return 1ull << a.shift;
        const double x = ((double)top - (double)z) * c;
        return x < F + 2.0 ? __double2ull_rn(exp2(F - x)) : 0ull;   // NaN and -inf: 0
    };
    const float cf = (float)c * SP_PER;
    auto bin_of = [&](float z) { return z == top ? 0 : (int)fminf((top - z) * cf, (float)(SP_BINS - 1)); };   // rises where z falls
    const double wmin = (double)min_p * full;
    auto likely = [&](u64 w) { return !(min_p > 0.f) || (double)w >= wmin; };

    // ---- counts by bins; all of the mass, where top-k does not cut it
    u64 all = 0;
    for (int i = tid; i < n; i += SP_THREADS) {
        const float z = logit(i);
        if (!(z > -INFINITY)) continue;
        atomicAdd(&sh.counts[bin_of(z)], 1);
        if (k <= 0 && (top_p < 1.f)) all += weight(z);
    }
    all = cluster_sum(all);   // and the counts are whole
    {
        constexpr int B = SP_BINS / SP_THREADS;
        int count[B] = {}, sum = 0;
        float lo = 0.f, hi = 0.f, los[B], his[B];
        for (int r = 0; r < C; ++r) {
            const int4 v = *reinterpret_cast<const int4 *>(cluster.map_shared_rank(sh.counts, r) + tid * B);
            count[0] += v.x; count[1] += v.y; count[2] += v.z; count[3] += v.w;
        }
        static_assert(B == 4, "bins of a thread");
#pragma unroll
        for (int j = 0; j < B; ++j) {   // in units of the likeliest token's
            const float edge = exp2f(-(float)(tid * B + j) / SP_PER);
            count[j] = sum += count[j];
            const int here = count[j] - (j ? count[j - 1] : 0);
            hi += (float)here * edge;
            lo += tid * B + j == SP_BINS - 1 ? 0.f : (float)here * edge * 0.97857206f;   // 2^(-1 / SP_PER)
            his[j] = hi;
            los[j] = lo;
        }
        int s = sum;
        float l = lo, h = hi;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int ps = __shfl_up_sync(0xffffffffu, s, o);
            const float pl = __shfl_up_sync(0xffffffffu, l, o), ph = __shfl_up_sync(0xffffffffu, h, o);
            if (lane >= o) { s += ps; l += pl; h += ph; }
        }
        __syncthreads();
        if (lane == 31) { sh.scan[0][warp] = __int_as_float(s); sh.scan[1][warp] = l; sh.scan[2][warp] = h; }
        if (tid < 4) sh.found[tid] = SP_BINS - 1;
        __syncthreads();
        s -= sum; l -= lo; h -= hi;
        for (int w = 0; w < warp; ++w) { s += __float_as_int(sh.scan[0][w]); l += sh.scan[1][w]; h += sh.scan[2][w]; }
#pragma unroll
        for (int j = 0; j < B; ++j) { sh.cum[tid * B + j] = s + count[j]; sh.least[tid * B + j] = l + los[j]; sh.most[tid * B + j] = h + his[j]; }
        __syncthreads();
    }
    const int valid = sh.cum[SP_BINS - 1];
    const bool by_k = k > 0 && k < valid, by_p = top_p < 1.f;
    // the first bin whose cumulative value is `least` or more
    auto first_bin = [&](auto cumulative, auto least, int which) {
        for (int b = tid; b < SP_BINS; b += SP_THREADS)
            if (cumulative[b] >= least && (b == 0 || !(cumulative[b - 1] >= least))) atomicMin(&sh.found[which], b);
        __syncthreads();
        return sh.found[which];
    };
    const int k_bin = by_k ? first_bin(sh.cum, k, 0) : SP_BINS - 1;
    if (by_p && k > 0 && !by_k) {   // more than there are: its mass has not been summed
        u64 s = 0;
        for (int i = tid; i < n; i += SP_THREADS) s += weight(logit(i));
        all = cluster_sum(s);
    }
    const double share = (double)fmaxf(top_p, 0.f);
    const float target0 = (float)(share * ((double)all / full));
    int last = k_bin;   // the last bin that the list needs; top-p takes its share of all that top-k left, those that min-p drops among them
    if (!by_k && by_p) last = first_bin(sh.least, target0 * 1.001f, 1);
    if (min_p > 0.f && !(by_k && by_p)) last = min(last, (int)fminf(fmaxf(-log2f(min_p), 0.f) * SP_PER + 1.f, (float)(SP_BINS - 1)));
    const bool filters = by_k || by_p || min_p > 0.f;

    // The largest key t such that the sum over tokens with keys of t or more reaches `target`, 0 if none does.  sum(t): that sum.
    auto find_key = [&](auto sum, u64 target, uint32_t lo, uint32_t hi) {
        if (sum(lo) < target) return 0u;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (sum(mid) >= target) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    // The lowest index such that the sum over tokens up to it reaches `target`.
    auto find_index = [&](auto sum, u64 target) {
        int lo = 0, hi = a.vocab - 1;
        while (lo < hi) {
            const int mid = lo + (hi - lo) / 2;
            if (sum(mid) >= target) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    };
    auto draw_target = [&](u64 mass) {   // the token's cumulative mass is more than this
        const double u = a.uniforms_64 ? ((const double *)a.uniforms)[row] : (double)((const float *)a.uniforms)[row];
        return u > 0.0 ? min((u64)fmin(u * (double)mass, 9.0e18), mass - 1) : 0ull;
    };
    // Of n things of equal weight w behind a mass of `before`, how many it takes to reach `target`: one at least.
    auto enough = [&](u64 target, u64 before, u64 w, u64 n) { return w == 0 || target <= before ? 1ull : min(n, (target - before + w - 1) / w); };
    auto whole = [&](double x) { return (u64)ceil(fmin(x, 9.0e18)); };   // a mass reaches x where it reaches this

    // Tokens of bins [b0, b1] to the first CTA's list; false, and no list, where it does not hold them.
    auto gather = [&](int b0, int b1) {
        if (sh.cum[b1] - (b0 > 0 ? sh.cum[b0 - 1] : 0) > SP_LIST) return false;
        SampleShared *there = cluster.map_shared_rank(&sh, 0);
        for (int i0 = 0; i0 < n; i0 += SP_THREADS) {
            const int i = i0 + tid;
            const float z = i < n ? logit(i) : -INFINITY;
            const int b = z > -INFINITY ? bin_of(z) : -1;
            const bool in = b >= b0 && b <= b1;
            const unsigned who = __ballot_sync(0xffffffffu, in);
            if (!who) continue;
            int at = 0;
            if (lane == 0) at = atomicAdd(&there->listed, __popc(who));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
            if (in) { there->list_z[at] = z; there->list_i[at] = first + i; }
        }
        cluster.sync();
        return true;
    };
    // The list's tokens, a few a thread, of which some have been dropped.
    uint32_t keys[SP_MINE];
    u64 weights[SP_MINE];
    int index[SP_MINE];
    auto take = [&]() {
#pragma unroll
        for (int j = 0; j < SP_MINE; ++j) {
            const int at = tid + j * SP_THREADS;
            const float z = at < sh.listed ? sh.list_z[at] : -INFINITY;
            keys[j] = key_of(z);
            index[j] = at < sh.listed ? sh.list_i[at] : 0x7fffffff;
            weights[j] = weight(z);
        }
    };
    auto list_sum = [&](auto value) {
        u64 s = 0;
#pragma unroll
        for (int j = 0; j < SP_MINE; ++j) s += value(keys[j], index[j], weights[j]);
        return block_sum(s);
    };
    auto slice_sum = [&](auto value) {   // of (key, index, logit)
        u64 s = 0;
        for (int i = tid; i < n; i += SP_THREADS) {
            const float z = logit(i);
            const uint32_t key = key_of(z);
            if (key) s += value(key, first + i, z);
        }
        return cluster_sum(s);
    };
    const uint32_t top_key = key_of(top);
    // Border of the first `count` (or, by mass, of the shortest prefix that reaches it): the last token that stays, as key and index.  total(f): the sum over all
    // tokens at hand of f(key, index).
    auto border = [&](auto total, u64 target, u64 each, auto value, uint32_t &key, int &idx) {   // value(key): what a token of that key counts; each: of one at the border, 0: value
        key = find_key([&](uint32_t t) { return total([&](uint32_t x, int) { return x >= t ? value(x) : 0ull; }); }, target, 1u, top_key);
        if (key == 0u) {   // all of them stay
            idx = 0x7fffffff;
            return;
        }
        const u64 before = total([&](uint32_t x, int) { return x > key ? value(x) : 0ull; }), ties = total([&](uint32_t x, int) { return x == key ? 1ull : 0ull; });
        const u64 need = enough(target, before, each ? each : value(key), ties);
        idx = need >= ties ? 0x7fffffff : find_index([&](int m) { return total([&](uint32_t x, int i) { return x == key && i <= m ? 1ull : 0ull; }); }, need);
    };
    auto stays = [&](uint32_t x, int i, uint32_t key, int idx) { return x > key || (x == key && i <= idx); };

    if (filters && sh.cum[last] <= SP_LIST) {
        // ---- all that can stay is in the list
        gather(0, last);
        if (rank != 0) return;   // nobody reads this CTA's memory any more
        take();
        auto drop = [&](uint32_t key, int idx) {
#pragma unroll
            for (int j = 0; j < SP_MINE; ++j)
                if (!stays(keys[j], index[j], key, idx)) { keys[j] = 0u; weights[j] = 0ull; }
        };
        uint32_t key;
        int idx;
        if (by_k && sh.listed > k) {
            border([&](auto f) { return list_sum([&](uint32_t x, int i, u64) { return f(x, i); }); }, (u64)k, 1ull, [&](uint32_t) { return 1ull; }, key, idx);
            drop(key, idx);
        }
        if (by_p) {
            const u64 mass = by_k ? list_sum([&](uint32_t, int, u64 w) { return w; }) : all, target = max(whole(share * (double)mass), 1ull);
            key = find_key([&](uint32_t t) { return list_sum([&](uint32_t x, int, u64 w) { return x >= t ? w : 0ull; }); }, target, 1u, top_key);
            if (key) {
                const u64 before = list_sum([&](uint32_t x, int, u64 w) { return x > key ? w : 0ull; }), ties = list_sum([&](uint32_t x, int, u64) { return x == key ? 1ull : 0ull; });
                const u64 need = enough(target, before, weight(logit_of(key)), ties);
                idx = need >= ties ? 0x7fffffff : find_index([&](int m) { return list_sum([&](uint32_t x, int i, u64) { return x == key && i <= m ? 1ull : 0ull; }); }, need);
                drop(key, idx);
            }
        }
#pragma unroll
        for (int j = 0; j < SP_MINE; ++j)
            if (!likely(weights[j])) weights[j] = 0ull;
        const u64 mass = list_sum([&](uint32_t, int, u64 w) { return w; }), target = draw_target(mass) + 1;
        const int token = find_index([&](int m) { return list_sum([&](uint32_t, int i, u64 w) { return i <= m ? w : 0ull; }); }, target);
        if (tid == 0) a.out[row] = token;
        return;
    }

    // ---- slices
    uint32_t key = 0u;   // the last token that stays
    int idx = 0x7fffffff;
    auto share_cut = [&]() {   // what the first CTA found, for all
        if (rank == 0 && tid == 0) { sh.cut_key = key; sh.cut_index = idx; sh.listed = 0; }
        cluster.sync();
        key = *cluster.map_shared_rank(&sh.cut_key, 0);
        idx = *cluster.map_shared_rank(&sh.cut_index, 0);
        cluster.sync();
    };
    if (by_k) {
        const int before = k_bin > 0 ? sh.cum[k_bin - 1] : 0;
        if (gather(k_bin, k_bin)) {
            if (rank == 0) {
                take();
                border([&](auto f) { return list_sum([&](uint32_t x, int i, u64) { return x ? f(x, i) : 0ull; }); }, (u64)(k - before), 1ull, [&](uint32_t) { return 1ull; }, key, idx);
            }
            share_cut();
        } else {
            border([&](auto f) { return slice_sum([&](uint32_t x, int i, float) { return f(x, i); }); }, (u64)k, 1ull, [&](uint32_t) { return 1ull; }, key, idx);
        }
        if (by_p) all = slice_sum([&](uint32_t x, int i, float z) { return stays(x, i, key, idx) ? weight(z) : 0ull; });
    }
    if (by_p) {
        const u64 target = max(whole(share * (double)all), 1ull);
        const float near = (float)((double)target / full);
        const int b0 = first_bin(sh.most, near * 0.999f, 2), b1 = min(max(first_bin(sh.least, near * 1.001f, 3), b0), k_bin);
        const uint32_t k_key = key;
        const int k_idx = idx;
        uint32_t p_key = 0u;
        int p_idx = 0x7fffffff;
        const u64 ahead = slice_sum([&](uint32_t, int, float z) { return bin_of(z) < b0 ? weight(z) : 0ull; });
        if (ahead < target && b0 <= b1 && gather(b0, b1)) {
            if (rank == 0) {
                take();
                border([&](auto f) { return list_sum([&](uint32_t x, int i, u64) { return x && stays(x, i, k_key, k_idx) ? f(x, i) : 0ull; }); }, target - ahead, 0ull, [&](uint32_t x) { return weight(logit_of(x)); }, key, idx);
            }
            share_cut();
            p_key = key; p_idx = idx;
        } else {
            border([&](auto f) { return slice_sum([&](uint32_t x, int i, float) { return stays(x, i, k_key, k_idx) ? f(x, i) : 0ull; }); }, target, 0ull, [&](uint32_t x) { return weight(logit_of(x)); }, p_key, p_idx);
        }
        // where all of what top-k left stays, of one key all that it left
        key = max(p_key, k_key);
        idx = p_key < k_key ? k_idx : p_key == k_key ? min(p_idx, k_idx) : p_idx;
    }
    // every warp's run of the slice, the CTAs', and the token
    const int run = ((n + SP_WARPS - 1) / SP_WARPS + 31) / 32 * 32, i0 = warp * run, i1 = min(n, i0 + run);
    auto kept = [&](int i) -> u64 {
        const float z = logit(i);
        const uint32_t x = key_of(z);
        if (!x || !stays(x, first + i, key, idx)) return 0ull;
        const u64 w = weight(z);
        return likely(w) ? w : 0ull;
    };
    u64 mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) mine += kept(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sh.part[warp] = mine;
    const u64 slice = block_sum(lane == 0 ? mine : 0ull);
    if (tid == 0) sh.slot[cphase] = slice;
    cluster.sync();
    u64 before = 0, mass = 0;
    for (int r = 0; r < C; ++r) {
        const u64 s = *cluster.map_shared_rank(&sh.slot[cphase], r);
        if (r < rank) before += s;
        mass += s;
    }
    const u64 target = draw_target(mass) + 1;
    if (before < target && target <= before + slice) {
        for (int w = 0; w < warp; ++w) before += sh.part[w];
        if (before < target && target <= before + mine) {   // in this warp's run
            for (int i = i0; i < i1; i += 32) {
                u64 up = i + lane < i1 ? kept(i + lane) : 0ull;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 v = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += v;
                }
                const unsigned there = __ballot_sync(0xffffffffu, before + up >= target);
                if (there) {
                    if (lane == 0) a.out[row] = first + i + __ffs(there) - 1;
                    break;
                }
                before += __shfl_sync(0xffffffffu, up, 31);
            }
        }
    }
    cluster.sync();   // the others may still read this CTA's sum
}

template <typename T, bool CACHED>
int launch_sample(const SampleArgs &a, int rows, int ctas, size_t smem, cudaStream_t s) {
    static size_t configured[64] = {0};  // the attribute is per device
    int dev = 0;
    AB2_CUDA(cudaGetDevice(&dev));
    AB2_REQUIRE(dev >= 0 && dev < 64, AB2_ERR_BAD_ARG, "device index %d out of range", dev);
    if (configured[dev] == 0) {
        AB2_CUDA(cudaFuncSetAttribute(sample_kernel<T, CACHED>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        configured[dev] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ctas)); cfg.blockDim = dim3(SP_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    AB2_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T, CACHED>, a));
    return AB2_OK;
}
template <typename T>
int launch_sample(SampleArgs a, int rows, cudaStream_t s) {
    // The most CTAs a row that are still resident at once, of 1024 tokens or more; more where a slice would not fit shared memory.
    constexpr size_t ROOM = 227 * 1024 - sizeof(SampleShared);
    auto slice = [&](int ctas) { return ((a.vocab + ctas - 1) / ctas + 31) / 32 * 32; };
    int ctas = 1;
    while (ctas < SP_CTAS && ((2 * ctas * rows <= device_sm_count() && a.vocab >= 2048 * ctas) || slice(ctas) * sizeof(T) > ROOM)) ctas *= 2;
    a.slice = slice(ctas);
    const size_t bytes = a.slice * sizeof(T);
    return bytes <= ROOM ? launch_sample<T, true>(a, rows, ctas, sizeof(SampleShared) + bytes, s) : launch_sample<T, false>(a, rows, ctas, sizeof(SampleShared), s);
}

}  // namespace
}  // namespace ab2

AB2_API int ab2_sample(const void *logits_dev, long long stride, int rows, int vocab, const void *uniforms_dev, int uniforms_64, const float *temperature_dev, const int *top_k_dev,
                       const float *top_p_dev, const float *min_p_dev, int *out_dev, ab2_dtype dtype, ab2_stream stream) {
    AB2_REQUIRE(rows >= 0 && vocab > 0, AB2_ERR_BAD_SHAPE, "logits of %d rows, %d tokens", rows, vocab);
    AB2_REQUIRE(vocab <= (1 << 24) && (long long)rows * SP_CTAS < (1ll << 31), AB2_ERR_UNSUPPORTED, "%d rows of %d tokens: up to 2^24 tokens and 2^28 rows are served", rows, vocab);
    AB2_REQUIRE(dtype == AB2_F32 || dtype == AB2_F16 || dtype == AB2_BF16, AB2_ERR_BAD_DTYPE, "unsupported dtype %d", (int)dtype);
    if (rows == 0) return AB2_OK;
    AB2_REQUIRE(logits_dev && uniforms_dev && out_dev, AB2_ERR_BAD_ARG, "null argument");
    AB2_REQUIRE(stride >= vocab, AB2_ERR_BAD_SHAPE, "rows of %d logits lie %lld apart", vocab, stride);
    AB2_REQUIRE((uintptr_t)logits_dev % dtype_size(dtype) == 0 && (uintptr_t)uniforms_dev % (uniforms_64 ? 8 : 4) == 0 && (((uintptr_t)temperature_dev | (uintptr_t)top_k_dev | (uintptr_t)top_p_dev | (uintptr_t)min_p_dev | (uintptr_t)out_dev) & 3) == 0,
                AB2_ERR_BAD_ALIGN, "logits, numbers and tokens must lie on their elements");
    const long long es = (long long)dtype_size(dtype);
    const RowsAt o = {out_dev, 4ll * rows, 4ll * rows, 1};
    AB2_REQUIRE(!rows_meet(o, {logits_dev, vocab * es, stride * es, rows}), AB2_ERR_BAD_ARG, "the tokens may not take the logits' place");
    for (const void *p : {(const void *)uniforms_dev, (const void *)temperature_dev, (const void *)top_k_dev, (const void *)top_p_dev, (const void *)min_p_dev}) {
        const long long bytes = (p == uniforms_dev && uniforms_64 ? 8ll : 4ll) * rows;
        AB2_REQUIRE(!rows_meet(o, {p, bytes, bytes, 1}), AB2_ERR_BAD_ARG, "the tokens may not take the place of what they are drawn by");
    }
    SampleArgs a = {};
    a.logits = logits_dev; a.stride = stride; a.vocab = vocab; a.uniforms = uniforms_dev; a.uniforms_64 = uniforms_64;
    a.temperature = temperature_dev; a.top_k = top_k_dev; a.top_p = top_p_dev; a.min_p = min_p_dev; a.out = out_dev;
    a.shift = 44;
    while (((long long)vocab << a.shift) > (1ll << 61)) --a.shift;
    switch (dtype) {
    case AB2_F32: return launch_sample<float>(a, rows, (cudaStream_t)stream);
    case AB2_F16: return launch_sample<__half>(a, rows, (cudaStream_t)stream);
    default: return launch_sample<__nv_bfloat16>(a, rows, (cudaStream_t)stream);
    }
}
