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
constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_BINS = 2048, SP_PER = 32, SP_LIST = 4096, SP_MINE = SP_LIST / SP_THREADS, SP_CTAS = 8, SP_TABLE = 256;

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
    union {
        struct {
            float least[SP_BINS], most[SP_BINS];      // bounds of the cumulative mass
        };
        struct {
            uint32_t low[SP_BINS], high[SP_BINS];     // exact masses of the slice's bins, in two words; read by the cluster's others
        };
    };
    u64 list[SP_LIST];            // tokens: key and, below it, what is larger for lower indices
    u64 weights[SP_LIST];
    double powers[SP_TABLE];      // 2^(-j / SP_TABLE)
    u64 red[2][SP_WARPS], slot[2], part[SP_WARPS];
    float scan[3][SP_WARPS];
    int top_bits, listed, found[4];
    u64 cut;
};

__device__ __forceinline__ uint32_t key_of(float z) {   // larger for larger logits; 0 for those that are never drawn (NaN and -inf)
    if (!(z > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(z + 0.f);   // -0 is 0
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) { return key == 0u ? -INFINITY : __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }
// A token among others: larger ones come first.
__device__ __forceinline__ u64 token_of(uint32_t key, int index) { return (u64)key << 32 | (0xffffffffu - (uint32_t)index); }
__device__ __forceinline__ int index_of(u64 token) { return (int)(0xffffffffu - (uint32_t)token); }

// Sorts list[0, n) by falling values; what lies behind n, up to the next power of two or SP_THREADS, becomes 0.  Bitonic: a thread an element, exchanged by shuffles
// where the partner is in the warp; longer lists in shared memory throughout.
__device__ __forceinline__ void sort_list(u64 *list, int n) {
    const int tid = threadIdx.x;
    if (n <= SP_THREADS) {
        u64 v = tid < n ? list[tid] : 0ull;
        for (int k = 2; k <= SP_THREADS; k <<= 1) {
            const bool falls = (tid & k) == 0;
            for (int j = k >> 1; j > 0; j >>= 1) {
                u64 o;
                if (j >= 32) {
                    __syncthreads();
                    list[tid] = v;
                    __syncthreads();
                    o = list[tid ^ j];
                } else {
                    o = __shfl_xor_sync(0xffffffffu, v, j);
                }
                const bool larger = ((tid & j) == 0) == falls;   // of the two this thread keeps the larger one
                v = (o > v) == larger ? o : v;
            }
        }
        __syncthreads();
        list[tid] = v;
        __syncthreads();
        return;
    }
    int all = SP_THREADS;
    while (all < n) all <<= 1;
    for (int i = n + tid; i < all; i += SP_THREADS) list[i] = 0ull;
    for (int k = 2; k <= all; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int t = tid; t < all / 2; t += SP_THREADS) {
                const int i = 2 * t - (t & (j - 1));
                const u64 x = list[i], y = list[i + j];
                if ((x < y) == ((i & k) == 0)) { list[i] = y; list[i + j] = x; }
            }
        }
    __syncthreads();
}

template <typename T, bool CACHED>
__global__ void __launch_bounds__(SP_THREADS, 1) sample_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared &sh = *(SampleShared *)smem;
    T *cache = (T *)(smem + sizeof(SampleShared));
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int first = rank * a.slice, n = max(0, min(a.slice, a.vocab - first));
    const T *in = (const T *)a.logits + row * a.stride + first;

    // ---- the slice, and the row's largest logit
    float top = -INFINITY;
    constexpr int V = 16 / sizeof(T);
    const bool wide = ((uintptr_t)in & 15) == 0;
    if (wide) {
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
        if (CACHED)   // whole pieces of V are read
            for (int i = n + tid; i < (n + V - 1) / V * V; i += SP_THREADS) cache[i] = from_f32<T>(-INFINITY);
    }
    for (int b = tid; b < SP_BINS; b += SP_THREADS) sh.counts[b] = 0;
    for (int j = tid; j < SP_TABLE; j += SP_THREADS) sh.powers[j] = exp2(-(double)j / SP_TABLE);
    if (tid == 0) sh.listed = 0;
    const float temperature = a.temperature ? a.temperature[row] : 1.f;
    const bool warm = temperature > 0.f;   // else the likeliest token
    const double c = warm ? 1.4426950408889634 / (double)temperature : INFINITY;
    const float top_p = a.top_p ? a.top_p[row] : 1.f;
    float min_p = a.min_p ? a.min_p[row] : 0.f;
    int k = a.top_k ? a.top_k[row] : 0;
    if (!warm || min_p > 1.f) k = 1;
    min_p = fminf(min_p, 1.f);   // NaN: 1, the likeliest and what is as likely
    const bool by_p = top_p < 1.f;

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
    auto block_before = [&](u64 v) {   // of the threads ahead
        u64 up = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 x = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += x;
        }
        if (lane == 31) sh.red[phase][warp] = up;
        __syncthreads();
        up -= v;
        for (int w = 0; w < warp; ++w) up += sh.red[phase][w];
        phase ^= 1;
        return up;
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
    const float cf = (float)c;
    const double c_table = c * SP_TABLE, full = (double)(1ull << a.shift), top_d = (double)top;
    const float far = (float)(a.shift + 2);
    // 2^F 2^-x as a whole number: x in units of 1 / SP_TABLE is a whole number k and a rest of a half at most, 2^-x the table's entry times a cubic polynomial of the rest
    // (2^-42 of it off).  Adding 2^52 to a double rounds it to a whole number, which its low bits then are.
    auto weight = [&](float z) -> u64 {
        if (z == top) return 1ull << a.shift;
        if (!((top - z) * cf < far)) return 0ull;   // NaN and -inf too
        const uint32_t b = __float_as_uint(z);      // as f64: exact but for 0 and subnormals, which come out below 2^-126
        const double d = __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
        const double t = (top_d - d) * c_table, whole = t + 6755399441055744.0;   // 1.5 2^52
        const int k = __double2loint(whole);
        const double r = t - (whole - 6755399441055744.0), u = r * -(0.6931471805599453 / SP_TABLE);
        const double p = sh.powers[k & (SP_TABLE - 1)] * fma(u, fma(u, fma(u, 1.0 / 6, 0.5), 1.0), 1.0);
        const double w = __hiloint2double(__double2hiint(p) + ((a.shift - (k >> 8)) << 20), __double2loint(p)) + 4503599627370496.0;   // 2^52
        return (u64)__double_as_longlong(w) & 0xfffffffffffffull;
    };
    static_assert(SP_TABLE == 256, "k >> 8");
    const float c_bin = cf * SP_PER;
    auto bin_of = [&](float z) { return z == top ? 0 : (int)fminf((top - z) * c_bin, (float)(SP_BINS - 1)); };   // rises where z falls
    const double wmin = (double)min_p * full;
    auto likely = [&](u64 w) { return !(min_p > 0.f) || (double)w >= wmin; };
    // f(logit, index in the slice) of all tokens of the slice that can be drawn; those of a thread are V neighbours at a time
    auto for_slice = [&](auto f) {
        if (CACHED || wide) {
            for (int i = tid * V; i < n; i += SP_THREADS * V) {
                alignas(16) T e[V];
                if (CACHED) *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(cache + i);
                else if (i + V <= n) *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(in + i);
                else
                    for (int j = 0; j < V; ++j) e[j] = i + j < n ? in[i + j] : from_f32<T>(-INFINITY);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float z = to_f32(e[j]);
                    if (z > -INFINITY) f(z, i + j);
                }
            }
        } else {
            for (int i = tid; i < n; i += SP_THREADS) {
                const float z = to_f32(in[i]);
                if (z > -INFINITY) f(z, i);
            }
        }
    };

    // ---- counts by bins; all of the mass, where top-k does not cut it
    u64 all = 0;
    if (k <= 0 && by_p) for_slice([&](float z, int) { atomicAdd(&sh.counts[bin_of(z)], 1); all += weight(z); });
    else for_slice([&](float z, int) { atomicAdd(&sh.counts[bin_of(z)], 1); });
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
    const bool by_k = k > 0 && k < valid;
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
        for_slice([&](float z, int) { s += weight(z); });
        all = cluster_sum(s);
    }
    const double share = (double)fmaxf(top_p, 0.f);
    int last = k_bin;   // the last bin that the list needs; top-p takes its share of all that top-k left, those that min-p drops among them
    if (!by_k && by_p) last = first_bin(sh.least, (float)(share * ((double)all / full)) * 1.001f, 1);
    if (min_p > 0.f && !(by_k && by_p)) last = min(last, (int)fminf(fmaxf(-log2f(min_p), 0.f) * SP_PER + 1.f, (float)(SP_BINS - 1)));
    const bool filters = by_k || by_p || min_p > 0.f;

    auto draw_target = [&](u64 mass) {   // the token's cumulative mass reaches this
        const double u = a.uniforms_64 ? ((const double *)a.uniforms)[row] : (double)((const float *)a.uniforms)[row];
        return (u > 0.0 ? min((u64)fmin(u * (double)mass, 9.0e18), mass - 1) : 0ull) + 1;
    };
    auto whole = [&](double x) { return max((u64)ceil(fmin(x, 9.0e18)), 1ull); };   // a mass reaches x where it reaches this

    // Tokens of bins [b0, b1] to the first CTA's list; false, and no list, where it does not hold them.
    auto gather = [&](int b0, int b1) {
        if (sh.cum[b1] - (b0 > 0 ? sh.cum[b0 - 1] : 0) > SP_LIST) return false;
        SampleShared *there = cluster.map_shared_rank(&sh, 0);
        for_slice([&](float z, int i) {
            const int b = bin_of(z);
            if (b >= b0 && b <= b1) there->list[atomicAdd(&there->listed, 1)] = token_of(key_of(z), first + i);
        });
        cluster.sync();
        return true;
    };
    // A thread's tokens of the sorted list, neighbours, and their weights (0: of those behind `count`, or below `least`); the mass ahead of the first.
    u64 mine[SP_MINE], w[SP_MINE], ahead = 0;
    int per = 1;   // tokens of a thread
    auto weigh = [&](int count, u64 least) {
        per = 1;
        while (per * SP_THREADS < sh.listed) per <<= 1;
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < SP_MINE; ++j) {
            w[j] = mine[j] = 0ull;
            if (j >= per) continue;
            const int at = tid * per + j;
            mine[j] = sh.list[at];
            if (at < count && mine[j] >= least) w[j] = weight(logit_of((uint32_t)(mine[j] >> 32)));
            sum += w[j];
        }
        ahead = block_before(sum);
        return sum;
    };

    if (filters && sh.cum[last] <= SP_LIST) {
        // ---- all that can stay is in the list
        gather(0, last);
        if (rank != 0) return;   // nobody reads this CTA's memory any more
        const int listed = sh.listed;
        sort_list(sh.list, listed);
        const u64 sum = weigh(by_k ? min(k, listed) : listed, 1ull);
        if (by_p) {
            const u64 target = whole(share * (double)(by_k ? block_sum(sum) : all));
            u64 at = ahead;
#pragma unroll
            for (int j = 0; j < SP_MINE; ++j) {
                const u64 next = at + w[j];
                if (at >= target) w[j] = 0ull;
                at = next;
            }
        }
        u64 stay = 0;
        int some = 0;   // behind the last of the thread's that stay
#pragma unroll
        for (int j = 0; j < SP_MINE; ++j) {
            if (!likely(w[j])) w[j] = 0ull;
            stay += w[j];
            if (w[j]) some = tid * per + j + 1;
        }
        // what stays is a prefix: it is sorted again, by index
        const u64 target = draw_target(block_sum(stay));
        const int kept = __reduce_max_sync(0xffffffffu, some);
        if (lane == 0) sh.scan[0][warp] = __int_as_float(kept);
        __syncthreads();   // and every thread has its tokens
        int m = 0;
#pragma unroll
        for (int i = 0; i < SP_WARPS; ++i) m = max(m, __float_as_int(sh.scan[0][i]));
#pragma unroll
        for (int j = 0; j < SP_MINE; ++j) {
            const int at = tid * per + j;
            if (j >= per || at >= m) continue;
            sh.weights[at] = w[j];
            sh.list[at] = (mine[j] & 0xffffffffull) << 32 | (uint32_t)at;
        }
        __syncthreads();
        sort_list(sh.list, m);
        const int run = (m + SP_THREADS - 1) / SP_THREADS;
        u64 here = 0;
        for (int j = 0; j < run; ++j)
            if (tid * run + j < m) here += sh.weights[(uint32_t)sh.list[tid * run + j]];
        u64 at = block_before(here);
        for (int j = 0; j < run; ++j) {
            if (tid * run + j >= m) break;
            const u64 token = sh.list[tid * run + j], next = at + sh.weights[(uint32_t)token];
            if (at < target && target <= next) a.out[row] = index_of(token >> 32);
            at = next;
        }
        return;
    }

    // ---- slices
    u64 cut = 0ull;   // the last token that stays
    auto share_cut = [&]() {   // what the first CTA found, for all
        if (rank == 0 && tid == 0) { sh.cut = cut; sh.listed = 0; }
        cluster.sync();
        cut = *cluster.map_shared_rank(&sh.cut, 0);
        cluster.sync();
    };
    // Where no list holds a bin: of its tokens that stay so far, those of which the sum of value(logit) reaches `target`, by halving keys and then indices.
    auto halve = [&](int bin, u64 target, auto value) {
        auto total = [&](auto counts) {
            u64 s = 0;
            for_slice([&](float z, int i) {
                const u64 token = token_of(key_of(z), first + i);
                if (bin_of(z) == bin && token >= cut && counts(token)) s += value(z);
            });
            return cluster_sum(s);
        };
        u64 lo = max(cut, 1ull), hi = token_of(key_of(top), 0);   // the largest token at which the sum from it on reaches the target
        if (total([&](u64 t) { return t >= lo; }) < target) return cut;
        while (lo < hi) {
            const u64 mid = lo + (hi - lo) / 2 + 1;
            if (total([&](u64 t) { return t >= mid; }) >= target) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    if (by_k) {
        const int before = k_bin > 0 ? sh.cum[k_bin - 1] : 0;
        if (gather(k_bin, k_bin)) {
            if (rank == 0) {
                sort_list(sh.list, sh.listed);
                cut = sh.list[k - before - 1];
            }
            __syncthreads();   // before listed is cleared
            share_cut();
        } else {
            cut = halve(k_bin, (u64)(k - before), [](float) { return 1ull; });
        }
        if (by_p) {
            u64 s = 0;
            for_slice([&](float z, int i) { if (token_of(key_of(z), first + i) >= cut) s += weight(z); });
            all = cluster_sum(s);
        }
    }
    if (by_p) {
        u64 target = whole(share * (double)all);
        const float near = (float)((double)target / full);
        int b0 = first_bin(sh.most, near * 0.999f, 2), b1 = min(max(first_bin(sh.least, near * 1.001f, 3), b0), k_bin);
        b0 = min(b0, b1);
        __syncthreads();   // the bounds have been read; the masses of bins b0 .. b1, exactly, take their place
        for (int b = b0 + tid; b <= b1; b += SP_THREADS) sh.low[b] = sh.high[b] = 0u;
        __syncthreads();
        u64 s = 0;
        for_slice([&](float z, int i) {
            const int b = bin_of(z);
            if (b > b1 || token_of(key_of(z), first + i) < cut) return;
            const u64 w = weight(z);
            if (b < b0) {
                s += w;
            } else {
                const uint32_t w0 = (uint32_t)w, carry = atomicAdd(&sh.low[b], w0) > ~w0 ? 1u : 0u, w1 = (uint32_t)(w >> 32) + carry;
                if (w1) atomicAdd(&sh.high[b], w1);
            }
        });
        s = cluster_sum(s);
        for (int b = b0 + tid; b <= b1; b += SP_THREADS) {
            u64 here = 0;
            for (int r = 0; r < C; ++r) here += ((u64)*cluster.map_shared_rank(&sh.high[b], r) << 32) + *cluster.map_shared_rank(&sh.low[b], r);
            sh.weights[b - b0] = here;
        }
        __syncthreads();
        int bin = b1;   // of the border
        for (int b = b0; b < b1; ++b) {
            const u64 here = sh.weights[b - b0];
            if (s + here >= target) { bin = b; break; }
            s += here;
        }
        target = target > s ? target - s : 1ull;
        if (gather(bin, bin)) {
            if (rank == 0) {
                sort_list(sh.list, sh.listed);
                weigh(sh.listed, max(cut, 1ull));
                // the last token whose mass ahead is below the target
                if (tid == 0) sh.cut = ~0ull;
                __syncthreads();
                u64 at = ahead, lowest = ~0ull;
#pragma unroll
                for (int j = 0; j < SP_MINE; ++j) {
                    if (mine[j] >= max(cut, 1ull) && at < target) lowest = mine[j];
                    at += w[j];
                }
                if (lowest != ~0ull) atomicMin(&sh.cut, lowest);
                __syncthreads();
                cut = sh.cut;
            }
            __syncthreads();
            share_cut();
        } else {
            cut = halve(bin, target, weight);
        }
    }
    // every warp's run of the slice, the CTAs', and the token
    auto logit = [&](int i) { return to_f32(CACHED ? cache[i] : in[i]); };
    const int run = ((n + SP_WARPS - 1) / SP_WARPS + 31) / 32 * 32, i0 = warp * run, i1 = min(n, i0 + run);
    auto kept = [&](int i) -> u64 {
        const float z = logit(i);
        if (!(z > -INFINITY) || token_of(key_of(z), first + i) < cut) return 0ull;
        const u64 w = weight(z);
        return likely(w) ? w : 0ull;
    };
    u64 part = 0;
    for (int i = i0 + lane; i < i1; i += 32) part += kept(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) sh.part[warp] = part;
    const u64 slice = block_sum(lane == 0 ? part : 0ull);
    if (tid == 0) sh.slot[cphase] = slice;
    cluster.sync();
    u64 before = 0, mass = 0;
    for (int r = 0; r < C; ++r) {
        const u64 s = *cluster.map_shared_rank(&sh.slot[cphase], r);
        if (r < rank) before += s;
        mass += s;
    }
    const u64 target = draw_target(mass);
    if (before < target && target <= before + slice) {
        for (int w = 0; w < warp; ++w) before += sh.part[w];
        if (before < target && target <= before + part) {   // in this warp's run
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
    while (ctas < SP_CTAS && ((2 * ctas * rows <= device_sm_count() && a.vocab >= 2048 * ctas) || (size_t)slice(ctas) * sizeof(T) > ROOM)) ctas *= 2;
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
