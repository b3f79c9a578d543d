// A token of every row of logits, drawn with a given number u in [0, 1):
//
//   p_v = 2^(-x_v),  x_v = (max z - z_v) log2(e) / temperature;  tokens in order of falling z, of equal ones the lower index first
//   top-k: the first k stay;  top-p: of these the shortest prefix whose mass is p of theirs or more;  min-p: of these the ones with p_v >= min_p
//   the token: the first one that stayed, in order of index, whose cumulative mass exceeds u times all of theirs
//
// Weights are whole numbers, round(2^F p_v), off by 2^-30.4 of themselves (quick_weight) and half of one: their sums are exact whatever the order, so that every run and
// every way of dealing the row out draws the same token, and a border between two tokens lies within that and 2^-(F + 1) a token of where real numbers have it (f32 sums would
// move it by more than a token's width in large vocabularies).  F is 44 up to 2^17 tokens and one less for every doubling beyond: a row's sum stays below 2^61.
//
// A cluster of CTAs has a row, each a slice of it, which it keeps in shared memory.  Most rows are decided by a few tokens: with top-k or min-p a logit is found that all
// which can stay reach (of the threads' largest ones, sorted, the one of which k reach it), what reaches it goes to the first CTA's list, which is sorted, cut and
// sorted again by index.  Otherwise tokens are counted by x in bins of 1/64 (of bf16 by logit); the bins up to the border go to the list where it holds them, or else the
// border's bin is found by the bins' exact masses, and the token by one more pass, in which the CTAs join their sums.  Where a bin has more tokens than the list takes
// (thousands of equal logits) its border is found by halving keys.
//
// Bound by its passes over the slice: instructions, not HBM, which a row crosses once.  64 rows of 128256 bf16 logits (16.4 MB, 2.5 us at a copy's rate), us: top-k of 50 or min-p 20,
// unfiltered 31 (a weight a token, some 25 instructions), top-p of 0.9 51, of which counts of logits and the pass that weighs are two (bins of x, weighed twice and masses joined by carries: 103),
// all kinds of rules in a batch 51; 4 rows of 32000 f32: 8, 12 to 13, 29, 18.  Weights looked up in a table by their logit instead of computed: 49 for 50, and unfiltered 36 for 28 (its reads of 8
// bytes meet in banks).
#include <algorithm>
#include <type_traits>
#include <cooperative_groups.h>

#include "common.cuh"

using namespace ab2;
namespace cg = cooperative_groups;

namespace ab2 {
int device_sm_count();
namespace {

typedef unsigned long long u64;
constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_BINS = 4096, SP_PER = 64, SP_LIST = 1024, SP_MINE = SP_LIST / SP_THREADS, SP_CTAS = 8;
constexpr float SP_MAGIC = 12582912.f;   // 1.5 2^23: added to a float, its low bits are the nearest whole number's

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
    u64 red[2][SP_WARPS], slot[2], part[SP_WARPS];
    u64 sums[2];                  // of the slice: mass ahead of top-p's border, and tokens on it; read by the cluster's others
    int ties[SP_WARPS];
    float scan[3][SP_WARPS];
    uint32_t powers[256];         // 2^(j / 256), times 2^31
    float tops[2];                // the slice's largest logit, and one that so many of its tokens reach; read by the cluster's others
    int listed, found[4], index;
    uint32_t key_range[2];        // read by the cluster's others
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

// 2^F 2^-x as a whole number, x = (top - z) c: for logits, temperatures and powers of two out of the ordinary.
__device__ __noinline__ u64 weight_of(float z, float top, double c, int shift) {
    if (z == top) return 1ull << shift;
    const double x = ((double)top - (double)z) * c;
    return x < (double)shift + 2.0 ? __double2ull_rn(exp2((double)shift - x)) : 0ull;   // NaN and -inf: 0
}

// Sorts E values of each thread, value e of thread t being e SP_THREADS + t, to fall.  Bitonic: partners are exchanged by shuffles where they are in the warp.
template <int E, typename X> __device__ __forceinline__ void sort_threads(X (&v)[E], X *buffer) {
    const int tid = threadIdx.x;
    for (int k = 2; k <= E * SP_THREADS; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (E == 2 && j == SP_THREADS) {
                const X a = v[0], b = v[E - 1];
                v[0] = a > b ? a : b;
                v[E - 1] = a > b ? b : a;
                continue;
            }
            X o[E];
            if (j >= 32) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; ++e) buffer[e * SP_THREADS + tid] = v[e];
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = j >= 32 ? buffer[(e * SP_THREADS + tid) ^ j] : __shfl_xor_sync(0xffffffffu, v[e], j & 31);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool falls = ((e * SP_THREADS + tid) & k) == 0, larger = ((tid & j) == 0) == falls;   // of the two this thread keeps the larger one
                v[e] = (o[e] > v[e]) == larger ? o[e] : v[e];
            }
        }
}
// Sorts list[0, n), up to 2 SP_THREADS, to fall; what lies behind becomes 0.
__device__ __forceinline__ void sort_list(u64 *list, int n) {
    const int tid = threadIdx.x;
    if (n <= SP_THREADS) {
        u64 v[1] = {tid < n ? list[tid] : 0ull};
        sort_threads<1>(v, list);
        __syncthreads();
        list[tid] = v[0];
    } else {
        u64 v[2] = {list[tid], tid + SP_THREADS < n ? list[tid + SP_THREADS] : 0ull};
        sort_threads<2>(v, list);
        __syncthreads();
        list[tid] = v[0];
        list[tid + SP_THREADS] = v[1];
    }
    __syncthreads();
}
static_assert(SP_LIST == 2 * SP_THREADS, "what a sort takes");

template <typename T, bool CACHED>
__global__ void __launch_bounds__(SP_THREADS, 1) sample_kernel(const __grid_constant__ SampleArgs a) {
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
    const float top_p = a.top_p ? a.top_p[row] : 1.f;
    float min_p = a.min_p ? a.min_p[row] : 0.f;
    int k = a.top_k ? a.top_k[row] : 0;
    if (!warm || min_p > 1.f) k = 1;
    min_p = fminf(min_p, 1.f);   // NaN: 1, the likeliest and what is as likely
    const bool by_p = top_p < 1.f;

    // ---- the slice, and the row's largest logit
    float top = -INFINITY;
    constexpr int V = 16 / sizeof(T);
    const bool wide = ((uintptr_t)in & 15) == 0;
    if (wide) {
#pragma unroll 4
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
#pragma unroll 4
        for (int i = tid; i < n; i += SP_THREADS) {
            const T e = in[i];
            if (CACHED) cache[i] = e;
            top = fmaxf(top, to_f32(e));
        }
        if (CACHED)   // whole pieces of V are read
            for (int i = n + tid; i < (n + V - 1) / V * V; i += SP_THREADS) cache[i] = from_f32<T>(-INFINITY);
    }
    if (tid < 256) sh.powers[tid] = (uint32_t)__double2ull_rn(exp2((double)tid / 256) * 2147483648.0);
    // With top-k: of the threads' largest logits the nth, n chosen so that k of the row's tokens at least reach the smallest of those of all CTAs, and not many more.
    const int nth = k > 0 && k <= 600 ? (k + C - 1) / C : 0;
    const bool few = nth > 0 && nth <= SP_THREADS;
    float reached = -INFINITY;
    if (few) {
        float v[1] = {top}, *buffer = (float *)sh.list;
        sort_threads<1>(v, buffer);
        __syncthreads();
        buffer[tid] = v[0];
        __syncthreads();
        reached = buffer[nth - 1];
        __syncthreads();   // the list may be written from here on
    }
    if (tid == 0) sh.listed = 0;

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
        if (tid == 0) { sh.tops[0] = top; sh.tops[1] = reached; }
        cluster.sync();
        for (int r = 0; r < C; ++r) {
            const float2 v = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(sh.tops, r));
            top = fmaxf(top, v.x);
            reached = fminf(reached, v.y);
        }
    }
    if (!(top > -INFINITY)) {   // no token can be drawn
        if (rank == 0 && tid == 0) a.out[row] = -1;
        if (C > 1) cluster.sync();   // the others may still read this CTA's maximum
        return;
    }
    // A token's weight.  z log2(e) / temperature = k / 256 + r + l: k a whole number, |r| a 512th at most, l what the product's rounding left.  The weight is, in units of
    // 2^-F of a power of two just above the largest, 2^((k - k0) / 256) e^v with v = (r + l) ln 2: the power from a table, e^v - 1 = v + v^2 / 2 + v^3 / 6 as a whole
    // number of 2^-31.  Some 2^-31 of the weight off, either way, one logit's apart from another's.  (In f64 it took four times as long: this GPU's f64 is slow.)
    const float ch = (float)c, cl = (float)(c - (double)ch);
    const double top_c = (double)top * c;
    const bool quick = c > 1e-30 && c < 1e30 && top_c > -1000.0 && top_c < 1000.0;
    const int k0 = quick ? (int)ceil(top_c * 256.0) : 0, up = a.shift + 1;   // F + 1
    const float lowest = quick ? top - (float)((a.shift + 3) / c) : 0.f;   // weighs nothing
    auto quick_weight = [&](float z) -> u64 {
        z = fmaxf(z, lowest);   // NaN and -inf too
        const float zc = z * ch, l = fmaf(z, cl, fmaf(z, ch, -zc));
        const float m = fmaf(z, ch * 256.f, SP_MAGIC), r = fmaf(m - SP_MAGIC, -0.00390625f, zc);
        const int q = __float_as_int(m) - 0x4b400000 - k0;
        const float v = fmaf(l, 0.693147182f, r * 0.693147182f), e = fmaf(v * v, fmaf(v, 1.6666667e-1f, 0.5f), v) + 5.859375e-3f;   // 1.5 2^(23 - 31)
        const int d = __float_as_int(e) - 0x3bc00000;
        const uint32_t p = sh.powers[q & 255];
        const uint32_t mantissa = p + (uint32_t)((long long)d * (int)(p >> 1) >> 30);   // 2^31 2^((q mod 256) / 256) e^v, up to 2^32: e^v is at most half a step of the table
        const int n = up + (q >> 8);   // 2^(n - 32) times it, rounded
        const u64 w = (u64)mantissa << (n & 31);
        return n >= 32 ? w : n < 0 ? 0ull : (w + 0x80000000ull) >> 32;
    };
    auto slow_weight = [&](float z) { return weight_of(z, top, c, a.shift); };
    auto weight = [&](float z) { return quick ? quick_weight(z) : slow_weight(z); };
    // f(weight) for a pass: decided once, so that the products of a thread's tokens run side by side
    auto by_weight = [&](auto f) {
        if (quick) f(quick_weight);
        else f(slow_weight);
    };
    const float c_bin = fminf(ch, 1e30f) * SP_PER;
    const bool infinite = top == INFINITY;
    auto bin_of = [&](float z) {   // rises where z falls
        if (infinite) return z == top ? 0 : SP_BINS - 1;
        return __float_as_int(fminf(fmaf(top - z, c_bin, SP_MAGIC), SP_MAGIC + (SP_BINS - 1))) - 0x4b400000;
    };
    const double full = (double)weight(top);
    const u64 wmin = min_p > 0.f ? (u64)ceil((double)min_p * full) : 0ull;
    auto likely = [&](u64 w) { return w >= wmin; };
    auto load = [&](int i, T (&e)[V]) {   // V tokens from i on, a multiple of V; -inf behind the slice
        if (CACHED) {
            *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(cache + i);
        } else if (wide && i + V <= n) {
            *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(in + i);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] = i + j < n ? in[i + j] : from_f32<T>(-INFINITY);
        }
    };
    // The row's counts of the thread's bins, behind a barrier of all.  With 4 CTAs or 8 each adds up its share of the bins first:
    // all bins read by all CTAs took 35 us for 27.5 (top-p alone, 4 rows of 32000 f32).
    auto counts_of_row = [&](int (&count)[SP_BINS / SP_THREADS]) {
        constexpr int B = SP_BINS / SP_THREADS;
        static_assert(B == 8 && SP_CTAS == 8 && SP_BINS / 4 == 2 * SP_THREADS, "bins of a thread");
        auto add = [&](int r) {
            const int4 *from = reinterpret_cast<const int4 *>(cluster.map_shared_rank(sh.counts, r) + tid * B), v = from[0], w = from[1];
            count[0] += v.x; count[1] += v.y; count[2] += v.z; count[3] += v.w;
            count[4] += w.x; count[5] += w.y; count[6] += w.z; count[7] += w.w;
        };
        if (C >= 4) {
            const int share = SP_BINS / C, mine = rank * share + tid;
            int sum[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (i * SP_THREADS < share)
#pragma unroll 4
                    for (int r = 0; r < C; ++r) sum[i] += cluster.map_shared_rank(sh.counts, r)[mine + i * SP_THREADS];
            cluster.sync();   // all have read their shares of the slices' counts: the row's take their place
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (i * SP_THREADS < share) sh.counts[mine + i * SP_THREADS] = sum[i];
            cluster.sync();
            add(tid * B / share);
        } else {
            for (int r = 0; r < C; ++r) add(r);
        }
    };
    // f(logit, index in the slice) of all tokens of the slice that can be drawn
    auto for_slice = [&](auto f) {
        for (int i = tid * V; i < n; i += SP_THREADS * V) {
            alignas(16) T e[V];
            load(i, e);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float z = to_f32(e[j]);
                if (z > -INFINITY) f(z, i + j);
            }
        }
    };
    // f of all of them, whether they can be drawn or not
    auto for_all = [&](auto f) {
        for (int i = tid * V; i < n; i += SP_THREADS * V) {
            alignas(16) T e[V];
            load(i, e);
#pragma unroll
            for (int j = 0; j < V; ++j) f(to_f32(e[j]), i + j);
        }
    };
    // found(index): of the token whose cumulative value(logit, index in the slice), in order of index, reaches target(the sum of all), called by one thread of the cluster.
    // Every warp sums a run of the slice; the one that the target falls into looks again.
    auto locate = [&](auto value, auto target_of, auto found) {
        const int run = ((n + SP_WARPS - 1) / SP_WARPS + 32 * V - 1) / (32 * V) * (32 * V), i0 = warp * run, i1 = min(n, i0 + run);
        u64 part = 0;
        for (int i = i0 + lane * V; i < i1; i += 32 * V) {
            alignas(16) T e[V];
            load(i, e);
#pragma unroll
            for (int j = 0; j < V; ++j) part += value(to_f32(e[j]), i + j);
        }
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
        cphase ^= 1;
        const u64 target = target_of(mass);
        if (before < target && target <= before + slice) {
            for (int w = 0; w < warp; ++w) before += sh.part[w];
            if (before < target && target <= before + part) {   // in this warp's run
                for (int i = i0; i < i1; i += 32 * V) {
                    alignas(16) T e[V];
                    u64 here = 0;
                    const int at = i + lane * V;
                    if (at < i1) load(at, e);
                    else
                        for (int j = 0; j < V; ++j) e[j] = from_f32<T>(-INFINITY);
#pragma unroll
                    for (int j = 0; j < V; ++j) here += value(to_f32(e[j]), at + j);
                    u64 up = here;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const u64 v = __shfl_up_sync(0xffffffffu, up, o);
                        if (lane >= o) up += v;
                    }
                    const unsigned there = __ballot_sync(0xffffffffu, before + up >= target);
                    if (there) {
                        if (lane == __ffs(there) - 1) {
                            u64 sum = before + up - here;
                            for (int j = 0; j < V; ++j) {
                                sum += value(to_f32(e[j]), at + j);
                                if (sum >= target) {
                                    found(first + at + j);
                                    break;
                                }
                            }
                        }
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, up, 31);
                }
            }
        }
        cluster.sync();   // the others may still read this CTA's sum
    };
    const double share = (double)fmaxf(top_p, 0.f);
    auto draw_target = [&](u64 mass) {   // the token's cumulative mass reaches this
        const double u = a.uniforms_64 ? ((const double *)a.uniforms)[row] : (double)((const float *)a.uniforms)[row];
        return (u > 0.0 ? min((u64)fmin(u * (double)mass, 9.0e18), mass - 1) : 0ull) + 1;
    };
    auto whole = [&](double x) { return max((u64)ceil(fmin(x, 9.0e18)), 1ull); };   // a mass reaches x where it reaches this

    // Tokens of which wanted(logit) to the first CTA's list, as many as it holds.
    auto gather = [&](auto wanted) {
        SampleShared *there = cluster.map_shared_rank(&sh, 0);
        for_slice([&](float z, int i) {
            if (!wanted(z)) return;
            const int at = atomicAdd(&there->listed, 1);
            if (at < SP_LIST) there->list[at] = token_of(key_of(z), first + i);
        });
        cluster.sync();
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
    // The token, where all that can stay is in the list: by the first CTA.  most: of top-k; mass: of all tokens, where top-p takes its share of that.
    auto from_list = [&](int most, bool cut_by_k, u64 mass) {
        sort_list(sh.list, sh.listed);
        const u64 sum = weigh(min(most, sh.listed), 1ull);
        if (by_p) {
            const u64 target = whole(share * (double)(cut_by_k ? block_sum(sum) : mass));
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
    };

    // ---- a logit that all which can stay reach: by top-k, or by min-p (whose share top-p does not take)
    if (few || (min_p > 0.f && !by_p)) {
        float from = reached;
        if (min_p > 0.f && !by_p) from = fmaxf(from, infinite ? top : (float)((double)top - (-log2((double)min_p) * 1.001 + 0.01) / c));
        gather([&](float z) { return z >= from; });
        if (*cluster.map_shared_rank(&sh.listed, 0) <= SP_LIST) {
            if (rank != 0) return;   // nobody reads this CTA's memory any more
            from_list(k > 0 ? k : SP_LIST, k > 0, 0ull);
            if (C > 1) cluster.sync();   // the others have read the list's length: those that have left count as arrived
            return;
        }
        cluster.sync();
        if (tid == 0) sh.listed = 0;   // of the first CTA; behind another barrier of all it is written again
    }

    // ---- bf16, top-p without top-k: a row has few logits that differ, so that counts of them and a weight for each give top-p's border exactly, ties and all, and one pass
    // over the weights gives the token.  A slot is a logit, in falling order, from the largest down to the last that weighs anything; those near zero, whose binades go
    // on down to 2^-126, share one (the band), are weighed token by token, and leave a border among them to what follows.
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const int kt = (int)(key_of(top) >> 16), kl = (int)(key_of(lowest) >> 16);   // the upper half of a key: all of a bf16's
        int bits = max(128, (kt - kl + 1 - SP_BINS + 255) / 256 * 128), positive, negative, slots;   // the band is of those below the power of two with these bits
        if (top < 0.f) {   // no band: its slot and the border's are never the same
            positive = 0x10000;
            negative = 0xfffe;
            slots = kt - kl + 1;
        } else for (;; bits += 128) {
            positive = 0x8000 + bits;       // the least key above the band
            negative = 0x7fff - bits;       // the largest below it
            slots = kt - kl + 1;
            if (kl <= negative) slots -= positive - negative - 2;
            else if (kl < positive) slots = kt - positive + 2;
            if (slots <= SP_BINS || positive > kt) break;
        }
        if (quick && k <= 0 && by_p && slots <= SP_BINS && (positive <= kt || top < 0.f)) {
            const int shut = positive - negative - 2;   // keys that the band closes up
            const int band = kt - positive + 1;         // its slot
            auto slot_of = [&](T z) -> int {            // less than 0, or `slots` and more: of those that weigh nothing (NaN, -inf)
                const int r = (int)__bfloat16_as_ushort(z), key = r ^ (r & 0x8000 ? 0xffff : 0x8000), d = kt - key;
                return key >= positive ? d : key > negative ? band : d - shut;
            };
            auto logit_at = [&](int slot) {             // not of the band
                const int key = kt - (slot < band ? slot : slot + shut);
                return __uint_as_float((uint32_t)(key ^ (key & 0x8000 ? 0x8000 : 0xffff)) << 16);
            };
            constexpr int B = SP_BINS / SP_THREADS;
            for (int b = tid; b < SP_BINS; b += SP_THREADS) sh.counts[b] = 0;
            __syncthreads();
            u64 in_band = 0;
            for (int i = tid * V; i < n; i += SP_THREADS * V) {
                alignas(16) T e[V];
                load(i, e);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int s = slot_of(e[j]);
                    if ((unsigned)s >= (unsigned)slots) continue;
                    if (s == band) in_band += quick_weight(to_f32(e[j]));
                    else atomicAdd(&sh.counts[s], 1);
                }
            }
            in_band = cluster_sum(in_band);
            if (C == 1) __syncthreads();
            int count[B] = {};
            counts_of_row(count);
            u64 weights[B], sum = 0;
#pragma unroll
            for (int j = 0; j < B; ++j) {
                const int s = tid * B + j;
                weights[j] = s < slots && s != band ? quick_weight(logit_at(s)) : 0ull;
                sum += s == band ? in_band : weights[j] * (u64)count[j];
            }
            const u64 target = whole(share * (double)block_sum(sum));
            u64 at = block_before(sum);
            if (at < target && target <= at + sum) {
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const u64 here = tid * B + j == band ? in_band : weights[j] * (u64)count[j];
                    if (at < target && target <= at + here) {
                        sh.found[0] = tid * B + j;
                        sh.cut = weights[j] ? (target - at + weights[j] - 1) / weights[j] : 0ull;
                    }
                    at += here;
                }
            }
            __syncthreads();
            const int border = sh.found[0];   // the slot in which top-p ends
            const u64 need = sh.cut;          // tokens of it that stay
            if (border != band) {
                const float edge = logit_at(border);
                const u64 weighed = quick_weight(edge), each = likely(weighed) ? weighed : 0ull;
                // of a token: its mass where it is ahead of the border, and whether it is on it
                auto add = [&](T e, u64 &mass, int &ties) {
                    const float z = to_f32(e);
                    const u64 w = quick_weight(z);
                    if (z > edge && likely(w)) mass += w;
                    ties += z == edge;
                };
                auto kept = [&](u64 mass, u64 ties) { return mass + each * min(ties, need); };   // of equal logits the first ones stay
                const int run = ((n + SP_WARPS - 1) / SP_WARPS + 32 * V - 1) / (32 * V) * (32 * V), i0 = warp * run, i1 = min(n, i0 + run);
                u64 mass = 0;
                int ties = 0;
                for (int i = i0 + lane * V; i < i1; i += 32 * V) {
                    alignas(16) T e[V];
                    load(i, e);
#pragma unroll
                    for (int j = 0; j < V; ++j) add(e[j], mass, ties);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
                ties = __reduce_add_sync(0xffffffffu, ties);
                if (lane == 0) { sh.part[warp] = mass; sh.ties[warp] = ties; }
                const u64 slice_mass = block_sum(lane == 0 ? mass : 0ull), slice_ties = block_sum(lane == 0 ? (u64)ties : 0ull);
                if (tid == 0) { sh.sums[0] = slice_mass; sh.sums[1] = slice_ties; }
                cluster.sync();
                u64 m = 0, t = 0, all_mass = 0, all_ties = 0;
                for (int r = 0; r < C; ++r) {
                    const ulonglong2 s = *reinterpret_cast<const ulonglong2 *>(cluster.map_shared_rank(sh.sums, r));
                    if (r < rank) { m += s.x; t += s.y; }
                    all_mass += s.x;
                    all_ties += s.y;
                }
                const u64 target = draw_target(kept(all_mass, all_ties));
                if (kept(m, t) < target && target <= kept(m + slice_mass, t + slice_ties)) {
                    for (int w = 0; w < warp; ++w) { m += sh.part[w]; t += sh.ties[w]; }
                    if (kept(m, t) < target && target <= kept(m + mass, t + ties)) {   // in this warp's run
                        for (int i = i0; i < i1; i += 32 * V) {
                            alignas(16) T e[V];
                            u64 up = 0;
                            int level = 0;
                            const int at = i + lane * V;
                            if (at < i1) load(at, e);
                            else
                                for (int j = 0; j < V; ++j) e[j] = from_f32<T>(-INFINITY);
#pragma unroll
                            for (int j = 0; j < V; ++j) add(e[j], up, level);
                            const u64 here = up;
                            const int tied = level;
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1) {
                                const u64 v = __shfl_up_sync(0xffffffffu, up, o);
                                const int l = __shfl_up_sync(0xffffffffu, level, o);
                                if (lane >= o) { up += v; level += l; }
                            }
                            const unsigned there = __ballot_sync(0xffffffffu, kept(m + up, t + level) >= target);
                            if (there) {
                                if (lane == __ffs(there) - 1) {
                                    u64 sum = m + up - here;
                                    int seen = level - tied;
                                    for (int j = 0; j < V; ++j) {
                                        add(e[j], sum, seen);
                                        if (kept(sum, t + seen) >= target) {
                                            a.out[row] = first + at + j;
                                            break;
                                        }
                                    }
                                }
                                break;
                            }
                            m += __shfl_sync(0xffffffffu, up, 31);
                            t += __shfl_sync(0xffffffffu, level, 31);
                        }
                    }
                }
                cluster.sync();   // the others may still read this CTA's sums
                return;
            }
            cluster.sync();   // the others may still read this CTA's counts
        }
    }

    u64 cut = 0ull;   // the last token that stays
    if (k > 0 || by_p || min_p > 0.f) {
        // ---- counts by bins; all of the mass, where top-k does not cut it
        for (int b = tid; b < SP_BINS; b += SP_THREADS) sh.counts[b] = 0;
        __syncthreads();
        u64 all = 0;
        if (k <= 0 && by_p)
            by_weight([&](auto weight) {
                for_all([&](float z, int) {
                    if (z > -INFINITY) atomicAdd(&sh.counts[bin_of(z)], 1);
                    all += weight(z);
                });
            });
        else for_slice([&](float z, int) { atomicAdd(&sh.counts[bin_of(z)], 1); });
        all = cluster_sum(all);   // and the counts are whole
        {
            constexpr int B = SP_BINS / SP_THREADS;
            int count[B] = {}, sum = 0;
            float lo = 0.f, hi = 0.f, los[B], his[B];
            counts_of_row(count);
            static_assert(B == 8, "bins of a thread");
#pragma unroll
            for (int j = 0; j < B; ++j) {   // in units of the likeliest token's; bin b is of x from (b - 1/2) / SP_PER to (b + 1/2) / SP_PER
                const float edge = exp2f(-((float)(tid * B + j) - 0.5f) / SP_PER);
                count[j] = sum += count[j];
                const int here = count[j] - (j ? count[j - 1] : 0);
                hi += (float)here * edge;
                lo += tid * B + j == SP_BINS - 1 ? 0.f : (float)here * edge * 0.98922801f;   // 2^(-1 / SP_PER)
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
        const bool by_k = k > 0 && k < sh.cum[SP_BINS - 1];
        // the first bin whose cumulative value is `least` or more
        auto first_bin = [&](auto cumulative, auto least, int which) {
            for (int b = tid; b < SP_BINS; b += SP_THREADS)
                if (cumulative[b] >= least && (b == 0 || !(cumulative[b - 1] >= least))) atomicMin(&sh.found[which], b);
            __syncthreads();
            return sh.found[which];
        };
        auto within = [&](int b0, int b1) { return sh.cum[b1] - (b0 > 0 ? sh.cum[b0 - 1] : 0) <= SP_LIST; };   // whether the list holds those bins
        const int k_bin = by_k ? first_bin(sh.cum, k, 0) : SP_BINS - 1;
        if (by_p && k > 0 && !by_k) {   // more than there are: its mass has not been summed
            u64 s = 0;
            for_slice([&](float z, int) { s += weight(z); });
            all = cluster_sum(s);
        }
        int last = k_bin;   // the last bin that the list needs; top-p takes its share of all that top-k left, those that min-p drops among them
        if (!by_k && by_p) last = first_bin(sh.least, (float)(share * ((double)all / full)) * 1.001f, 1);
        if (min_p > 0.f && !(by_k && by_p)) last = min(last, (int)fminf(fmaxf(-log2f(min_p), 0.f) * SP_PER + 2.f, (float)(SP_BINS - 1)));
        if ((by_k || by_p || min_p > 0.f) && within(0, last)) {
            gather([&](float z) { return bin_of(z) <= last; });
            if (rank == 0) from_list(by_k ? k : SP_LIST, by_k, all);
            return;
        }

        // ---- slices
        auto share_cut = [&]() {   // what the first CTA found, for all
            if (rank == 0 && tid == 0) { sh.cut = cut; sh.listed = 0; }
            cluster.sync();
            cut = *cluster.map_shared_rank(&sh.cut, 0);
            cluster.sync();
        };
        // Where no list holds a bin: of its tokens that stay so far, the last one of the shortest prefix of which the sum of value(logit) reaches `target`, by halving keys;
        // of equal ones, by their count.
        auto halve = [&](int bin, u64 target, auto value) {
            if (tid == 0) { sh.key_range[0] = 0xffffffffu; sh.key_range[1] = 0u; }
            __syncthreads();
            uint32_t lo = 0xffffffffu, hi = 0u;
            for_slice([&](float z, int i) {
                if (bin_of(z) != bin || token_of(key_of(z), first + i) < cut) return;
                lo = min(lo, key_of(z));
                hi = max(hi, key_of(z));
            });
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            if (lane == 0) { atomicMin(&sh.key_range[0], lo); atomicMax(&sh.key_range[1], hi); }
            __syncthreads();
            cluster.sync();
            for (int r = 0; r < C; ++r) {
                lo = min(lo, *cluster.map_shared_rank(&sh.key_range[0], r));
                hi = max(hi, *cluster.map_shared_rank(&sh.key_range[1], r));
            }
            auto total = [&](uint32_t from, bool one) {   // of keys from `from` on, or of that one
                u64 s = 0;
                for_slice([&](float z, int i) {
                    const uint32_t key = key_of(z);
                    if (bin_of(z) == bin && (one ? key == from : key >= from) && token_of(key, first + i) >= cut) s += value(z);
                });
                return cluster_sum(s);
            };
            while (lo < hi) {   // the largest key at which the sum from it on reaches the target
                const uint32_t mid = lo + (hi - lo) / 2 + 1;
                if (total(mid, false) >= target) lo = mid;
                else hi = mid - 1;
            }
            const uint32_t key = lo;
            const u64 ties = total(key, true), each = value(logit_of(key)), before = total(key, false) - ties;
            if (each == 0 || before + ties <= target) return max(cut, token_of(key, 0x7fffffff));   // all of them
            const u64 need = target > before ? (target - before + each - 1) / each : 1ull;
            locate([&](float z, int i) -> u64 { return key_of(z) == key && token_of(key, first + i) >= cut; }, [&](u64) { return need; },
                   [&](int i) { *cluster.map_shared_rank(&sh.index, 0) = i; });
            const int index = *cluster.map_shared_rank(&sh.index, 0);   // behind locate's barrier
            cluster.sync();
            return token_of(key, index);
        };
        if (by_k) {
            const int before = k_bin > 0 ? sh.cum[k_bin - 1] : 0;
            if (within(k_bin, k_bin)) {
                gather([&](float z) { return bin_of(z) == k_bin; });
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
            const int b1 = min(first_bin(sh.least, near * 1.001f, 3), k_bin), b0 = min(first_bin(sh.most, near * 0.999f, 2), b1);
            __syncthreads();   // the bounds have been read; the masses of bins b0 .. b1, exactly, take their place
            for (int b = b0 + tid; b <= b1; b += SP_THREADS) sh.low[b] = sh.high[b] = 0u;
            __syncthreads();
            u64 s = 0;
            by_weight([&](auto weight) {
                for_all([&](float z, int i) {
                    const int b = z > -INFINITY ? bin_of(z) : SP_BINS;
                    const u64 w = weight(z);
                    if (b < b0) s += w;   // ahead of the bins of the border: top-k left them
                    if (b >= b0 && b <= b1 && token_of(key_of(z), first + i) >= cut) {
                        const uint32_t w0 = (uint32_t)w, carry = atomicAdd(&sh.low[b], w0) > ~w0 ? 1u : 0u, w1 = (uint32_t)(w >> 32) + carry;
                        if (w1) atomicAdd(&sh.high[b], w1);
                    }
                });
            });
            s = cluster_sum(s);
            u64 masses[SP_BINS / SP_THREADS];
#pragma unroll
            for (int i = 0; i < SP_BINS / SP_THREADS; ++i) {
                const int b = b0 + tid + i * SP_THREADS;
                masses[i] = 0ull;
                if (b <= b1)
                    for (int r = 0; r < C; ++r) masses[i] += ((u64)*cluster.map_shared_rank(&sh.high[b], r) << 32) + *cluster.map_shared_rank(&sh.low[b], r);
            }
            cluster.sync();   // all have read the slices' masses: the row's take their place
#pragma unroll
            for (int i = 0; i < SP_BINS / SP_THREADS; ++i) {
                const int b = b0 + tid + i * SP_THREADS;
                if (b <= b1) { sh.low[b] = (uint32_t)masses[i]; sh.high[b] = (uint32_t)(masses[i] >> 32); }
            }
            __syncthreads();
            int bin = b1;   // of the border
            for (int b = b0; b < b1; ++b) {
                const u64 here = (u64)sh.high[b] << 32 | sh.low[b];
                if (s + here >= target) { bin = b; break; }
                s += here;
            }
            target = target > s ? target - s : 1ull;
            if (within(bin, bin)) {
                gather([&](float z) { return bin_of(z) == bin; });
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
    }

    // ---- what stays of every warp's run of the slice, of the CTAs', and the token
    const auto found = [&](int i) { a.out[row] = i; };
    if (cut == 0ull && !(min_p > 0.f)) {   // all: nothing weighs what cannot be drawn
        by_weight([&](auto weight) { locate([&](float z, int) { return weight(z); }, draw_target, found); });
    } else {
        by_weight([&](auto weight) {
            locate([&](float z, int i) {
                const u64 w = weight(z);
                return token_of(key_of(z), first + i) >= cut && likely(w) ? w : 0ull;
            }, draw_target, found);
        });
    }
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
    while (vocab > (1ll << 61 >> a.shift)) --a.shift;   // a row's weights add up to 2^61 at most
    switch (dtype) {
    case AB2_F32: return launch_sample<float>(a, rows, (cudaStream_t)stream);
    case AB2_F16: return launch_sample<__half>(a, rows, (cudaStream_t)stream);
    default: return launch_sample<__nv_bfloat16>(a, rows, (cudaStream_t)stream);
    }
}
