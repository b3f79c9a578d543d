// Attention of a ragged batch of new tokens over a paged cache: row b's new tokens are its last ones, and its i-th sees the keys up to its own
// position, len - new + i.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = scale log2(e) q k_j,   m the running maximum
//
// One pass over the keys: each tile of scores moves m, rescales what has been summed, and adds its weights and values.  Scores, weights,
// their sums and the sums of values are f32.  A query that sees no key answers zeros.
//
// This file: f32, on CUDA cores; attention_paged_mma.cu and attention_paged_tc.cu: bf16.
// A CTA multiplies the queries of a KV head's whole group (tokens x heads of the group, up to QR rows) with a tile of 32 keys on CUDA cores;
// keys and values come by cp.async, the next tile's while this one's are looked at.  Values are summed over a tile and
// then joined to the others', which rounds once a tile.  500 tokens behind 1000, 16 / 4 heads of 128: 170 us, 30 TFLOP/s, by tiles of 64 rows, whose scores
// load 16 bytes from shared memory eight times for 64 multiplications; by tiles of 32, six times for 32, 229.  Three rows of up to 130 tokens behind 380,
// 6 / 2 heads of 64: 22.4 us (a kernel of 18 and a merge of 7 by
// themselves, before a launch was set up while the one before it ended).
#include <algorithm>

#include "paged.cuh"

using namespace ab2;

namespace ab2 {
int paged_check(const ab2_paged *c, ab2_dtype dtype);
PagedView paged_view(const ab2_paged *c);
size_t paged_mma_bytes(int hd);
int paged_mma_attention(const PagedAttnArgs &a, int hd, int max_new, void *workspace, size_t bytes, cudaStream_t s);
size_t paged_tc_bytes(int hd);
int paged_tc_attention(const PagedAttnArgs &a, int hd, void *workspace, size_t bytes, cudaStream_t s);
// A batch of chunks and single tokens: one launch for both up to this many rows times KV heads, since a launch for the single tokens and its merge cost more than
// they save; but in the kernel of chunks each of them takes a tile of 128 rows, and loses by its context, which the host does not know.  A chunk of 512 among
// single tokens, us by two launches and by one: 32 / 8 heads of 128, 32 rows behind 500 65 and 56, behind 4000 168 and 163, behind 16000 487 and 559; 64 rows 82 and 80,
// 247 and 274; 16 / 1 heads of 128, 128 rows behind 500 57 and 40, behind 4000 118 and 98; 16 / 4 heads of 64, 16 rows behind 500 43 and 29, behind 4000 61 and 62, behind 16000
// 141 and 178, 32 rows 42 and 33, 80 and 90, 180 and 284.
constexpr int paged_few_items(int hd) { return hd == 128 ? 256 : 64; }
constexpr int PAGED_FEW_ROWS = 16;   // query rows of a KV head up to which the tensor-memory kernel's tiles of 128 would be nearly empty
namespace {

constexpr int PA_THREADS = 128, PA_KEYS = 32;
constexpr int TALL_ROWS = 512, TALL_ALL = 2560;

template <int HD, int QR> struct SimtShape {
    static constexpr int TX = QR == 8 ? 16 : 8, TY = PA_THREADS / TX, RPT = QR / TY, KPT = PA_KEYS / TX, DPT = HD / TX;
    // Row i of a thread: two are neighbours, which see much the same keys; four lie TY apart, or those of a warp would meet in the same banks.
    static constexpr int STEP = RPT == 4 ? TY : 1, FIRST = RPT == 4 ? 1 : RPT;
    static constexpr int KROW = HD + 4, PROW = PA_KEYS + 4;   // a row's bank moves on by 16 bytes
    static constexpr int BUF = PA_KEYS * KROW * 4;
    static constexpr int SMEM = 4 * BUF + QR * KROW * 4 + QR * PROW * 4;
    static constexpr int CTAS = HD == 128 ? 2 : QR == 64 ? 3 : 4;   // of an SM: what shared memory holds
};

__device__ __forceinline__ void cp16(void *dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
template <int HD, int QR>
__global__ void __launch_bounds__(PA_THREADS, SimtShape<HD, QR>::CTAS) paged_simt_kernel(const __grid_constant__ PagedAttnArgs a) {
    using S = SimtShape<HD, QR>;
    pdl_wait();
    constexpr int TX = S::TX, RPT = S::RPT, KPT = S::KPT, DPT = S::DPT, KROW = S::KROW, PROW = S::PROW, STEP = S::STEP, CH = 4;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ long long warp_sums[PA_THREADS / 32];
    __shared__ int2 found[2];
    float *kbuf = (float *)smem, *vbuf = kbuf + 2 * PA_KEYS * KROW;
    float *qs = (float *)(smem + 4 * S::BUF), *ps = qs + QR * KROW;
    const int tx = threadIdx.x % TX, row0 = threadIdx.x / TX * S::FIRST;
    const PagedView &p = a.plan.p;
    PagedRun run = paged_run<PA_THREADS>(a.plan, blockIdx.x, gridDim.x, warp_sums, found, a.status);
    if (threadIdx.x == 0) paged_uncut(a, blockIdx.x);
    PagedPiece w;
    while (paged_next(a.plan, run, w)) {
        const PagedSpan sp = paged_span(a.plan, w);
        if (threadIdx.x == 0) paged_cut(a, run, w, sp, blockIdx.x);
        const int t0 = sp.t0, ntok = sp.ntok, base = sp.base, lo = sp.lo, hi = sp.hi, group = a.plan.group;
        __syncthreads();
        for (int i = threadIdx.x; i < QR * HD / 4; i += PA_THREADS) {
            const int r = i / (HD / 4), d = i % (HD / 4) * 4, tok = paged_token(a.plan, r), g = r - tok * group;
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (tok < ntok) f = load4((const float *)a.q + (size_t)(w.r.first + t0 + tok) * a.q_stride + (size_t)(w.head * group + g) * HD + d);
            *reinterpret_cast<float4 *>(qs + r * KROW + d) = make_float4(f.x * a.sl, f.y * a.sl, f.z * a.sl, f.w * a.sl);
        }
        // rows past the last key read as zeros
        auto fetch = [&](int key0, int buf) {
            for (int i = threadIdx.x; i < PA_KEYS * HD / CH; i += PA_THREADS) {
                const int j = i / (HD / CH), d = i % (HD / CH) * CH, key = key0 + j;
                const bool in = key < hi;
                const int at = in ? key : lo;
                const size_t row = (((size_t)paged_page(p, w.row, at, a.status) * p.kv_heads + w.head) << p.page_shift) + (at & ((1 << p.page_shift) - 1));
                cp16(kbuf + (buf * PA_KEYS + j) * KROW + d, (const float *)a.k + row * HD + d, in);
                cp16(vbuf + (buf * PA_KEYS + j) * KROW + d, (const float *)a.v + row * HD + d, in);
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
        float top[RPT], sum[RPT], o[RPT][DPT];
        int lim[RPT], seen = -1, sure = hi - 1;   // the last key that any row of the thread sees, and the last that all do
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int tok = paged_token(a.plan, row0 + STEP * i);
            lim[i] = tok < ntok ? base + t0 + tok : 0x7fffffff;   // a row without a token is not looked at, and keeps no other from what all see
            if (tok < ntok) seen = lim[i];                        // rows go by tokens
            sure = min(sure, lim[i]);
            top[i] = -INFINITY;
            sum[i] = 0.f;
#pragma unroll
            for (int d = 0; d < DPT; ++d) o[i][d] = 0.f;
        }
        if (lo < hi) fetch(lo, 0);
        for (int key0 = lo, buf = 0; key0 < hi; key0 += PA_KEYS, buf ^= 1) {
            if (key0 + PA_KEYS < hi) {
                fetch(key0 + PA_KEYS, buf ^ 1);
                asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;\n" ::: "memory");
            }
            __syncthreads();
            float4 s4[RPT][KPT];   // a score as four sums: shorter chains, for time and for rounding
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) s4[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                float4 qv[RPT], kv[KPT];
#pragma unroll
                for (int i = 0; i < RPT; ++i) qv[i] = *reinterpret_cast<const float4 *>(qs + (row0 + STEP * i) * KROW + d);
#pragma unroll
                for (int j = 0; j < KPT; ++j) kv[j] = load4(kbuf + (buf * PA_KEYS + tx + TX * j) * KROW + d);
#pragma unroll
                for (int i = 0; i < RPT; ++i)
#pragma unroll
                    for (int j = 0; j < KPT; ++j) {
                        s4[i][j].x = fmaf(qv[i].x, kv[j].x, s4[i][j].x); s4[i][j].y = fmaf(qv[i].y, kv[j].y, s4[i][j].y);
                        s4[i][j].z = fmaf(qv[i].z, kv[j].z, s4[i][j].z); s4[i][j].w = fmaf(qv[i].w, kv[j].w, s4[i][j].w);
                    }
            }
            // the sums of this tile's values alone, joined to the others' at its end: one chain over all keys would round once a key and not once a tile
            float s[RPT][KPT], keep[RPT], here[RPT][DPT];
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
                float best = top[i];
#pragma unroll
                for (int j = 0; j < KPT; ++j) {
                    const int key = key0 + tx + TX * j;
                    s[i][j] = (s4[i][j].x + s4[i][j].y) + (s4[i][j].z + s4[i][j].w);
                    if (key > lim[i] || key >= hi) s[i][j] = -INFINITY;   // out of sight, whatever it holds
                    best = fmaxf(best, s[i][j]);
                }
#pragma unroll
                for (int m = TX / 2; m > 0; m >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, m));
                const float m = best == -INFINITY ? 0.f : best;
                keep[i] = exp2f(top[i] - m);
                top[i] = best;
                float weights = 0.f;
#pragma unroll
                for (int d = 0; d < DPT; ++d) here[i][d] = 0.f;
#pragma unroll
                for (int j = 0; j < KPT; ++j) {
                    const int key = key0 + tx + TX * j;
                    const float e = key > lim[i] || key >= hi ? 0.f : exp2f(s[i][j] - m);
                    weights += e;
                    ps[(row0 + STEP * i) * PROW + tx + TX * j] = e;
                }
                sum[i] = fmaf(sum[i], keep[i], weights);
            }
            __syncwarp();  // a row's weights come from lanes of one warp
            // keys that no row of the thread sees may hold anything: their weight is 0, and 0 times Inf is not
            const bool every = RPT > 1 && seen >= 0 && key0 + PA_KEYS - 1 <= sure;   // of the tile's keys is seen by every row of the thread
            if (every) {
#pragma unroll 2
                for (int j = 0; j < PA_KEYS; j += 4) {
                    float4 e[RPT];
#pragma unroll
                    for (int i = 0; i < RPT; ++i) e[i] = load4(ps + (row0 + STEP * i) * PROW + j);
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                        for (int d = 0; d < DPT; d += 4) {
                            const float4 v = load4(vbuf + (buf * PA_KEYS + j + jj) * KROW + tx * 4 + d * TX);
#pragma unroll
                            for (int i = 0; i < RPT; ++i) {
                                const float f = jj == 0 ? e[i].x : jj == 1 ? e[i].y : jj == 2 ? e[i].z : e[i].w;
                                here[i][d] = fmaf(f, v.x, here[i][d]);
                                here[i][d + 1] = fmaf(f, v.y, here[i][d + 1]);
                                here[i][d + 2] = fmaf(f, v.z, here[i][d + 2]);
                                here[i][d + 3] = fmaf(f, v.w, here[i][d + 3]);
                            }
                        }
                }
            }
            const int n = every ? 0 : min(PA_KEYS, min(hi - key0, seen + 1 - key0));
            for (int j = 0; j < n; ++j) {
                float e[RPT];
#pragma unroll
                for (int i = 0; i < RPT; ++i) e[i] = ps[(row0 + STEP * i) * PROW + j];
#pragma unroll
                for (int d = 0; d < DPT; d += 4) {
                    const float4 v = load4(vbuf + (buf * PA_KEYS + j) * KROW + tx * 4 + d * TX);
#pragma unroll
                    for (int i = 0; i < RPT; ++i) {
                        if (RPT > 1 && key0 + j > lim[i]) continue;
                        here[i][d] = fmaf(e[i], v.x, here[i][d]);
                        here[i][d + 1] = fmaf(e[i], v.y, here[i][d + 1]);
                        here[i][d + 2] = fmaf(e[i], v.z, here[i][d + 2]);
                        here[i][d + 3] = fmaf(e[i], v.w, here[i][d + 3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int d = 0; d < DPT; ++d) o[i][d] = fmaf(o[i][d], keep[i], here[i][d]);
            __syncthreads();
        }
        const bool all = w.k0 == 0 && w.k1 == w.k_tiles;
        const size_t slot = 2 * (size_t)blockIdx.x + (w.k0 == 0);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = row0 + STEP * i, tok = paged_token(a.plan, r), g = r - tok * group;
#pragma unroll
            for (int m = TX / 2; m > 0; m >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], m);
            if (tok >= ntok) continue;
            if (all) {
                const float f = sum[i] == 0.f ? 0.f : 1.f / sum[i];
                float *dst = (float *)a.out + (size_t)(w.r.first + t0 + tok) * a.o_stride + (size_t)(w.head * group + g) * HD;
#pragma unroll
                for (int d = 0; d < DPT; d += 4) *reinterpret_cast<float4 *>(dst + tx * 4 + d * TX) = make_float4(o[i][d] * f, o[i][d + 1] * f, o[i][d + 2] * f, o[i][d + 3] * f);
            } else {
                float *dst = a.acc + (slot * QR + r) * HD;
#pragma unroll
                for (int d = 0; d < DPT; d += 4) *reinterpret_cast<float4 *>(dst + tx * 4 + d * TX) = make_float4(o[i][d], o[i][d + 1], o[i][d + 2], o[i][d + 3]);
                if (tx == 0) { a.ml[(slot * QR + r) * 2] = top[i]; a.ml[(slot * QR + r) * 2 + 1] = sum[i]; }
            }
        }
    }
}

// The pieces of cut items: CTA (c, y) finishes rows of the item that run c of the launch before began and did not end.  GROUPS times 128 threads share an
// item's pieces out: there are two or three where a run is a CTA's, and up to as many as there are runs where it is a warp's.  With one group a
// thread's first pieces are asked for before the rows' maxima, on which their factors wait (64 tokens behind 4000, 18 pieces an item: 33 us for 35).
constexpr int MERGE_ROWS = 16;   // of a CTA
template <typename T, int HD, int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS) paged_merge_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int LANES = 8 * GROUPS;   // of a row, for its maximum
    constexpr int POS = GROUPS == 1 ? MERGE_ROWS * HD / 512 : 1, BATCH = 2;   // places of a thread and, with one group, pieces that it holds at once
    __shared__ float tops[MERGE_ROWS], sums[MERGE_ROWS];
    __shared__ float4 others[GROUPS][128];
    pdl_wait();
    pdl_launch_dependents();   // behind the wait, so that no more than one launch waits at a time
    const int c = blockIdx.x, group = a.plan.group, part = threadIdx.x / 128, me = threadIdx.x % 128;
    const size_t row0 = (size_t)blockIdx.y * MERGE_ROWS;
    const int4 cut = a.cut[c];
    const int rows = min(cut.y * group - (int)row0, MERGE_ROWS), pieces = cut.w - c + 1;
    if (rows <= 0) return;
    // run c's piece is its last, the others' is their first: slots 2 c + 1, 2 c + 2, 2 c + 4, ...
    auto slot = [&](int j) { return (2 * (size_t)(c + j) + (j == 0)) * a.tile_rows + row0; };
    float4 v[BATCH][POS];
    auto fetch = [&](int i0, int j0) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
#pragma unroll
            for (int k = 0; k < POS; ++k) {
                const int j = j0 + b * GROUPS, i = i0 + 128 * k + me, r = i / (HD / 4);
                v[b][k] = j < pieces && r < rows ? *reinterpret_cast<const float4 *>(a.acc + (slot(j) + r) * HD + i % (HD / 4) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
    };
    if (GROUPS == 1) fetch(0, part);
    {   // a row's maximum over all pieces, and the sum of its weights relative to it
        const int r = threadIdx.x / LANES;
        float top = -INFINITY, sum = 0.f;
        if (r < rows)
#pragma unroll 4
            for (int j = threadIdx.x % LANES; j < pieces; j += LANES) top = fmaxf(top, a.ml[(slot(j) + r) * 2]);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m = top == -INFINITY ? 0.f : top;
        if (r < rows)
#pragma unroll 4
            for (int j = threadIdx.x % LANES; j < pieces; j += LANES) {
                const float2 ml = *reinterpret_cast<const float2 *>(a.ml + (slot(j) + r) * 2);
                sum = fmaf(ml.y, exp2f(ml.x - m), sum);
            }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x % LANES == 0) { tops[r] = m; sums[r] = sum; }
    }
    __syncthreads();
    for (int i0 = 0; i0 < rows * (HD / 4); i0 += 128 * POS) {
        float4 o[POS];
#pragma unroll
        for (int k = 0; k < POS; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (GROUPS > 1) {
            const int i = i0 + me, r = i / (HD / 4), d = i % (HD / 4) * 4;
            if (r < rows)
#pragma unroll 8
                for (int j = part; j < pieces; j += GROUPS) {
                    const float f = exp2f(a.ml[(slot(j) + r) * 2] - tops[r]);
                    const float4 x = *reinterpret_cast<const float4 *>(a.acc + (slot(j) + r) * HD + d);
                    o[0].x = fmaf(f, x.x, o[0].x); o[0].y = fmaf(f, x.y, o[0].y); o[0].z = fmaf(f, x.z, o[0].z); o[0].w = fmaf(f, x.w, o[0].w);
                }
        }
        for (int j0 = part; GROUPS == 1 && j0 < pieces; j0 += BATCH) {
            if (i0 > 0 || j0 > part) fetch(i0, j0);
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
#pragma unroll
                for (int k = 0; k < POS; ++k) {
                    const int j = j0 + b * GROUPS, r = (i0 + 128 * k + me) / (HD / 4);
                    const float f = j < pieces && r < rows ? exp2f(a.ml[(slot(j) + r) * 2] - tops[r]) : 0.f;
                    o[k].x = fmaf(f, v[b][k].x, o[k].x); o[k].y = fmaf(f, v[b][k].y, o[k].y);
                    o[k].z = fmaf(f, v[b][k].z, o[k].z); o[k].w = fmaf(f, v[b][k].w, o[k].w);
                }
        }
        if (GROUPS > 1) {
            if (i0 > 0) __syncthreads();   // the sums before have been taken
            others[part][me] = o[0];
            __syncthreads();
            if (part > 0) continue;
            for (int g = 1; g < GROUPS; ++g) {
                const float4 x = others[g][me];
                o[0].x += x.x; o[0].y += x.y; o[0].z += x.z; o[0].w += x.w;
            }
        }
#pragma unroll
        for (int k = 0; k < POS; ++k) {
            const int i = i0 + 128 * k + me, r = i / (HD / 4), d = i % (HD / 4) * 4;
            if (r >= rows) continue;
            const float f = sums[r] == 0.f ? 0.f : 1.f / sums[r];
            const int row = (int)row0 + r, tok = paged_token(a.plan, row);
            T *dst = (T *)a.out + (size_t)(cut.x + tok) * a.o_stride + (size_t)(cut.z * group + row - tok * group) * HD + d;
            alignas(16) T y[4] = {from_f32<T>(o[k].x * f), from_f32<T>(o[k].y * f), from_f32<T>(o[k].z * f), from_f32<T>(o[k].w * f)};
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(y);
            else *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(y);
        }
    }
}

template <int HD, int QR> size_t simt_bytes() { return paged_piece_bytes(SimtShape<HD, QR>::CTAS * device_sm_count(), QR, HD); }

template <int HD, int QR>
int launch_simt(PagedAttnArgs a, void *workspace, size_t bytes, cudaStream_t s) {
    using S = SimtShape<HD, QR>;
    static bool configured[64] = {false};  // the attribute is per device
    int dev = 0;
    AB2_CUDA(cudaGetDevice(&dev));
    AB2_REQUIRE(dev >= 0 && dev < 64, AB2_ERR_BAD_ARG, "device index %d out of range", dev);
    if (!configured[dev]) {
        AB2_CUDA(cudaFuncSetAttribute(paged_simt_kernel<HD, QR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        configured[dev] = true;
    }
    paged_deal(a, S::CTAS * device_sm_count(), QR, 5, 1, HD, workspace, bytes);
    ChainedLaunches chained(true);   // the launch before it, an append or a merge, need not have ended when this one is set up: it waits in the kernel
    AB2_CUDA(launch_kernel(paged_simt_kernel<HD, QR>, dim3(a.ctas), dim3(PA_THREADS), S::SMEM, s, a));
    return a.plan.whole ? AB2_OK : paged_merge(a, HD, AB2_F32, s);
}

int simt_attention(const PagedAttnArgs &a, int hd, int max_new, void *workspace, size_t bytes, cudaStream_t s) {
    // Tiles of 64 rows load a third less from shared memory but are half as many, with more rows that no token fills.  They pay for long chunks: from 512 query
    // rows a KV head of a sequence, where the batch has 2560 of all heads to share out (us by tiles of 32 and of
    // 64: 500 tokens behind 1000, 16 heads of 128, 229 and 170; 200 behind 1000 88 and 78; 5 x 60 behind 500 41 and 43; 100 behind 1000, 6 heads of 64, 26 and 33).
    const long long rows = max_new * (long long)a.plan.group, all = (long long)a.plan.p.tokens * a.plan.group * a.plan.p.kv_heads;
    const bool tall = rows >= TALL_ROWS && all >= TALL_ALL;
    if (hd == 128) return rows <= 8 ? launch_simt<128, 8>(a, workspace, bytes, s) : tall ? launch_simt<128, 64>(a, workspace, bytes, s) : launch_simt<128, 32>(a, workspace, bytes, s);
    return rows <= 8 ? launch_simt<64, 8>(a, workspace, bytes, s) : tall ? launch_simt<64, 64>(a, workspace, bytes, s) : launch_simt<64, 32>(a, workspace, bytes, s);
}

}  // namespace

int paged_merge(const PagedAttnArgs &a, int hd, ab2_dtype dtype, cudaStream_t s) {
    ChainedLaunches chained(true);
    const dim3 grid(a.ctas, (a.tile_rows + MERGE_ROWS - 1) / MERGE_ROWS);
    const bool tall = a.tile_rows > 32;   // a run is a CTA's, and few of them share an item
    auto kernel = dtype == AB2_F32 ? (tall ? (hd == 128 ? paged_merge_kernel<float, 128, 1> : paged_merge_kernel<float, 64, 1>)
                                           : (hd == 128 ? paged_merge_kernel<float, 128, 4> : paged_merge_kernel<float, 64, 4>))
                  : tall           ? (hd == 128 ? paged_merge_kernel<__nv_bfloat16, 128, 1> : paged_merge_kernel<__nv_bfloat16, 64, 1>)
                                   : (hd == 128 ? paged_merge_kernel<__nv_bfloat16, 128, 4> : paged_merge_kernel<__nv_bfloat16, 64, 4>);
    cudaError_t e = launch_kernel(kernel, grid, dim3(tall ? 128 : 512), 0, s, a);
    if (e != cudaSuccess) return fail(AB2_ERR_CUDA, "paged attention launch failed: %s", cudaGetErrorString(e));
    return AB2_OK;
}

}  // namespace ab2

AB2_API int ab2_paged_workspace(int head_dim, size_t *bytes) {
    AB2_REQUIRE(bytes, AB2_ERR_BAD_ARG, "null argument");
    AB2_REQUIRE(head_dim == 64 || head_dim == 128, AB2_ERR_UNSUPPORTED, "paged caches have heads of 64 or 128, not %d", head_dim);
    const size_t simt = head_dim == 128 ? std::max(simt_bytes<128, 32>(), simt_bytes<128, 64>()) : std::max(simt_bytes<64, 32>(), simt_bytes<64, 64>());
    *bytes = std::max(simt, std::max(paged_mma_bytes(head_dim), paged_tc_bytes(head_dim)));
    return AB2_OK;
}

AB2_API int ab2_paged_attention(const ab2_paged *cache, const void *q_dev, long long q_stride, int heads, void *out_dev, long long out_stride, int max_new, float scale,
                                void *workspace_dev, size_t workspace_bytes, ab2_dtype dtype, ab2_stream stream) {
    int rc = paged_check(cache, dtype);
    if (rc != AB2_OK) return rc;
    AB2_REQUIRE(heads > 0 && heads % cache->kv_heads == 0 && heads / cache->kv_heads <= 32, AB2_ERR_BAD_SHAPE, "%d query heads over %d KV heads: a multiple of them up to 32 is served", heads, cache->kv_heads);
    AB2_REQUIRE(max_new > 0, AB2_ERR_BAD_SHAPE, "rows of at most %d new tokens", max_new);
    if (cache->tokens == 0) return AB2_OK;
    AB2_REQUIRE(q_dev && out_dev, AB2_ERR_BAD_ARG, "null argument");
    const long long row = (long long)heads * cache->head_dim;
    AB2_REQUIRE(q_stride >= row && out_stride >= row, AB2_ERR_BAD_SHAPE, "a token's heads lie one after the other, and tokens do not overlap");
    const size_t esize = dtype_size(dtype);
    AB2_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)workspace_dev) & 15) == 0 && ((q_stride | out_stride) * esize & 15) == 0, AB2_ERR_BAD_ALIGN, "queries, outputs and their rows must be 16-byte aligned");
    // a query, key or value may be read after outputs have been written
    const long long es = (long long)esize, pool = (long long)cache->pages * cache->page_size * cache->kv_heads * cache->head_dim * es;
    const RowsAt o_at = {out_dev, row * es, out_stride * es, cache->tokens};
    AB2_REQUIRE(!rows_meet(o_at, {q_dev, row * es, q_stride * es, cache->tokens}) && !rows_meet(o_at, {cache->k_pages, pool, pool, 1}) && !rows_meet(o_at, {cache->v_pages, pool, pool, 1}), AB2_ERR_BAD_ARG,
                "the outputs may not take the place of queries or pages");
    PagedAttnArgs a = {};
    a.plan.p = paged_view(cache);
    a.q = q_dev; a.k = cache->k_pages; a.v = cache->v_pages; a.out = out_dev; a.q_stride = q_stride; a.o_stride = out_stride;
    a.plan.group = heads / cache->kv_heads; a.plan.above = 0; a.plan.most = 0x7fffffff; a.sl = scale * 1.44269504088896341f;
    rc = device_status_word(&a.status);
    if (rc != AB2_OK) return rc;
    if (!cache->starts) max_new = 1;
    if (dtype == AB2_F32) return simt_attention(a, cache->head_dim, max_new, workspace_dev, workspace_bytes, (cudaStream_t)stream);
    // Rows of up to 16 query rows a KV head go to the warp-level kernel, the others to the tensor-memory kernel; a launch for which there can be no row is
    // left out.  Rows with more new tokens than they were said to have are served all the same.
    const bool chunks = (long long)max_new * a.plan.group > PAGED_FEW_ROWS, few = a.plan.group <= PAGED_FEW_ROWS && !(chunks && (long long)cache->rows * cache->kv_heads <= paged_few_items(cache->head_dim));
    if (few) {
        if (chunks) a.plan.most = PAGED_FEW_ROWS;
        rc = paged_mma_attention(a, cache->head_dim, max_new, workspace_dev, workspace_bytes, (cudaStream_t)stream);
        if (rc != AB2_OK || !chunks) return rc;
        a.plan.above = PAGED_FEW_ROWS;
        a.plan.most = 0x7fffffff;
    }
    return paged_tc_attention(a, cache->head_dim, workspace_dev, workspace_bytes, (cudaStream_t)stream);
}
