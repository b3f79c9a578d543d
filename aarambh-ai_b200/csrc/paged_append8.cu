// Append of new keys (rotated) and values to pages of 8 bits, the queries rotated beside them.  A block is PAGED_BLOCK tokens of a row, at positions 16 b to
// 16 b + 15, of one KV head, keys and values apart; its values are e4m3 codes times its scale
//
//   s = max(2^e, old),   2^e the least power of two with max |x| <= 448 2^e over the new finite x,   old the block's scale if it holds earlier tokens, else 0
//
// Earlier tokens' codes become those of code old / s.  Powers of two move e4m3's exponents and no bits but those that fall below its smallest step, so a block that
// grew token by token holds what one append of all of them would have made, but for 2^-10 of its scale, and a value of 2^e is exact in bf16 too.  448 rather
// than a scale that puts the largest value there exactly: codes are floats, whose relative step does not depend on where they lie.  Inf and NaN become NaN.
//
// A CTA has a block's new tokens (or, where blocks are few, a part of their heads): it turns their angles once into shared memory, and each warp takes heads of q,
// k and v one after the other.  A block's scale is its warp's alone: no atomics, no order.  Heads of keys and values stay in registers from the load to the codes.
//
// Bound by the instructions of a block for prompts, ahead of HBM: issue slots are 44 % busy, and shared memory and registers hold four CTAs on an SM.  Five of up to 2001 tokens, 16 / 4 heads of
// 128 (66 MB), take 24.4 us among other calls, 2.7 TB/s, and 18.4 back to back, where L2 still holds half of it; one of 8192, 32 / 8 heads (185 MB), 48, 3.8 TB/s.  Single tokens by latency: 64 of
// 32 / 8 heads 4.8 us, one 3.4.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

using namespace ab2;

namespace ab2 {
namespace {

constexpr int A8_WARPS = 4, A8_LEAST = -118;   // the smallest exponent of a scale: its inverse is far from f32's end

struct Append8Args {
    const void *q, *k, *v;
    void *qo;
    uint8_t *kp, *vp;
    float *ks, *vs;
    long long q_stride, k_stride, v_stride, qo_stride;   // elements from a token to the next
    int heads, pairs, parts, slots;
    const double *freq;
    float mag;
    PagedView cache;
    int *status;
};

// Two elements: of bf16 in a word, of f32 as they are.
template <typename T> struct Two {
    uint32_t w;
    __device__ __forceinline__ float2 floats() const {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    __device__ __forceinline__ void set(float x, float y) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
        w = *reinterpret_cast<const uint32_t *>(&b);
    }
    __device__ __forceinline__ void load(const T *p) { w = *reinterpret_cast<const uint32_t *>(p); }
    __device__ __forceinline__ void load(const T *p, const T *r) { w = (uint32_t) * reinterpret_cast<const uint16_t *>(p) | (uint32_t) * reinterpret_cast<const uint16_t *>(r) << 16; }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint32_t *>(p) = w; }
    __device__ __forceinline__ void store(T *p, T *r) const { *reinterpret_cast<uint16_t *>(p) = (uint16_t)w; *reinterpret_cast<uint16_t *>(r) = (uint16_t)(w >> 16); }
};
template <> struct Two<float> {
    float2 f;
    __device__ __forceinline__ float2 floats() const { return f; }
    __device__ __forceinline__ void set(float x, float y) { f = make_float2(x, y); }
    __device__ __forceinline__ void load(const float *p) { f = *reinterpret_cast<const float2 *>(p); }
    __device__ __forceinline__ void load(const float *p, const float *r) { f = make_float2(*p, *r); }
    __device__ __forceinline__ void store(float *p) const { *reinterpret_cast<float2 *>(p) = f; }
    __device__ __forceinline__ void store(float *p, float *r) const { *p = f.x; *r = f.y; }
};
__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// HALF: pairs (i, i + n); WIDE: two elements of a lane lie side by side on their boundary, else they are taken one by one; STEP: most rows have a new token each.
template <typename T, int HD, bool HALF, bool WIDE, bool STEP>
__global__ void __launch_bounds__(32 * A8_WARPS, 4) append8_kernel(const __grid_constant__ Append8Args a) {
    constexpr int LANES = HD / 4, AT_ONCE = 32 / LANES;   // lanes of a token's head, tokens a warp has at once
    __shared__ float2 turns[PAGED_BLOCK][HD / 2];
    __shared__ unsigned long long per_position[HD / 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagedView &p = a.cache;
    if (blockIdx.x == 0 && blockIdx.y == 0 && p.starts)   // rows that no block is of are looked over too
        for (int r = threadIdx.x; r < p.rows; r += 32 * A8_WARPS) (void)paged_row(p, r, a.status);
    // The row whose block this is: row b's are numbered from first / 16 + 2 b on, which leaves room for those of any alignment.
    int row = blockIdx.x, number = 0;
    if (p.starts) {
        row = -1;
        for (int r = 0; r < p.rows; r += 32) row += __popc(__ballot_sync(0xffffffffu, r + lane < p.rows && min(max(p.starts[r + lane], 0), p.tokens) / PAGED_BLOCK + 2 * (r + lane) <= (int)blockIdx.x));
        if (row < 0) return;
        number = blockIdx.x - (min(max(p.starts[row], 0), p.tokens) / PAGED_BLOCK + 2 * row);
    }
    const PagedRow r = paged_row(p, row, p.starts ? nullptr : a.status);
    const int before = r.len - r.count;   // tokens ahead of the new ones; negative where a row has more new tokens than tokens, the first of which have no place
    if (before < 0 && threadIdx.x == 0) paged_bad(a.status);
    const int block = max(before, 0) / PAGED_BLOCK + number, pos0 = max(before, block * PAGED_BLOCK), n = min(r.len, (block + 1) * PAGED_BLOCK) - pos0;
    if (n <= 0) return;
    const int skip = pos0 % PAGED_BLOCK;   // earlier tokens of the block
    const long long t0 = r.first + (pos0 - before);
    for (int j = threadIdx.x; j < a.pairs; j += 32 * A8_WARPS) per_position[j] = turns_per_position(__ldg(a.freq + j));
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.pairs; i += 32 * A8_WARPS) {
        const int t = i / a.pairs, j = i - t * a.pairs;
        float2 v;
        turn_cos_sin((unsigned long long)(pos0 + t) * per_position[j], a.mag, v.x, v.y);
        turns[t][j] = v;
    }
    __syncthreads();
    const int id = __ldg(p.table + row * p.table_stride + (pos0 >> p.page_shift));
    const bool kept = (unsigned)id < (unsigned)p.pages;
    if (!kept && threadIdx.x == 0) paged_bad(a.status);
    // a lane has pairs 2 i and 2 i + 1 of a token's head: elements 2 p and 2 p + 1, or those that are turned with the other half's
    const int sub = lane / LANES, p0 = 2 * (lane % LANES);
    auto first_of = [&](int pair, bool turned) { return HALF && turned && pair < a.pairs ? pair : 2 * pair; };
    auto second_of = [&](int pair, bool turned) { return HALF && turned && pair < a.pairs ? pair + a.pairs : 2 * pair + 1; };
    const int tasks = a.heads + 2 * p.kv_heads;
    // The heads of this warp, with room for `steps` tokens a lane.
    auto heads = [&](auto steps) {
        constexpr int STEPS = decltype(steps)::value;
        for (int task = blockIdx.y * A8_WARPS + warp; task < tasks; task += a.parts * A8_WARPS) {
            const bool is_q = task < a.heads, is_v = task >= a.heads + p.kv_heads, turned = !is_v;
            const int head = is_q ? task : (task - a.heads) % p.kv_heads;
            if (!is_q && !kept) continue;
            const long long stride = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;
            const T *src = (const T *)(is_q ? a.q : is_v ? a.v : a.k) + t0 * stride + head * HD;
            const int x0 = first_of(p0, turned), y0 = second_of(p0, turned), x1 = first_of(p0 + 1, turned), y1 = second_of(p0 + 1, turned);
            // with WIDE the two pairs are of one kind: (x0 x1 | y0 y1) of halves, (x0 y0 | x1 y1) otherwise
            const bool halves = HALF && turned && p0 < a.pairs;
            const int o0 = x0, o1 = halves ? x1 : y0, o2 = halves ? y0 : x1, o3 = y1;
            Two<T> u[STEPS], w[STEPS];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int t = i * AT_ONCE + sub;
                u[i].set(0.f, 0.f);
                w[i].set(0.f, 0.f);
                if (t >= n) continue;
                const T *from = src + t * stride;
                if (WIDE) {
                    u[i].load(from + o0);
                    w[i].load(from + o2);
                } else {
                    u[i].load(from + o0, from + o1);
                    w[i].load(from + o2, from + o3);
                }
            }
            if (turned) {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int t = i * AT_ONCE + sub;
                    if (t >= n) continue;
                    float2 e = u[i].floats(), f = w[i].floats();
                    auto turn = [&](float &x, float &y, int pair) {
                        if (pair >= a.pairs) return;
                        const float2 cs = turns[t][pair];
                        const float s = x, v = y;
                        x = s * cs.x - v * cs.y;
                        y = s * cs.y + v * cs.x;
                    };
                    if (halves) {
                        turn(e.x, f.x, p0);
                        turn(e.y, f.y, p0 + 1);
                    } else {
                        turn(e.x, e.y, p0);
                        turn(f.x, f.y, p0 + 1);
                    }
                    u[i].set(e.x, e.y);
                    w[i].set(f.x, f.y);
                }
            }
            if (is_q) {
                T *dst = (T *)a.qo + t0 * a.qo_stride + head * HD;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int t = i * AT_ONCE + sub;
                    if (t >= n) continue;
                    T *to = dst + t * a.qo_stride;
                    if (WIDE) {
                        u[i].store(to + o0);
                        w[i].store(to + o2);
                    } else {
                        u[i].store(to + o0, to + o1);
                        w[i].store(to + o2, to + o3);
                    }
                }
                continue;
            }
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const float2 e = u[i].floats(), f = w[i].floats();
                for (float x : {e.x, e.y, f.x, f.y}) most = is_finite(x) ? fmaxf(most, fabsf(x)) : most;
            }
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
            const uint32_t bits = __float_as_uint(most);
            const int e = max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u), A8_LEAST);   // 448 = 1.75 2^8
            const size_t slot0 = ((((size_t)id * p.kv_heads + head) << p.page_shift) + (size_t)(pos0 & ((1 << p.page_shift) - 1))) - skip;   // the block's first token
            float *scales = (is_v ? a.vs : a.ks) + slot0 / PAGED_BLOCK;
            uint8_t *codes = (is_v ? a.vp : a.kp) + slot0 * HD;
            const float need = __uint_as_float((uint32_t)(e + 127) << 23), old = skip ? *scales : 0.f, scale = fmaxf(need, old), inverse = 1.f / scale;
            __syncwarp();
            if (lane == 0) *scales = scale;
            if (skip && old < scale) {   // earlier tokens' codes in units of the new scale
                const float f = old * inverse;
                for (int t = sub; t < skip; t += AT_ONCE) {
                    uint32_t *at = reinterpret_cast<uint32_t *>(codes + t * HD + 2 * p0);
                    const float2 lo = floats_of_codes(*at), hi = floats_of_codes(*at >> 16);
                    *at = codes_of(lo.x * f, lo.y * f) | codes_of(hi.x * f, hi.y * f) << 16;
                }
            }
            codes += skip * HD;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int t = i * AT_ONCE + sub;
                if (t >= n) continue;
                auto code = [&](float x) { return is_finite(x) ? x * inverse : __uint_as_float(0x7fc00000u); };
                const float2 e = u[i].floats(), f = w[i].floats();
                const uint32_t c0 = codes_of(code(e.x), code(e.y)), c1 = codes_of(code(f.x), code(f.y));
                uint8_t *to = codes + t * HD;
                if (WIDE) {
                    *reinterpret_cast<uint16_t *>(to + o0) = (uint16_t)c0;
                    *reinterpret_cast<uint16_t *>(to + o2) = (uint16_t)c1;
                } else {
                    to[o0] = (uint8_t)c0; to[o1] = (uint8_t)(c0 >> 8);
                    to[o2] = (uint8_t)c1; to[o3] = (uint8_t)(c1 >> 8);
                }
            }
        }
    };
    // Single tokens have a text of their own in steps: the block's unrolled one has to come to the instruction cache first, and took 7.8 us for 4.8 (64 rows, 32 / 8 heads; 512
    // rows 28 for 10.8).  Other batches go without it: five prompts took 20.0 us with both for 18.4, back to back.
    if (STEP && n <= AT_ONCE) heads(std::integral_constant<int, 1>{});
    else heads(std::integral_constant<int, PAGED_BLOCK / AT_ONCE>{});
}

template <typename T, int HD, bool STEP>
int launch_append8(const Append8Args &a, bool half, bool wide, cudaStream_t s) {
    const dim3 grid(a.slots, a.parts);
    auto kernel = half ? (wide ? append8_kernel<T, HD, true, true, STEP> : append8_kernel<T, HD, true, false, STEP>)
                       : (wide ? append8_kernel<T, HD, false, true, STEP> : append8_kernel<T, HD, false, false, STEP>);
    kernel<<<grid, 32 * A8_WARPS, 0, s>>>(a);
    AB2_LAUNCH_CHECK();
    return AB2_OK;
}
template <typename T>
int launch_append8(const Append8Args &a, int head_dim, bool half, bool wide, cudaStream_t s) {
    if (a.cache.tokens <= a.cache.rows) return head_dim == 128 ? launch_append8<T, 128, true>(a, half, wide, s) : launch_append8<T, 64, true>(a, half, wide, s);
    return head_dim == 128 ? launch_append8<T, 128, false>(a, half, wide, s) : launch_append8<T, 64, false>(a, half, wide, s);
}

}  // namespace
}  // namespace ab2

AB2_API int ab2_paged_append_e4m3(const ab2_paged *cache, float *k_scales_dev, float *v_scales_dev, const void *k_dev, long long k_stride, const void *v_dev, long long v_stride, const void *q_dev,
                                  long long q_stride, int heads, void *q_out_dev, long long q_out_stride, const double *frequencies_dev, int rot_dims, int layout, float magnitude, ab2_dtype dtype,
                                  ab2_stream stream) {
    int rc = append_check(cache, 1, k_dev, k_stride, v_dev, v_stride, q_dev, q_stride, heads, q_out_dev, q_out_stride, frequencies_dev, rot_dims, layout, dtype);
    if (rc != AB2_OK) return rc;
    AB2_REQUIRE(k_scales_dev && v_scales_dev, AB2_ERR_BAD_ARG, "null scales");
    AB2_REQUIRE((((uintptr_t)k_scales_dev | (uintptr_t)v_scales_dev) & 3) == 0, AB2_ERR_BAD_ALIGN, "scales must lie on their elements");
    if (cache->tokens == 0) return AB2_OK;
    const long long es = (long long)dtype_size(dtype), pool = (long long)cache->pages * cache->page_size * cache->kv_heads * cache->head_dim, blocks = pool / cache->head_dim / PAGED_BLOCK * 4;
    const long long row = (long long)heads * cache->head_dim, krow = (long long)cache->kv_heads * cache->head_dim;
    const RowsAt ks = {k_scales_dev, blocks, blocks, 1}, vs = {v_scales_dev, blocks, blocks, 1}, kp = {cache->k_pages, pool, pool, 1}, vp = {cache->v_pages, pool, pool, 1};
    const RowsAt read[4] = {{k_dev, krow * es, k_stride * es, cache->tokens}, {v_dev, krow * es, v_stride * es, cache->tokens}, {heads ? q_dev : nullptr, row * es, q_stride * es, cache->tokens},
                            {heads ? q_out_dev : nullptr, row * es, q_out_stride * es, cache->tokens}};
    for (const RowsAt &x : read)
        AB2_REQUIRE(!rows_meet(ks, x) && !rows_meet(vs, x) && !rows_meet(kp, x) && !rows_meet(vp, x), AB2_ERR_BAD_ARG, "pages and scales lie apart from queries, keys and values");
    AB2_REQUIRE(!rows_meet(ks, vs) && !rows_meet(ks, kp) && !rows_meet(ks, vp) && !rows_meet(vs, kp) && !rows_meet(vs, vp), AB2_ERR_BAD_ARG, "pages and scales of keys and of values lie apart");
    Append8Args a = {};
    a.k = k_dev; a.v = v_dev; a.k_stride = k_stride; a.v_stride = v_stride;
    if (heads) { a.q = q_dev; a.qo = q_out_dev; a.q_stride = q_stride; a.qo_stride = q_out_stride; }
    a.heads = heads; a.pairs = rot_dims / 2; a.freq = frequencies_dev; a.mag = magnitude;
    a.cache = paged_view(cache); a.kp = (uint8_t *)cache->k_pages; a.vp = (uint8_t *)cache->v_pages; a.ks = k_scales_dev; a.vs = v_scales_dev;
    rc = device_status_word(&a.status);
    if (rc != AB2_OK) return rc;
    const long long slots = cache->starts ? cache->tokens / PAGED_BLOCK + 2ll * cache->rows + 1 : cache->rows;
    AB2_REQUIRE(slots < (1ll << 31), AB2_ERR_BAD_SHAPE, "%d tokens of %d rows are more than one launch takes", cache->tokens, cache->rows);
    a.slots = (int)slots;
    // A CTA has all heads of a block where there are blocks enough for four CTAs on every SM, else fewer: a head a warp at least.  Sharing a block out makes its angles
    // anew in every CTA: for 4 and 8 CTAs on an SM, us, five prompts of up to 2001 tokens 18.5 and 17.7, one of 8192 55 and 56.
    const int tasks = heads + 2 * cache->kv_heads, most = (tasks + A8_WARPS - 1) / A8_WARPS;
    const long long filled = std::max(1ll, cache->starts ? std::min<long long>(slots, cache->tokens / PAGED_BLOCK + cache->rows) : slots);
    a.parts = (int)std::min<long long>(std::min(most, 65535), std::max(1ll, (4ll * device_sm_count() + filled - 1) / filled));
    uintptr_t where = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.qo;
    const bool wide = a.pairs % 2 == 0 && where % (2 * es) == 0 && (a.q_stride | a.k_stride | a.v_stride | a.qo_stride) % 2 == 0, half = layout == AB2_ROTARY_HALF;
    cudaStream_t s = (cudaStream_t)stream;
    return dtype == AB2_F32 ? launch_append8<float>(a, cache->head_dim, half, wide, s) : launch_append8<__nv_bfloat16>(a, cache->head_dim, half, wide, s);
}
