// Rotary positions of a batch of tokens, alone or together with the append of their keys and values to a paged cache.
//
//   turned pair i of a head at position p = m R(p f_i) (x_i, y_i),   R a rotation, f_i radians a position, m a magnitude
//
// Pairs are (i, i + n) with the half layout and (2i, 2i + 1) with the interleaved one, n = rot / 2 of them; the dimensions from rot on pass
// as they are.  One pass over q and k (and v, which is copied into its pages): bound by HBM from some hundred tokens on, by the launch
// below: 8192 tokens of 32 / 8 heads of 128 in bf16 31 us, 5.3 TB/s (0.82 of a copy's); 5891 tokens of 16 / 4 appended 19 us; 8 tokens 4 us.
// A warp has one token (or a part of its heads where tokens are few): its lanes turn the token's angles once, into shared memory, and then take
// (head, P pairs) of q, k and v one tensor after the other; where a head's chunks divide 32 a lane keeps its pairs from head to head.  The first
// form, whose lanes made every angle for themselves, took 35 us; this one with elements of 16 bits held as such, not in words, 39.
#include <algorithm>

#include "paged.cuh"

using namespace ab2;

namespace ab2 {
namespace {

constexpr int ROT_WARPS = 4, ROT_BATCH = 4;  // heads of a lane in flight

struct RotArgs {
    const void *q, *k, *v;
    void *qo, *ko;
    long long q_stride, k_stride, v_stride, qo_stride, ko_stride;  // elements from a token to the next
    int heads, kv_heads, dim, pairs, tokens, chunks;               // chunks of P pairs a head has, the unturned dimensions among them
    int per_warp, parts;                                           // heads of q, k and v of a warp, warps of a token
    const void *pos;
    int pos64;
    const double *freq;
    float mag;
    PagedView cache;  // with PAGED: k and v go there, and positions are those in their rows
    void *kp, *vp;
    int *status;
};

// E elements in loads and stores of up to 16 bytes, held as 32-bit words (one element: as itself).
template <typename T, int E> struct Vec {
    static constexpr int WORDS = E * (int)sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (WORDS % 4 == 0) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) { const uint4 v = *reinterpret_cast<const uint4 *>((const uint32_t *)p + i); w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w; }
        } else {
            static_assert(WORDS == 2, "chunks of 8 or 16 bytes");
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x; w[1] = v.y;
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (WORDS % 4 == 0) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) *reinterpret_cast<uint4 *>((uint32_t *)p + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        }
    }
};
template <typename T> struct Vec<T, 1> {
    T e;
    __device__ __forceinline__ void load(const T *p) { e = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = e; }
};
__device__ __forceinline__ float2 two_of(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 two_of(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ uint32_t word_of(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
__device__ __forceinline__ uint32_t word_of(float lo, float hi, __half) {
    const __half2 b = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
__device__ __forceinline__ void turn(float &x, float &y, float c, float s) {
    const float u = x, v = y;
    x = u * c - v * s;
    y = u * s + v * c;
}

// A chunk of P pairs turned: x and y are its first P elements and its others.  (Interleaved: pair j is elements 2 j and 2 j + 1 of the 2 P.)
template <typename T, int P, bool HALF> __device__ __forceinline__ void rot_turn(Vec<T, P> &x, Vec<T, P> &y, const float (&c)[P], const float (&s)[P]) {
    if constexpr (P == 1) {
        float u = to_f32(x.e), v = to_f32(y.e);
        turn(u, v, c[0], s[0]);
        x.e = from_f32<T>(u);
        y.e = from_f32<T>(v);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            uint32_t &e0 = HALF ? x.w[j] : 2 * j < P ? x.w[(2 * j) % P] : y.w[(2 * j) % P];
            uint32_t &e1 = HALF ? y.w[j] : 2 * j + 1 < P ? x.w[(2 * j + 1) % P] : y.w[(2 * j + 1) % P];
            float u = __uint_as_float(e0), v = __uint_as_float(e1);
            turn(u, v, c[j], s[j]);
            e0 = __float_as_uint(u);
            e1 = __float_as_uint(v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < P / 2; ++j) {
            float2 u = two_of(x.w[j], T()), v = two_of(y.w[j], T());
            if (HALF) {
                turn(u.x, v.x, c[2 * j], s[2 * j]);
                turn(u.y, v.y, c[2 * j + 1], s[2 * j + 1]);
            } else {
                turn(u.x, u.y, c[j], s[j]);
                turn(v.x, v.y, c[P / 2 + j], s[P / 2 + j]);
            }
            x.w[j] = word_of(u.x, u.y, T());
            y.w[j] = word_of(v.x, v.y, T());
        }
    }
}

// EVEN: a head's chunks divide 32, so that a lane keeps its chunk from head to head.
template <typename T, int P, bool HALF, bool PAGED, bool EVEN>
__global__ void __launch_bounds__(32 * ROT_WARPS, 6) rotary_kernel(const __grid_constant__ RotArgs a) {
    extern __shared__ __align__(16) float2 turns[];   // [warps][pairs] cos and sin, times the magnitude
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long w = (long long)blockIdx.x * ROT_WARPS + warp;
    const int t = (int)(w / a.parts), part = (int)(w % a.parts);
    if (t >= a.tokens) return;
    long long pos = 0;
    size_t slot = 0;      // of the token in its page, in rows of a head
    bool kept = true;     // the token has a place in the cache
    if (PAGED) {
        // the row whose new tokens t is among: as many rows end at or before it
        int row = t;
        if (a.cache.starts) {
            row = 0;
            for (int r = 0; r < a.cache.rows; r += 32) row += __popc(__ballot_sync(0xffffffffu, r + lane < a.cache.rows && a.cache.starts[r + lane + 1] <= t));
        }
        if (row >= a.cache.rows) return;  // behind the last row: left as it was
        const PagedRow r = paged_row(a.cache, row, part == 0 && lane == 0 ? a.status : nullptr);
        if (t < r.first || t >= r.first + r.count) return;
        pos = r.len - (r.first + r.count) + t;
        kept = pos >= 0;
        if (kept) {
            const int id = __ldg(a.cache.table + row * a.cache.table_stride + (pos >> a.cache.page_shift));
            kept = (unsigned)id < (unsigned)a.cache.pages;
            slot = ((size_t)id * a.cache.kv_heads << a.cache.page_shift) + (size_t)(pos & ((1 << a.cache.page_shift) - 1));
        }
        if (!kept && lane == 0) paged_bad(a.status);
    } else {
        pos = a.pos64 ? ((const long long *)a.pos)[t] : ((const int *)a.pos)[t];
    }
    const int turned = a.pairs / P;          // chunks that turn
    float2 *cs = turns + warp * a.pairs;
    for (int j = lane; j < a.pairs; j += 32) {   // a pair a lane
        float2 v;
        turn_cos_sin((unsigned long long)pos * turns_per_position(__ldg(a.freq + j)), a.mag, v.x, v.y);
        cs[j] = v;
    }
    __syncwarp();
    float c[P], s[P];
    int known = -1;                          // the chunk whose angles c and s are
    auto angles = [&](int chunk) {
        if (chunk == known || chunk >= turned) return;
        known = chunk;
#pragma unroll
        for (int j = 0; j < P; ++j) { const float2 v = cs[chunk * P + j]; c[j] = v.x; s[j] = v.y; }
    };
    auto start = [&](int chunk) { return chunk < turned ? (HALF ? chunk * P : chunk * 2 * P) : 2 * a.pairs + (chunk - turned) * 2 * P; };
    // Heads [h0, h1) of a tensor whose first lies at src, and goes to dst: `gap` elements from a head to the next there.
    const int step = EVEN ? 32 / a.chunks : 0, sub = EVEN ? lane / a.chunks : 0, chunk0 = EVEN ? lane % a.chunks : 0;
    if (EVEN) angles(chunk0);
    auto heads = [&](const T *src, T *dst, size_t gap, int h0, int h1, bool turns) {
        if (EVEN) {
            const bool turn = turns && chunk0 < turned;
            const int at = start(chunk0), other = HALF && chunk0 < turned ? a.pairs : P;
            for (int h = h0 + sub; h < h1; h += step * ROT_BATCH) {
                Vec<T, P> x[ROT_BATCH], y[ROT_BATCH];
                const T *from = src + (h * a.dim + at);
                T *to = dst + (size_t)h * gap + at;
#pragma unroll
                for (int b = 0; b < ROT_BATCH; ++b)
                    if (h + b * step < h1) {
                        x[b].load(from + b * step * a.dim);
                        y[b].load(from + b * step * a.dim + other);
                    }
#pragma unroll
                for (int b = 0; b < ROT_BATCH; ++b)
                    if (h + b * step < h1) {
                        if (turn) rot_turn<T, P, HALF>(x[b], y[b], c, s);
                        x[b].store(to + (size_t)(b * step) * gap);
                        y[b].store(to + (size_t)(b * step) * gap + other);
                    }
            }
        } else {
            for (int i = h0 * a.chunks + lane; i < h1 * a.chunks; i += 32) {
                const int h = i / a.chunks, chunk = i - h * a.chunks, at = start(chunk), other = HALF && chunk < turned ? a.pairs : P;
                Vec<T, P> x, y;
                x.load(src + (h * a.dim + at));
                y.load(src + (h * a.dim + at + other));
                if (turns && chunk < turned) {
                    angles(chunk);
                    rot_turn<T, P, HALF>(x, y, c, s);
                }
                x.store(dst + (size_t)h * gap + at);
                y.store(dst + (size_t)h * gap + at + other);
            }
        }
    };
    // the warp's share of the heads of q, k and v, one after the other
    const int h0 = part * a.per_warp, h1 = h0 + a.per_warp, dim = a.dim;
    auto share = [&](int first, int count, int &lo, int &hi) { lo = min(max(h0 - first, 0), count); hi = min(max(h1 - first, 0), count); };
    int lo, hi;
    share(0, a.heads, lo, hi);
    if (lo < hi) heads((const T *)a.q + (size_t)t * a.q_stride, (T *)a.qo + (size_t)t * a.qo_stride, dim, lo, hi, true);
    if (!kept) return;
    share(a.heads, a.kv_heads, lo, hi);
    if (lo < hi) {
        if (PAGED) heads((const T *)a.k + (size_t)t * a.k_stride, (T *)a.kp + slot * dim, (size_t)dim << a.cache.page_shift, lo, hi, true);
        else heads((const T *)a.k + (size_t)t * a.k_stride, (T *)a.ko + (size_t)t * a.ko_stride, dim, lo, hi, true);
    }
    if (!PAGED) return;
    share(a.heads + a.kv_heads, a.kv_heads, lo, hi);
    if (lo < hi) heads((const T *)a.v + (size_t)t * a.v_stride, (T *)a.vp + slot * dim, (size_t)dim << a.cache.page_shift, lo, hi, false);
}

template <typename T, int P, bool EVEN>
int launch_rotary(const RotArgs &a, bool half, bool paged, cudaStream_t s) {
    const dim3 grid((unsigned)(((long long)a.tokens * a.parts + ROT_WARPS - 1) / ROT_WARPS));
    const size_t smem = (size_t)ROT_WARPS * a.pairs * sizeof(float2);
    if (paged) (half ? rotary_kernel<T, P, true, true, EVEN> : rotary_kernel<T, P, false, true, EVEN>)<<<grid, 32 * ROT_WARPS, smem, s>>>(a);
    else (half ? rotary_kernel<T, P, true, false, EVEN> : rotary_kernel<T, P, false, false, EVEN>)<<<grid, 32 * ROT_WARPS, smem, s>>>(a);
    AB2_LAUNCH_CHECK();
    return AB2_OK;
}

// Chunks of P pairs that make loads of 16 bytes where every piece starts on such a boundary, else of 4 pairs, else single pairs.
int rotary_go(RotArgs a, bool half, bool paged, ab2_dtype dtype, cudaStream_t s) {
    const int rest = a.dim - 2 * a.pairs;
    uintptr_t where = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.qo | (uintptr_t)a.ko | (uintptr_t)a.kp | (uintptr_t)a.vp;
    const size_t esize = dtype_size(dtype);
    const long long steps = a.q_stride | a.k_stride | a.v_stride | a.qo_stride | a.ko_stride | a.dim;
    int P = dtype == AB2_F32 ? 4 : 8;
    while (P > 1 && (a.pairs % P || rest % (2 * P) || steps % P || where % std::min<size_t>(16, P * esize))) P = P == 8 ? 4 : 1;
    a.chunks = a.dim / (2 * P);
    // A warp has all heads of a token where there are tokens enough for some warps on every scheduler, else fewer: a load a lane at least.
    const int vheads = a.heads + a.kv_heads * (paged ? 2 : 1), want = std::max(1, device_sm_count() * 16 / std::max(1, a.tokens)), least = std::max(1, 32 / a.chunks);
    a.per_warp = std::max(least, (vheads + want - 1) / want);
    a.parts = (vheads + a.per_warp - 1) / a.per_warp;
    AB2_REQUIRE(((long long)a.tokens * a.parts + ROT_WARPS - 1) / ROT_WARPS < (1ll << 31), AB2_ERR_BAD_SHAPE, "%d tokens of %d heads are more than one launch takes", a.tokens, a.heads);
    const bool even = 32 % a.chunks == 0;
#define AB2_ROTARY(T)                                                                                                                                   \
    (sizeof(T) == 2 && P == 8 ? (even ? launch_rotary<T, 16 / sizeof(T), true>(a, half, paged, s) : launch_rotary<T, 16 / sizeof(T), false>(a, half, paged, s))                                     \
     : P == 4 ? (even ? launch_rotary<T, 4, true>(a, half, paged, s) : launch_rotary<T, 4, false>(a, half, paged, s)) : launch_rotary<T, 1, false>(a, half, paged, s))
    switch (dtype) {
    case AB2_F32: return AB2_ROTARY(float);
    case AB2_F16: return AB2_ROTARY(__half);
    default: return AB2_ROTARY(__nv_bfloat16);
    }
#undef AB2_ROTARY
}

int check_layout(int layout, int dim, int rot, const double *freq) {
    AB2_REQUIRE(layout == AB2_ROTARY_HALF || layout == AB2_ROTARY_INTERLEAVED, AB2_ERR_BAD_ARG, "unknown rotary layout %d", layout);
    AB2_REQUIRE(dim > 0 && dim % 2 == 0 && rot >= 0 && rot % 2 == 0 && rot <= dim, AB2_ERR_BAD_SHAPE, "rotary positions turn an even number of an even head's dimensions, got %d of %d", rot, dim);
    AB2_REQUIRE(rot <= 2048, AB2_ERR_UNSUPPORTED, "up to 2048 dimensions of a head are rotated, got %d", rot);
    AB2_REQUIRE(rot == 0 || freq, AB2_ERR_BAD_ARG, "null frequencies");
    return AB2_OK;
}

// Elements, strides and pointers on boundaries of their own type.
bool on_elements(std::initializer_list<const void *> ps, ab2_dtype dtype) {
    uintptr_t all = 0;
    for (const void *p : ps) all |= (uintptr_t)p;
    return all % dtype_size(dtype) == 0;
}

}  // namespace

int paged_check(const ab2_paged *c, ab2_dtype dtype) {
    AB2_REQUIRE(c, AB2_ERR_BAD_ARG, "null paged cache");
    AB2_REQUIRE(c->k_pages && c->v_pages && c->table && c->lens, AB2_ERR_BAD_ARG, "null buffer of a paged cache");
    AB2_REQUIRE(dtype == AB2_F32 || dtype == AB2_BF16, AB2_ERR_BAD_DTYPE, "paged caches hold f32 or bf16, not dtype %d", (int)dtype);
    AB2_REQUIRE(c->head_dim == 64 || c->head_dim == 128, AB2_ERR_UNSUPPORTED, "paged caches have heads of 64 or 128, not %d", c->head_dim);
    AB2_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && !(c->page_size & (c->page_size - 1)), AB2_ERR_UNSUPPORTED, "a page holds 16, 32, 64, 128 or 256 tokens, not %d", c->page_size);
    AB2_REQUIRE(c->pages > 0 && c->kv_heads > 0 && c->rows > 0 && c->tokens >= 0 && c->table_width > 0, AB2_ERR_BAD_SHAPE,
                "paged cache of %d pages, %d heads, %d rows of %d pages, %d tokens", c->pages, c->kv_heads, c->rows, c->table_width, c->tokens);
    AB2_REQUIRE(c->table_stride >= c->table_width, AB2_ERR_BAD_SHAPE, "table rows of %d pages lie %lld apart", c->table_width, c->table_stride);
    AB2_REQUIRE((long long)c->table_width * c->page_size <= (1ll << 30) && (long long)c->kv_heads * c->page_size < (1ll << 31) && (long long)c->kv_heads * c->pages < (1ll << 31), AB2_ERR_BAD_SHAPE, "rows of more than 2^30 tokens, or 2^31 pages and heads");
    AB2_REQUIRE(c->starts || c->tokens == c->rows, AB2_ERR_BAD_SHAPE, "%d tokens for %d rows of one token each", c->tokens, c->rows);
    AB2_REQUIRE((((uintptr_t)c->k_pages | (uintptr_t)c->v_pages) & 15) == 0, AB2_ERR_BAD_ALIGN, "pages must be 16-byte aligned");
    return AB2_OK;
}
PagedView paged_view(const ab2_paged *c) {
    PagedView v;
    v.table = c->table; v.lens = c->lens; v.starts = c->starts;
    v.rows = c->rows; v.tokens = c->tokens; v.width = c->table_width; v.table_stride = c->table_stride; v.pages = c->pages; v.kv_heads = c->kv_heads;
    v.page_shift = __builtin_ctz(c->page_size);
    return v;
}

// What the appends look their arguments over for; `page_es`: bytes of an element of the pages.
int append_check(const ab2_paged *cache, long long page_es, const void *k_dev, long long k_stride, const void *v_dev, long long v_stride, const void *q_dev, long long q_stride, int heads, void *q_out_dev,
                 long long q_out_stride, const double *frequencies_dev, int rot_dims, int layout, ab2_dtype dtype) {
    int rc = paged_check(cache, dtype);
    if (rc != AB2_OK) return rc;
    rc = check_layout(layout, cache->head_dim, rot_dims, frequencies_dev);
    if (rc != AB2_OK) return rc;
    AB2_REQUIRE(heads >= 0, AB2_ERR_BAD_SHAPE, "%d heads", heads);
    if (cache->tokens == 0) return AB2_OK;
    AB2_REQUIRE(k_dev && v_dev && (heads == 0 || (q_dev && q_out_dev)), AB2_ERR_BAD_ARG, "null argument");
    AB2_REQUIRE(on_elements({k_dev, v_dev, heads ? q_dev : nullptr, heads ? q_out_dev : nullptr}, dtype), AB2_ERR_BAD_ALIGN, "tensors must lie on their elements");
    const long long row = (long long)heads * cache->head_dim, krow = (long long)cache->kv_heads * cache->head_dim;
    AB2_REQUIRE((heads + 2ll * cache->kv_heads) * cache->head_dim < (1ll << 30), AB2_ERR_BAD_SHAPE, "%d and %d heads of %d are too many", heads, cache->kv_heads, cache->head_dim);
    AB2_REQUIRE(k_stride >= krow && v_stride >= krow && (heads == 0 || (q_stride >= row && q_out_stride >= row)), AB2_ERR_BAD_SHAPE, "a token's heads lie one after the other, and tokens do not overlap");
    const long long es = (long long)dtype_size(dtype), pool = (long long)cache->pages * cache->page_size * krow * page_es;
    const RowsAt qo_at = {heads ? q_out_dev : nullptr, row * es, q_out_stride * es, cache->tokens}, kp_at = {cache->k_pages, pool, pool, 1}, vp_at = {cache->v_pages, pool, pool, 1};
    AB2_REQUIRE(in_place_or_apart(qo_at, {heads ? q_dev : nullptr, row * es, q_stride * es, cache->tokens}) && !rows_meet(qo_at, {k_dev, krow * es, k_stride * es, cache->tokens}) &&
                    !rows_meet(qo_at, {v_dev, krow * es, v_stride * es, cache->tokens}),
                AB2_ERR_BAD_ARG, "the rotated queries take the queries' place, or lie apart from queries, keys and values");
    AB2_REQUIRE(!rows_meet(kp_at, vp_at) && !rows_meet(qo_at, kp_at) && !rows_meet(qo_at, vp_at), AB2_ERR_BAD_ARG, "pages of keys, pages of values and the rotated queries lie apart");
    return AB2_OK;
}

}  // namespace ab2

AB2_API int ab2_rotary_apply(const void *q_dev, long long q_stride, int heads, const void *k_dev, long long k_stride, int kv_heads, int head_dim,
                             const void *positions_dev, int positions_64, int tokens, const double *frequencies_dev, int rot_dims, int layout, float magnitude,
                             void *q_out_dev, long long q_out_stride, void *k_out_dev, long long k_out_stride, ab2_dtype dtype, ab2_stream stream) {
    AB2_REQUIRE(dtype == AB2_F32 || dtype == AB2_F16 || dtype == AB2_BF16, AB2_ERR_BAD_DTYPE, "unsupported dtype %d", (int)dtype);
    AB2_REQUIRE(heads >= 0 && kv_heads >= 0 && heads + (long long)kv_heads > 0 && tokens >= 0, AB2_ERR_BAD_SHAPE, "%d tokens of %d and %d heads", tokens, heads, kv_heads);
    int rc = check_layout(layout, head_dim, rot_dims, frequencies_dev);
    if (rc != AB2_OK) return rc;
    if (tokens == 0) return AB2_OK;
    AB2_REQUIRE((heads == 0 || (q_dev && q_out_dev)) && (kv_heads == 0 || (k_dev && k_out_dev)) && positions_dev, AB2_ERR_BAD_ARG, "null argument");
    AB2_REQUIRE(on_elements({heads ? q_dev : nullptr, heads ? q_out_dev : nullptr, kv_heads ? k_dev : nullptr, kv_heads ? k_out_dev : nullptr}, dtype), AB2_ERR_BAD_ALIGN, "tensors must lie on their elements");
    const long long row = (long long)heads * head_dim, krow = (long long)kv_heads * head_dim;
    AB2_REQUIRE((long long)(heads + kv_heads) * head_dim < (1ll << 30), AB2_ERR_BAD_SHAPE, "%d and %d heads of %d are too many", heads, kv_heads, head_dim);
    AB2_REQUIRE((heads == 0 || (q_stride >= row && q_out_stride >= row)) && (kv_heads == 0 || (k_stride >= krow && k_out_stride >= krow)), AB2_ERR_BAD_SHAPE, "a token's heads lie one after the other, and tokens do not overlap");
    const long long es = (long long)dtype_size(dtype);
    const RowsAt q_at = {heads ? q_dev : nullptr, row * es, q_stride * es, tokens}, k_at = {kv_heads ? k_dev : nullptr, krow * es, k_stride * es, tokens};
    const RowsAt qo_at = {heads ? q_out_dev : nullptr, row * es, q_out_stride * es, tokens}, ko_at = {kv_heads ? k_out_dev : nullptr, krow * es, k_out_stride * es, tokens};
    AB2_REQUIRE(in_place_or_apart(qo_at, q_at) && in_place_or_apart(ko_at, k_at) && !rows_meet(qo_at, k_at) && !rows_meet(ko_at, q_at) && !rows_meet(qo_at, ko_at), AB2_ERR_BAD_ARG,
                "an output takes its input's place, or lies apart from both inputs and the other output");
    RotArgs a = {};
    if (heads) { a.q = q_dev; a.qo = q_out_dev; a.q_stride = q_stride; a.qo_stride = q_out_stride; }
    if (kv_heads) { a.k = k_dev; a.ko = k_out_dev; a.k_stride = k_stride; a.ko_stride = k_out_stride; }
    a.heads = heads; a.kv_heads = kv_heads; a.dim = head_dim; a.pairs = rot_dims / 2; a.tokens = tokens;
    a.pos = positions_dev; a.pos64 = positions_64; a.freq = frequencies_dev; a.mag = magnitude;
    return rotary_go(a, layout == AB2_ROTARY_HALF, false, dtype, (cudaStream_t)stream);
}

AB2_API int ab2_paged_append(const ab2_paged *cache, const void *k_dev, long long k_stride, const void *v_dev, long long v_stride, const void *q_dev, long long q_stride,
                             int heads, void *q_out_dev, long long q_out_stride, const double *frequencies_dev, int rot_dims, int layout, float magnitude, ab2_dtype dtype, ab2_stream stream) {
    int rc = append_check(cache, (long long)dtype_size(dtype), k_dev, k_stride, v_dev, v_stride, q_dev, q_stride, heads, q_out_dev, q_out_stride, frequencies_dev, rot_dims, layout, dtype);
    if (rc != AB2_OK || cache->tokens == 0) return rc;
    RotArgs a = {};
    a.k = k_dev; a.v = v_dev; a.k_stride = k_stride; a.v_stride = v_stride;
    if (heads) { a.q = q_dev; a.qo = q_out_dev; a.q_stride = q_stride; a.qo_stride = q_out_stride; }
    a.heads = heads; a.kv_heads = cache->kv_heads; a.dim = cache->head_dim; a.pairs = rot_dims / 2; a.tokens = cache->tokens;
    a.freq = frequencies_dev; a.mag = magnitude;
    a.cache = paged_view(cache); a.kp = cache->k_pages; a.vp = cache->v_pages;
    rc = device_status_word(&a.status);
    if (rc != AB2_OK) return rc;
    return rotary_go(a, layout == AB2_ROTARY_HALF, true, dtype, (cudaStream_t)stream);
}
