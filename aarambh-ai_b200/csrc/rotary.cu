// Rotary positions of a batch of tokens, alone or together with the append of their keys and values to a paged cache.
//
//   turned pair i of a head at position p = m R(p f_i) (x_i, y_i),   R a rotation, f_i radians a position, m a magnitude
//
// Pairs are (i, i + n) with the half layout and (2i, 2i + 1) with the interleaved one, n = rot / 2 of them; the dimensions from rot on pass
// as they are.  One pass over q and k (and v, which is copied into its pages): bound by HBM from some hundred tokens on, by the launch
// below.  A warp has one token (or a part of its heads where tokens are few): its lanes turn the token's angles once, into shared memory,
// and then take items (head, P pairs) of it; where a head's chunks divide 32 a lane keeps its pairs from head to head.
#include <algorithm>

#include "paged.cuh"

using namespace ab2;

namespace ab2 {
namespace {

constexpr int ROT_WARPS = 4, ROT_BATCH = 2;  // items of a lane in flight

struct RotArgs {
    const void *q, *k, *v;
    void *qo, *ko;
    long long q_stride, k_stride, v_stride, qo_stride, ko_stride;  // elements from a token to the next
    int heads, kv_heads, dim, pairs, tokens, chunks;               // chunks of P pairs a head has, the unturned dimensions among them
    int per_warp, parts;                                           // items (head, chunk) of a warp, warps of a token
    const void *pos;
    int pos64;
    const double *freq;
    float mag;
    PagedView cache;  // with PAGED: k and v go there, and positions are those in their rows
    void *kp, *vp;
    int *status;
};

// E elements in one load or store (E * sizeof(T) is 2, 4, 8, 16 or 32 bytes)
template <typename T, int E> struct Vec {
    static constexpr int BYTES = E * (int)sizeof(T), WORD = BYTES >= 16 ? 16 : BYTES;
    T e[E];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < BYTES; i += WORD) {
            if constexpr (WORD == 16) *reinterpret_cast<uint4 *>((char *)e + i) = *reinterpret_cast<const uint4 *>((const char *)p + i);
            else if constexpr (WORD == 8) *reinterpret_cast<uint2 *>((char *)e + i) = *reinterpret_cast<const uint2 *>((const char *)p + i);
            else if constexpr (WORD == 4) *reinterpret_cast<uint32_t *>((char *)e + i) = *reinterpret_cast<const uint32_t *>((const char *)p + i);
            else *reinterpret_cast<uint16_t *>((char *)e + i) = *reinterpret_cast<const uint16_t *>((const char *)p + i);
        }
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < BYTES; i += WORD) {
            if constexpr (WORD == 16) *reinterpret_cast<uint4 *>((char *)p + i) = *reinterpret_cast<const uint4 *>((const char *)e + i);
            else if constexpr (WORD == 8) *reinterpret_cast<uint2 *>((char *)p + i) = *reinterpret_cast<const uint2 *>((const char *)e + i);
            else if constexpr (WORD == 4) *reinterpret_cast<uint32_t *>((char *)p + i) = *reinterpret_cast<const uint32_t *>((const char *)e + i);
            else *reinterpret_cast<uint16_t *>((char *)p + i) = *reinterpret_cast<const uint16_t *>((const char *)e + i);
        }
    }
};

// Where an item (a head's chunk) lies: its first P elements, and the others `gap` further.
template <typename T> struct RotItem {
    const T *src;
    T *dst;
    int gap, chunk;   // from `turned` on: passes as it is
    bool kept;
};

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
    const int lo = part * a.per_warp, vheads = a.heads + a.kv_heads * (PAGED ? 2 : 1), hi = min(lo + a.per_warp, vheads * a.chunks);
    auto item = [&](int h, int chunk) {
        RotItem<T> it;
        const int at = chunk < turned ? (HALF ? chunk * P : chunk * 2 * P) : 2 * a.pairs + (chunk - turned) * 2 * P;
        it.gap = HALF && chunk < turned ? a.pairs : P;
        it.chunk = chunk;
        it.kept = true;
        if (h < a.heads) {
            it.src = (const T *)a.q + ((size_t)t * a.q_stride + (size_t)(h * a.dim + at));
            it.dst = (T *)a.qo + ((size_t)t * a.qo_stride + (size_t)(h * a.dim + at));
        } else {
            const int g = h - a.heads;
            const bool value = PAGED && g >= a.kv_heads;
            const int of = (value ? g - a.kv_heads : g) * a.dim + at;
            if (value) it.chunk = turned;
            it.src = (value ? (const T *)a.v + (size_t)t * a.v_stride : (const T *)a.k + (size_t)t * a.k_stride) + of;
            if (PAGED) {
                it.dst = (T *)(value ? a.vp : a.kp) + (slot + ((size_t)(value ? g - a.kv_heads : g) << a.cache.page_shift)) * a.dim + at;
                it.kept = kept;
            } else {
                it.dst = (T *)a.ko + (size_t)t * a.ko_stride + of;
            }
        }
        return it;
    };
    const int step = EVEN ? 32 / a.chunks : 0;
    int head = (lo + lane) / a.chunks;
    const int chunk0 = (lo + lane) % a.chunks;
    float2 *cs = turns + warp * a.pairs;
    float c[P], s[P];
    int known = -1;                          // the chunk whose angles c and s are
    bool first = true;
    for (int i0 = lo + lane; __any_sync(0xffffffffu, i0 < hi); i0 += 32 * ROT_BATCH) {
        RotItem<T> it[ROT_BATCH];
        Vec<T, P> x[ROT_BATCH], y[ROT_BATCH];
#pragma unroll
        for (int b = 0; b < ROT_BATCH; ++b) {
            const int i = i0 + 32 * b;
            it[b] = EVEN ? item(head, chunk0) : item(i / a.chunks, i % a.chunks);
            head += step;
            if (i < hi) {
                x[b].load(it[b].src);
                y[b].load(it[b].src + it[b].gap);
            }
        }
        if (first) {   // while the first items come, a pair a lane
            first = false;
            for (int j = lane; j < a.pairs; j += 32) {
                float2 v;
                turn_cos_sin((unsigned long long)pos * turns_per_position(__ldg(a.freq + j)), a.mag, v.x, v.y);
                cs[j] = v;
            }
            __syncwarp();
        }
#pragma unroll
        for (int b = 0; b < ROT_BATCH; ++b) {
            if (i0 + 32 * b >= hi) continue;
            if (it[b].chunk < turned) {
                if (EVEN ? known < 0 : it[b].chunk != known) {
                    known = it[b].chunk;
#pragma unroll
                    for (int j = 0; j < P; ++j) { const float2 v = cs[known * P + j]; c[j] = v.x; s[j] = v.y; }
                }
                if (HALF) {
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        const float u = to_f32(x[b].e[j]), v = to_f32(y[b].e[j]);
                        x[b].e[j] = from_f32<T>(u * c[j] - v * s[j]);
                        y[b].e[j] = from_f32<T>(u * s[j] + v * c[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < P; ++j) {  // pair j: elements 2j and 2j + 1 of the 2 P of x and y
                        T &e0 = 2 * j < P ? x[b].e[(2 * j) % P] : y[b].e[(2 * j) % P];
                        T &e1 = 2 * j + 1 < P ? x[b].e[(2 * j + 1) % P] : y[b].e[(2 * j + 1) % P];
                        const float u = to_f32(e0), v = to_f32(e1);
                        e0 = from_f32<T>(u * c[j] - v * s[j]);
                        e1 = from_f32<T>(u * s[j] + v * c[j]);
                    }
                }
            }
            if (!it[b].kept) continue;
            x[b].store(it[b].dst);
            y[b].store(it[b].dst + it[b].gap);
        }
    }
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
    // A warp's items: all of a token's where there are tokens enough for some warps on every scheduler, else fewer (a lane has one at least).
    const int items = (a.heads + a.kv_heads * (paged ? 2 : 1)) * a.chunks, want = std::max(1, device_sm_count() * 16 / std::max(1, a.tokens));
    a.parts = std::max(1, std::min(want, (items + 31) / 32));
    a.per_warp = ((items + a.parts - 1) / a.parts + 31) / 32 * 32;
    a.parts = (items + a.per_warp - 1) / a.per_warp;
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
    AB2_REQUIRE((long long)c->table_width * c->page_size < (1ll << 31) && (long long)c->kv_heads * c->page_size < (1ll << 31) && (long long)c->kv_heads * c->pages < (1ll << 31), AB2_ERR_BAD_SHAPE, "rows of 2^31 tokens or more");
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
    RotArgs a = {};
    if (heads) { a.q = q_dev; a.qo = q_out_dev; a.q_stride = q_stride; a.qo_stride = q_out_stride; }
    if (kv_heads) { a.k = k_dev; a.ko = k_out_dev; a.k_stride = k_stride; a.ko_stride = k_out_stride; }
    a.heads = heads; a.kv_heads = kv_heads; a.dim = head_dim; a.pairs = rot_dims / 2; a.tokens = tokens;
    a.pos = positions_dev; a.pos64 = positions_64; a.freq = frequencies_dev; a.mag = magnitude;
    return rotary_go(a, layout == AB2_ROTARY_HALF, false, dtype, (cudaStream_t)stream);
}

AB2_API int ab2_paged_append(const ab2_paged *cache, const void *k_dev, long long k_stride, const void *v_dev, long long v_stride, const void *q_dev, long long q_stride,
                             int heads, void *q_out_dev, long long q_out_stride, const double *frequencies_dev, int rot_dims, int layout, float magnitude, ab2_dtype dtype, ab2_stream stream) {
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
