// Rules of a sampler on the logits of a batch: with c the times token v occurs in the row's history,
//
//   z <- z / rho if z > 0 else z rho       where c > 0        (repetition)
//   z <- z - presence - frequency c        where c > 0
//   z <- z + bias_v                        where v is biased
//   z <- -inf                              where the row's mask has v's bit 0
//
// each step in f32, the result rounded to the logits' type.  A CTA has a slice of a row's vocabulary: it counts the history's tokens of its slice in shared memory
// (integer additions, whose order changes nothing) and notes which entry of the bias list is each token's last, with a bit for each token that says whether there is
// anything to look up for it.  Then it passes over the slice twice: 16 bytes a load, storing logits as they are and -inf where the mask says so; and again over the
// words of those bits, changing the few tokens that the history or the biases touch.  Every CTA of a row reads the row's history, from L2 after the first.  Bound
// by HBM for large batches, by the launch, the clearing of the counts and the history's latency for small ones.
#include <algorithm>

#include "common.cuh"

using namespace ab2;

namespace ab2 {
int device_sm_count();
namespace {

constexpr int LG_THREADS = 256, LG_CTAS = 5;
// Tokens a CTA at most: its loads of logits are all in flight, a token at a time fewer, and a table each takes the room of two.
template <int V, bool PACKED> constexpr int LG_SLICE = (V == 1 ? 2048 : 8192) / (PACKED ? 1 : 2);
constexpr int LG_COUNT = 20;                       // bits of a table's word for the count, the others are the bias list's entry

struct LogitArgs {
    const void *logits;
    void *out;
    long long stride;
    int vocab, slice;
    const int *history, *lengths;
    long long history_stride;
    int history_width;
    const float *rules;
    const int *bias_ids;
    const float *bias_values;
    int biases;
    const uint32_t *allowed;
    int words;
};

template <typename T> __device__ __forceinline__ uint32_t lowest_bits();   // of -inf
template <> __device__ __forceinline__ uint32_t lowest_bits<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ uint32_t lowest_bits<__half>() { return 0xfc00u; }
template <> __device__ __forceinline__ uint32_t lowest_bits<__nv_bfloat16>() { return 0xff80u; }

// V elements a load.  PACKED: a token's count and its entry of the bias list, + 1, share a word (fewer than 2^20 and 2^12 of them), else a table each.
template <typename T, int V, bool PACKED>
__global__ void __launch_bounds__(LG_THREADS, LG_CTAS) adjust_logits_kernel(const __grid_constant__ LogitArgs a) {
    // [slice / 32] which tokens the history or the biases touch, [slice] counts, not PACKED [slice] entries
    extern __shared__ __align__(16) uint32_t touched[];
    int *counts = (int *)touched + a.slice / 32, *entry = counts + (PACKED ? 0 : a.slice);
    constexpr int ENTRY = PACKED ? LG_COUNT : 0;   // where a word's entry begins
    const int row = blockIdx.y, first = blockIdx.x * a.slice, n = min(a.slice, a.vocab - first);
    const T *in = (const T *)a.logits + row * a.stride + first;
    const uint32_t *mask = a.allowed ? a.allowed + (size_t)row * a.words + (first >> 5) : nullptr;
    constexpr int LOADS = LG_SLICE<V, PACKED> / (LG_THREADS * V);   // the slice's logits are on their way while the tables are made
    alignas(16) T e[LOADS][V];
    uint32_t bits[LOADS];
#pragma unroll
    for (int b = 0; b < LOADS; ++b) {
        const int i = (threadIdx.x + b * LG_THREADS) * V;
        if (i >= n) continue;
        if constexpr (V > 1) *reinterpret_cast<uint4 *>(e[b]) = *reinterpret_cast<const uint4 *>(in + i);
        else e[b][0] = in[i];
        bits[b] = mask ? mask[i >> 5] >> (i & 31) : 0xffffffffu;
    }
    const int tables = a.slice / 32 + (a.history || a.biases ? (PACKED ? 1 : 2) * a.slice : 0);
    for (int i = threadIdx.x * 4; i < tables; i += LG_THREADS * 4) *reinterpret_cast<uint4 *>(touched + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    for (int i = threadIdx.x; i < a.biases; i += LG_THREADS) {
        const int v = a.bias_ids[(size_t)row * a.biases + i] - first;
        if ((unsigned)v >= (unsigned)n) continue;
        atomicMax((unsigned *)entry + v, (unsigned)(i + 1) << ENTRY);
        atomicOr(touched + (v >> 5), 1u << (v & 31));
    }
    if (PACKED && a.biases) __syncthreads();   // the counts come below the entries
    float rho = 1.f, presence = 0.f, frequency = 0.f, inverse = 1.f, half0 = 1.f, half1 = 1.f;
    if (a.history) {
        rho = a.rules[3 * row]; presence = a.rules[3 * row + 1]; frequency = a.rules[3 * row + 2];
        // A quotient of f32 logits is rounded once.  Logits of 16 bits are multiplied by the reciprocal of the penalty's significand and by its power of two in halves,
        // which no penalty takes out of range; the second rounding (2^-24) is nothing beside theirs.  Made here, while the history is on its way (64 x 128256 in bf16 16.7 us;
        // behind it 18.2, with a division 18.4).
        if constexpr (sizeof(T) == 2) {
            int power;
            inverse = 1.f / frexpf(rho, &power);
            half0 = ldexpf(1.f, -power >> 1);
            half1 = ldexpf(1.f, -power - (-power >> 1));
        }
        const int *h = a.history + row * a.history_stride;
        const int len = min(a.lengths ? a.lengths[row] : a.history_width, a.history_width);
        auto count = [&](int v) {
            if ((unsigned)v >= (unsigned)n) return;
            atomicAdd(counts + v, 1);
            atomicOr(touched + (v >> 5), 1u << (v & 31));
        };
        int done = 0;
        if (((uintptr_t)h & 15) == 0) {   // four ids a load, four loads in flight
            done = max(len, 0) & ~3;
            for (int i = threadIdx.x * 4; i < done; i += LG_THREADS * 16) {
                int4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = i + u * LG_THREADS * 4 < done ? *reinterpret_cast<const int4 *>(h + i + u * LG_THREADS * 4) : make_int4(-1, -1, -1, -1);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (i + u * LG_THREADS * 4 >= done) continue;
                    count(v[u].x - first); count(v[u].y - first); count(v[u].z - first); count(v[u].w - first);
                }
            }
        }
        for (int i = done + threadIdx.x; i < len; i += LG_THREADS) count(h[i] - first);
    }
    // the slice as it is, and -inf where the mask says so: most tokens are in no history and no list
    T *out = (T *)a.out + (size_t)row * a.vocab + first;
#pragma unroll
    for (int b = 0; b < LOADS; ++b) {
        const int i = (threadIdx.x + b * LG_THREADS) * V;
        if (i >= n) continue;
        if constexpr (V > 1) {
            uint32_t q[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                q[m] = reinterpret_cast<const uint32_t *>(e[b])[m];
                if constexpr (sizeof(T) == 4) {
                    if (!((bits[b] >> m) & 1)) q[m] = lowest_bits<T>();
                } else {
                    const uint32_t keep = ((bits[b] >> (2 * m)) & 1 ? 0xffffu : 0u) | ((bits[b] >> (2 * m + 1)) & 1 ? 0xffff0000u : 0u);
                    q[m] = (q[m] & keep) | (lowest_bits<T>() * 0x10001u & ~keep);
                }
            }
            *reinterpret_cast<uint4 *>(out + i) = make_uint4(q[0], q[1], q[2], q[3]);
        } else {
            out[i] = bits[b] & 1 ? e[b][0] : from_f32<T>(-INFINITY);
        }
    }
    __syncthreads();   // the tables are whole, and the tokens stored
    // then the tokens that are in one, where the mask allows them (what has been stored is their logit): a word of 32 tokens a thread
    const float *bias = a.bias_values + (size_t)row * a.biases;
    auto divided = [&](float z) { return sizeof(T) == 4 ? z / rho : z * half0 * inverse * half1; };
    for (int w = threadIdx.x; w * 32 < n; w += LG_THREADS)
        for (uint32_t left = touched[w] & (mask ? mask[w] : 0xffffffffu); left; left &= left - 1) {
            const int i = w * 32 + __ffs(left) - 1, word = counts[i], count = PACKED ? word & ((1 << LG_COUNT) - 1) : word;
            const unsigned k = (unsigned)entry[i] >> ENTRY;
            float z = to_f32(out[i]);
            if (count > 0) z = (z > 0.f ? divided(z) : z * rho) - (presence + frequency * (float)count);
            if (k) z += bias[k - 1];
            out[i] = from_f32<T>(z);
        }
}

template <typename T, int V>
int launch_adjust(LogitArgs a, int rows, cudaStream_t s) {
    // Slices of 8192 tokens, smaller ones where those are fewer than two CTAs an SM; 512 at least.  64 x 128256 bf16 behind 4096 tokens take 16.6 us
    // (33 MB: 5.3 us of HBM); what bounds them is every slice's walk through its row's history and the look-ups of what that touches.
    const bool packed = a.history_width < (1 << LG_COUNT) && a.biases < (1 << (32 - LG_COUNT)) - 1;
    a.slice = packed ? LG_SLICE<V, true> : LG_SLICE<V, false>;
    while (a.slice > 512 && (long long)rows * ((a.vocab + a.slice - 1) / a.slice) < 2 * device_sm_count()) a.slice /= 2;
    const dim3 grid((a.vocab + a.slice - 1) / a.slice, rows);
    const size_t smem = (size_t)a.slice * 4 * (a.history || a.biases ? (packed ? 1 : 2) : 0) + a.slice / 8;
    if (packed) adjust_logits_kernel<T, V, true><<<grid, LG_THREADS, smem, s>>>(a);
    else adjust_logits_kernel<T, V, false><<<grid, LG_THREADS, smem, s>>>(a);
    AB2_LAUNCH_CHECK();
    return AB2_OK;
}
template <typename T>
int launch_adjust(const LogitArgs &a, int rows, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool wide = a.vocab % V == 0 && a.stride % V == 0 && (((uintptr_t)a.logits | (uintptr_t)a.out) & 15) == 0;
    return wide ? launch_adjust<T, V>(a, rows, s) : launch_adjust<T, 1>(a, rows, s);
}

}  // namespace
}  // namespace ab2

AB2_API int ab2_adjust_logits(const void *logits_dev, long long stride, int rows, int vocab, const int *history_dev, long long history_stride, int history_width,
                              const int *lengths_dev, const float *rules_dev, const int *bias_ids_dev, const float *bias_values_dev, int biases, const uint32_t *allowed_dev,
                              void *out_dev, ab2_dtype dtype, ab2_stream stream) {
    AB2_REQUIRE(rows >= 0 && vocab > 0, AB2_ERR_BAD_SHAPE, "logits of %d rows, %d tokens", rows, vocab);
    AB2_REQUIRE(rows <= 65535, AB2_ERR_BAD_SHAPE, "%d rows are more than the 65535 of a launch", rows);
    AB2_REQUIRE(dtype == AB2_F32 || dtype == AB2_F16 || dtype == AB2_BF16, AB2_ERR_BAD_DTYPE, "unsupported dtype %d", (int)dtype);
    if (rows == 0) return AB2_OK;
    AB2_REQUIRE(logits_dev && out_dev, AB2_ERR_BAD_ARG, "null argument");
    AB2_REQUIRE(stride >= vocab, AB2_ERR_BAD_SHAPE, "rows of %d logits lie %lld apart", vocab, stride);
    AB2_REQUIRE((((uintptr_t)logits_dev | (uintptr_t)out_dev) & (dtype_size(dtype) - 1)) == 0, AB2_ERR_BAD_ALIGN, "logits must lie on their elements");
    AB2_REQUIRE(history_width >= 0 && biases >= 0, AB2_ERR_BAD_SHAPE, "history of %d, %d biases", history_width, biases);
    AB2_REQUIRE(history_width == 0 || (history_dev && rules_dev && history_stride >= history_width), AB2_ERR_BAD_ARG, "a history needs its tokens, rows that do not overlap, and rules");
    AB2_REQUIRE(biases == 0 || (bias_ids_dev && bias_values_dev), AB2_ERR_BAD_ARG, "null bias list");
    const long long es = (long long)dtype_size(dtype);
    AB2_REQUIRE(in_place_or_apart({out_dev, vocab * es, vocab * es, rows}, {logits_dev, vocab * es, stride * es, rows}), AB2_ERR_BAD_ARG, "the result takes the logits' place, or lies apart from them");
    LogitArgs a = {};
    a.logits = logits_dev; a.out = out_dev; a.stride = stride; a.vocab = vocab;
    if (history_width > 0) { a.history = history_dev; a.history_stride = history_stride; a.history_width = history_width; a.lengths = lengths_dev; a.rules = rules_dev; }
    a.bias_ids = bias_ids_dev; a.bias_values = bias_values_dev; a.biases = biases;
    a.allowed = allowed_dev; a.words = (vocab + 31) / 32;
    switch (dtype) {
    case AB2_F32: return launch_adjust<float>(a, rows, (cudaStream_t)stream);
    case AB2_F16: return launch_adjust<__half>(a, rows, (cudaStream_t)stream);
    default: return launch_adjust<__nv_bfloat16>(a, rows, (cudaStream_t)stream);
    }
}
