// Attention of a batch of cached sequences that takes its sequence lengths from device memory, in two forms:
//  - cppinf_tree_attention: T drafted tokens per sequence behind its committed cache rows, each seeing all committed
//    rows and the drafted ones that a mask names (a tree's ancestors);
//  - cppinf_decoder_attention_weights: T causal tokens per sequence, with the attention weight that each cached row
//    received added to an f32 array (what an eviction ranks rows by).
//
// With s_j = q k_j / sqrt(D) over the rows j that a query sees, M their maximum and l = sum exp(s_j - M):
// ctx = sum exp(s_j - M) v_j / l, and row j's weight is the sum over the queries and the query heads of a key-value
// head of exp(s_j - M) / l. Scores, M, l and both sums are f32; exponentials are taken in base 2 with log2(e) / sqrt(D)
// folded into one factor.
//
// One warp per (query, head) walks the visible rows with the running maximum and sum of a softmax, lanes over the head
// dimension; a second kernel, one warp per cached row and key-value head, reads the queries back with each one's M and
// l and adds the row's probabilities up in a fixed order.
#include "common.cuh"
#include "runtime.h"

namespace cppinf::device {
namespace {

constexpr int kMaxNodes = 256;  // drafted tokens of a sequence
constexpr int kMaxGroup = 128;  // query heads of a key-value head

struct CacheAttentionParams {
    const bf16* q;  // [B, T, Hq, D]
    const bf16* k;  // rows of D elements, element strides {batch, row, head}
    const bf16* v;
    int64_t ks[3];
    int64_t vs[3];
    const int64_t* lengths;  // [B] committed rows
    const int64_t* counts;   // [B] valid queries, or null: all T
    const uint8_t* mask;     // tree: [T, T] at mask + b * mask_stride; null: causal
    int64_t mask_stride;
    bf16* ctx;        // [B, T, Hq, D]
    float2* stats;    // [B, T, Hq] (M in base 2, 1 / l), or null
    float* weights;   // [B, Hkv, capacity]
    int64_t batch;
    int64_t tokens;
    int64_t q_heads;
    int64_t kv_heads;
    int64_t capacity;
};

// Committed rows and valid queries of a sequence, forced into the ranges that keep every access inside the cache: a
// query whose own row would lie past the capacity is not valid.
__device__ __forceinline__ int64_t committed_rows(const CacheAttentionParams& p, int64_t b) {
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : (n > p.capacity ? p.capacity : n);
}

__device__ __forceinline__ int64_t valid_queries(const CacheAttentionParams& p, int64_t b) {
    const int64_t room = p.capacity - committed_rows(p, b);
    const int64_t most = room < p.tokens ? room : p.tokens;
    const int64_t n = p.counts == nullptr ? p.tokens : p.counts[b];
    return n < 0 ? 0 : (n > most ? most : n);
}

// Whether query t sees new row j (0 <= j < the sequence's valid queries).
__device__ __forceinline__ bool sees(const CacheAttentionParams& p, int64_t b, int64_t t, int64_t j) {
    return p.mask == nullptr ? j <= t : p.mask[b * p.mask_stride + t * p.tokens + j] != 0;
}

template <int kDims>
__device__ __forceinline__ void load_row(const bf16* row, int lane, float (&f)[kDims / 32]) {
#pragma unroll
    for (int i = 0; i < kDims / 32; ++i) {
        f[i] = __bfloat162float(row[i * 32 + lane]);
    }
}

template <int kDims>
__global__ void __launch_bounds__(128) cache_attention_kernel(const CacheAttentionParams p) {
    grid_dependency_begin();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);  // (b, t, head)
    if (row >= p.batch * p.tokens * p.q_heads) {
        return;
    }
    const int64_t h = row % p.q_heads;
    const int64_t t = row / p.q_heads % p.tokens;
    const int64_t b = row / p.q_heads / p.tokens;
    const int64_t kvh = h / (p.q_heads / p.kv_heads);
    const int64_t len = committed_rows(p, b);
    const int64_t n = valid_queries(p, b);
    const float c = 1.4426950408889634f / sqrtf(static_cast<float>(kDims));
    float q[kDims / 32];
    float o[kDims / 32] = {};
    load_row<kDims>(p.q + row * kDims, lane, q);
    const bf16* k = p.k + b * p.ks[0] + kvh * p.ks[2];
    const bf16* v = p.v + b * p.vs[0] + kvh * p.vs[2];
    float top = -INFINITY;
    float sum = 0.0f;
    for (int64_t j = 0; t < n && j < len + n; ++j) {
        if (j >= len && !sees(p, b, t, j - len)) {
            continue;
        }
        float kf[kDims / 32];
        load_row<kDims>(k + j * p.ks[1], lane, kf);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kDims / 32; ++i) {
            s = __fmaf_rn(q[i], kf[i], s);
        }
        s = group_sum<32>(s) * c;
        const float m = fmaxf(top, s);
        const float old = top == -INFINITY ? 0.0f : exp2f(top - m);
        const float e = exp2f(s - m);
        top = m;
        sum = __fmaf_rn(sum, old, e);
        load_row<kDims>(v + j * p.vs[1], lane, kf);
#pragma unroll
        for (int i = 0; i < kDims / 32; ++i) {
            o[i] = __fmaf_rn(o[i], old, e * kf[i]);
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kDims / 32; ++i) {
        p.ctx[row * kDims + i * 32 + lane] = __float2bfloat16(o[i] * inv);
    }
    if (p.stats != nullptr && lane == 0) {
        p.stats[row] = make_float2(top == -INFINITY ? 0.0f : top, inv);
    }
}

template <int kDims>
__global__ void __launch_bounds__(128) cache_weights_kernel(const CacheAttentionParams p) {
    grid_dependency_begin();
    const int lane = threadIdx.x & 31;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);  // (b, kv head, cached row)
    if (at >= p.batch * p.kv_heads * p.capacity) {
        return;
    }
    const int64_t j = at % p.capacity;
    const int64_t kvh = at / p.capacity % p.kv_heads;
    const int64_t b = at / p.capacity / p.kv_heads;
    const int64_t len = committed_rows(p, b);
    const int64_t n = valid_queries(p, b);
    if (j >= len + n) {
        return;
    }
    const int64_t group = p.q_heads / p.kv_heads;
    const float c = 1.4426950408889634f / sqrtf(static_cast<float>(kDims));
    float kf[kDims / 32];
    load_row<kDims>(p.k + b * p.ks[0] + j * p.ks[1] + kvh * p.ks[2], lane, kf);
    float sum = 0.0f;
    for (int64_t t = j < len ? 0 : j - len; t < n; ++t) {
        for (int64_t g = 0; g < group; ++g) {
            const int64_t row = (b * p.tokens + t) * p.q_heads + kvh * group + g;
            float q[kDims / 32];
            load_row<kDims>(p.q + row * kDims, lane, q);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kDims / 32; ++i) {
                s = __fmaf_rn(q[i], kf[i], s);
            }
            s = group_sum<32>(s) * c;
            const float2 st = p.stats[row];
            sum = __fmaf_rn(exp2f(s - st.x), st.y, sum);
        }
    }
    if (lane == 0) {
        p.weights[at] += sum;
    }
}

template <int kDims>
cudaError_t launch_cache_attention(const CacheAttentionParams& p, cudaStream_t s) {
    const int64_t rows = p.batch * p.tokens * p.q_heads;
    return runtime::launch(cache_attention_kernel<kDims>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), s, 1u,
                           p);
}

template <int kDims>
cudaError_t launch_cache_weights(const CacheAttentionParams& p, cudaStream_t s) {
    const int64_t rows = p.batch * p.kv_heads * p.capacity;
    return runtime::launch(cache_weights_kernel<kDims>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), s, 1u, p);
}

int check_sizes(const char* op, int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                int64_t capacity) {
    const std::string name(op);
    CPPINF_REQUIRE(batch >= 0 && tokens >= 0 && capacity >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                   name + " requires non-negative sizes.");
    CPPINF_REQUIRE(q_heads > 0 && kv_heads > 0, CPPINF_ERR_INVALID_ARGUMENT,
                   name + " requires non-zero head configuration.");
    CPPINF_REQUIRE(q_heads % kv_heads == 0, CPPINF_ERR_INVALID_ARGUMENT,
                   name + " requires query heads to divide by key/value heads.");
    CPPINF_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, CPPINF_ERR_UNSUPPORTED,
                   name + " supports head sizes 64, 128 and 256.");
    CPPINF_REQUIRE(q_heads / kv_heads <= kMaxGroup, CPPINF_ERR_UNSUPPORTED,
                   name + " supports up to 128 query heads per key/value head.");
    constexpr int64_t kMost = int64_t{1} << 31;
    CPPINF_REQUIRE(capacity < kMost && q_heads < (1 << 16) && batch < (1 << 24) &&
                       (batch == 0 || tokens == 0 || tokens * q_heads < kMost / batch) &&
                       (batch == 0 || capacity == 0 || kv_heads < kMost * 4 / (batch * capacity)),
                   CPPINF_ERR_OVERFLOW, name + " sizes exceed the kernels' index range.");
    return CPPINF_OK;
}

int check_cache(const char* op, const void* cache, const int64_t* strides) {
    const std::string name(op);
    CPPINF_REQUIRE(cache && strides, CPPINF_ERR_INVALID_ARGUMENT, name + " received a null pointer.");
    for (int i = 0; i < 3; ++i) {
        CPPINF_REQUIRE(strides[i] >= 0, CPPINF_ERR_INVALID_ARGUMENT, name + " requires non-negative cache strides.");
        CPPINF_REQUIRE(strides[i] % 8 == 0, CPPINF_ERR_UNSUPPORTED,
                       name + " requires cache strides in multiples of 8 elements.");
    }
    CPPINF_REQUIRE(runtime::aligned16(cache), CPPINF_ERR_UNSUPPORTED, name + " requires 16-byte aligned caches.");
    return CPPINF_OK;
}

int run_attention(const char* op, const CacheAttentionParams& p, int64_t head_dim, cudaStream_t s) {
    const cudaError_t err = head_dim == 64    ? launch_cache_attention<64>(p, s)
                            : head_dim == 128 ? launch_cache_attention<128>(p, s)
                                              : launch_cache_attention<256>(p, s);
    return runtime::launched(err, op);
}

int run_weights(const char* op, const CacheAttentionParams& p, int64_t head_dim, cudaStream_t s) {
    const cudaError_t err = head_dim == 64    ? launch_cache_weights<64>(p, s)
                            : head_dim == 128 ? launch_cache_weights<128>(p, s)
                                              : launch_cache_weights<256>(p, s);
    return runtime::launched(err, op);
}

}  // namespace
}  // namespace cppinf::device

using namespace cppinf::device;
namespace rt = cppinf::runtime;

extern "C" {

int64_t cppinf_cache_attention_scratch_bytes(int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                                             int64_t head_dim, int64_t capacity, int with_weights) {
    if (check_sizes("cache_attention_scratch_bytes", batch, tokens, q_heads, kv_heads, head_dim, capacity) !=
        CPPINF_OK) {
        return -1;
    }
    return with_weights ? batch * tokens * q_heads * static_cast<int64_t>(sizeof(float2)) : 0;
}

int cppinf_tree_attention(const void* q, const void* k_cache, const int64_t* k_strides, const void* v_cache,
                          const int64_t* v_strides, const int64_t* lengths, const uint8_t* mask,
                          int64_t mask_batch_stride, const int64_t* nodes, void* ctx, int64_t batch, int64_t tokens,
                          int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t capacity, void* scratch,
                          int64_t scratch_bytes, unsigned int* error, void* stream) {
    constexpr const char* kOp = "tree_attention";
    (void)scratch;
    (void)scratch_bytes;
    (void)error;
    if (const int st = check_sizes(kOp, batch, tokens, q_heads, kv_heads, head_dim, capacity); st != CPPINF_OK) {
        return st;
    }
    CPPINF_REQUIRE(tokens <= kMaxNodes, CPPINF_ERR_UNSUPPORTED,
                   "tree_attention supports up to 256 drafted tokens per sequence.");
    CPPINF_REQUIRE(mask_batch_stride >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                   "tree_attention requires a non-negative mask stride.");
    if (batch == 0 || tokens == 0) {
        return rt::ok();
    }
    CPPINF_REQUIRE(q && lengths && mask && ctx, CPPINF_ERR_INVALID_ARGUMENT, "tree_attention received a null pointer.");
    if (const int st = check_cache(kOp, k_cache, k_strides); st != CPPINF_OK) {
        return st;
    }
    if (const int st = check_cache(kOp, v_cache, v_strides); st != CPPINF_OK) {
        return st;
    }
    CPPINF_REQUIRE(rt::aligned16(q) && rt::aligned16(ctx), CPPINF_ERR_UNSUPPORTED,
                   "tree_attention requires 16-byte aligned queries and contexts.");
    CacheAttentionParams p{};
    p.q = static_cast<const bf16*>(q);
    p.k = static_cast<const bf16*>(k_cache);
    p.v = static_cast<const bf16*>(v_cache);
    for (int i = 0; i < 3; ++i) {
        p.ks[i] = k_strides[i];
        p.vs[i] = v_strides[i];
    }
    p.lengths = lengths;
    p.counts = nodes;
    p.mask = mask;
    p.mask_stride = mask_batch_stride;
    p.ctx = static_cast<bf16*>(ctx);
    p.batch = batch;
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.capacity = capacity;
    return run_attention(kOp, p, head_dim, rt::as_stream(stream));
}

int cppinf_decoder_attention_weights(const void* q, const void* k_cache, const int64_t* k_strides, const void* v_cache,
                                     const int64_t* v_strides, const int64_t* lengths, const int64_t* counts, void* ctx,
                                     float* weights, int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                                     int64_t head_dim, int64_t capacity, void* scratch, int64_t scratch_bytes,
                                     unsigned int* error, void* stream) {
    constexpr const char* kOp = "decoder_attention_weights";
    (void)error;
    if (const int st = check_sizes(kOp, batch, tokens, q_heads, kv_heads, head_dim, capacity); st != CPPINF_OK) {
        return st;
    }
    if (batch == 0 || tokens == 0) {
        return rt::ok();
    }
    CPPINF_REQUIRE(q && lengths && ctx && weights, CPPINF_ERR_INVALID_ARGUMENT,
                   "decoder_attention_weights received a null pointer.");
    if (const int st = check_cache(kOp, k_cache, k_strides); st != CPPINF_OK) {
        return st;
    }
    if (const int st = check_cache(kOp, v_cache, v_strides); st != CPPINF_OK) {
        return st;
    }
    CPPINF_REQUIRE(rt::aligned16(q) && rt::aligned16(ctx), CPPINF_ERR_UNSUPPORTED,
                   "decoder_attention_weights requires 16-byte aligned queries and contexts.");
    const int64_t need =
        cppinf_cache_attention_scratch_bytes(batch, tokens, q_heads, kv_heads, head_dim, capacity, 1);
    CPPINF_REQUIRE(scratch_bytes >= need && (need == 0 || scratch), CPPINF_ERR_INVALID_ARGUMENT,
                   "decoder_attention_weights requires a scratch of cppinf_cache_attention_scratch_bytes.");
    CPPINF_REQUIRE(rt::aligned16(scratch), CPPINF_ERR_UNSUPPORTED,
                   "decoder_attention_weights requires a 16-byte aligned scratch.");
    CacheAttentionParams p{};
    p.q = static_cast<const bf16*>(q);
    p.k = static_cast<const bf16*>(k_cache);
    p.v = static_cast<const bf16*>(v_cache);
    for (int i = 0; i < 3; ++i) {
        p.ks[i] = k_strides[i];
        p.vs[i] = v_strides[i];
    }
    p.lengths = lengths;
    p.counts = counts;
    p.ctx = static_cast<bf16*>(ctx);
    p.stats = static_cast<float2*>(scratch);
    p.weights = weights;
    p.batch = batch;
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.capacity = capacity;
    if (const int st = run_attention(kOp, p, head_dim, rt::as_stream(stream)); st != CPPINF_OK) {
        return st;
    }
    return run_weights(kOp, p, head_dim, rt::as_stream(stream));
}

}  // extern "C"
