// Eviction of cached rows by accumulated attention weight: of each sequence's rows, per key-value head, the first
// `sinks`, the last `recent` and the heaviest of the others stay, `keep` in all, in their order.
//
// Two kernels. The first finds the kept rows: weights map to unsigned keys of the same order (NaN lowest, -0 as +0),
// a radix select of four 8-bit digits finds the key of the last row that stays and how many rows of that very key do
// (the lowest rows first), and one pass in row order writes the kept rows' indices and weights. The second copies the
// kept K and V rows, one 16-byte vector per thread, and is bound by their bytes.
#include "common.cuh"
#include "runtime.h"

namespace cppinf::device {
namespace {

constexpr int kSelectThreads = 1024;

struct EvictParams {
    const char* k;
    const char* v;
    int64_t ks[3];  // byte strides {batch, row, head}
    int64_t vs[3];
    const float* weights;     // [B, Hkv, capacity]
    const int64_t* lengths;   // [B]
    char* k_out;              // [B, out_capacity, Hkv, D]
    char* v_out;
    float* weights_out;       // [B, Hkv, out_capacity]
    int64_t* lengths_out;     // [B]
    int64_t* index;           // [B, Hkv, keep]
    int64_t batch;
    int64_t kv_heads;
    int64_t columns;          // 16-byte columns of a row
    int64_t capacity;
    int64_t keep;
    int64_t recent;
    int64_t sinks;
    int64_t out_capacity;
};

__device__ __forceinline__ int64_t cached_rows(const EvictParams& p, int64_t b) {
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : (n > p.capacity ? p.capacity : n);
}

// Unsigned key in the order of the weights: NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) {
        return 0u;
    }
    const uint32_t bits = __float_as_uint(w + 0.0f);
    return (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
}

// Sum over the block of each thread's flag before the thread (exclusive prefix), with the total.
__device__ __forceinline__ int block_rank(bool flag, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const unsigned who = __ballot_sync(0xffffffffu, flag);
    if (lane == 0) {
        warp_sums[warp] = __popc(who);
    }
    __syncthreads();
    int before = 0;
    int all = 0;
    for (int w = 0; w < kSelectThreads / 32; ++w) {
        const int n = warp_sums[w];
        before += w < warp ? n : 0;
        all += n;
    }
    __syncthreads();
    *total = all;
    return before + __popc(who & ((1u << lane) - 1u));
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams p) {
    __shared__ int histogram[256];
    __shared__ int warp_sums[kSelectThreads / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    grid_dependency_begin();
    const int tid = threadIdx.x;
    const int64_t h = blockIdx.x % p.kv_heads;
    const int64_t b = blockIdx.x / p.kv_heads;
    const int64_t len = cached_rows(p, b);
    const float* w = p.weights + (b * p.kv_heads + h) * p.capacity;
    float* w_out = p.weights_out + (b * p.kv_heads + h) * p.out_capacity;
    int64_t* index = p.index + (b * p.kv_heads + h) * p.keep;
    const int64_t left = len < p.keep ? len : p.keep;
    if (h == 0 && tid == 0) {
        p.lengths_out[b] = left;
    }
    for (int64_t i = left + tid; i < p.out_capacity; i += kSelectThreads) {
        w_out[i] = 0.0f;
    }
    if (len <= p.keep) {
        for (int64_t i = tid; i < p.keep; i += kSelectThreads) {
            index[i] = i < len ? i : -1;
            if (i < len) {
                w_out[i] = w[i];
            }
        }
        return;
    }
    const int64_t lo = p.sinks;
    const int64_t hi = len - p.recent;
    uint32_t prefix = 0;
    uint32_t known = 0;
    int need = static_cast<int>(p.keep - p.sinks - p.recent);  // of the rows [lo, hi)
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelectThreads) {
            histogram[i] = 0;
        }
        __syncthreads();
        for (int64_t i = lo + tid; i < hi; i += kSelectThreads) {
            const uint32_t key = order_key(w[i]);
            if ((key & known) == prefix) {
                atomicAdd(&histogram[(key >> shift) & 255u], 1);
            }
        }
        __syncthreads();
        if (tid == 0) {
            int above = 0;
            int digit = 255;
            while (digit > 0 && above + histogram[digit] < need) {
                above += histogram[digit];
                --digit;
            }
            s_prefix = prefix | (static_cast<uint32_t>(digit) << shift);
            s_need = need - above;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        known |= 255u << shift;
    }
    // Rows in order: those that stay are the fixed ones, keys above the last kept key, and the first `need` equal to it.
    int64_t out = 0;
    int equal = 0;
    for (int64_t i0 = 0; i0 < len; i0 += kSelectThreads) {
        const int64_t i = i0 + tid;
        const bool inside = i < len;
        const float value = inside ? w[i] : 0.0f;
        const uint32_t key = order_key(value);
        const bool ranked = inside && i >= lo && i < hi;
        const bool tie = ranked && key == prefix;
        int ties = 0;
        const int tie_rank = equal + block_rank(tie, warp_sums, &ties);
        const bool stays = inside && (!ranked || key > prefix || (tie && tie_rank < need));
        int kept = 0;
        const int64_t at = out + block_rank(stays, warp_sums, &kept);
        if (stays) {
            index[at] = i;
            w_out[at] = value;
        }
        equal += ties;
        out += kept;
    }
}

__global__ void __launch_bounds__(256) evict_copy_kernel(const EvictParams p) {
    grid_dependency_begin();
    int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t each = p.batch * p.out_capacity * p.kv_heads * p.columns;
    if (i >= 2 * each) {
        return;
    }
    const bool value = i >= each;
    i -= value ? each : 0;
    uint4* out = reinterpret_cast<uint4*>(value ? p.v_out : p.k_out) + i;
    const int64_t column = i % p.columns;
    i /= p.columns;
    const int64_t h = i % p.kv_heads;
    i /= p.kv_heads;
    const int64_t row = i % p.out_capacity;
    const int64_t b = i / p.out_capacity;
    const int64_t len = cached_rows(p, b);
    uint4 data = make_uint4(0u, 0u, 0u, 0u);
    if (row < (len < p.keep ? len : p.keep)) {
        const int64_t from = p.index[(b * p.kv_heads + h) * p.keep + row];
        const char* base = value ? p.v + b * p.vs[0] + from * p.vs[1] + h * p.vs[2]
                                 : p.k + b * p.ks[0] + from * p.ks[1] + h * p.ks[2];
        data = *reinterpret_cast<const uint4*>(base + column * 16);
    }
    *out = data;
}

}  // namespace
}  // namespace cppinf::device

using namespace cppinf::device;
namespace rt = cppinf::runtime;

extern "C" {

int cppinf_cache_evict(cppinf_dtype dtype, const void* k_cache, const int64_t* k_strides, const void* v_cache,
                       const int64_t* v_strides, const float* weights, const int64_t* lengths, void* k_out,
                       void* v_out, float* weights_out, int64_t* lengths_out, int64_t* index, int64_t batch,
                       int64_t kv_heads, int64_t head_dim, int64_t capacity, int64_t keep, int64_t recent,
                       int64_t sinks, int64_t out_capacity, void* stream) {
    CPPINF_REQUIRE(rt::valid_dtype(dtype), CPPINF_ERR_INVALID_ARGUMENT, "cache_evict received an unsupported dtype.");
    CPPINF_REQUIRE(batch >= 0 && kv_heads >= 0 && head_dim >= 0 && capacity >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                   "cache_evict requires non-negative sizes.");
    CPPINF_REQUIRE(recent >= 0 && sinks >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                   "cache_evict requires non-negative recent and sinks.");
    CPPINF_REQUIRE(keep >= 1 && sinks <= keep && recent <= keep - sinks, CPPINF_ERR_INVALID_ARGUMENT,
                   "cache_evict requires keep to be at least one and to cover recent and sinks.");
    CPPINF_REQUIRE(out_capacity >= keep, CPPINF_ERR_OUT_OF_RANGE, "cache_evict output is too small for the kept rows.");
    const int64_t size = static_cast<int64_t>(rt::dtype_size(dtype));
    CPPINF_REQUIRE(head_dim * size % 16 == 0, CPPINF_ERR_UNSUPPORTED,
                   "cache_evict requires head sizes in multiples of 16 bytes.");
    constexpr int64_t kMost = int64_t{1} << 31;
    CPPINF_REQUIRE(capacity < kMost && out_capacity < kMost && batch < (1 << 24) && kv_heads < (1 << 16) &&
                       head_dim < (1 << 16) && batch * kv_heads < kMost &&
                       (batch * kv_heads == 0 || head_dim == 0 ||
                        out_capacity < (int64_t{1} << 38) / (batch * kv_heads * head_dim)),
                   CPPINF_ERR_OVERFLOW, "cache_evict sizes exceed the launch range.");
    if (batch == 0 || kv_heads == 0 || head_dim == 0) {
        return rt::ok();
    }
    CPPINF_REQUIRE((capacity == 0 || (k_cache && v_cache && weights)) && k_strides && v_strides && lengths && k_out &&
                       v_out && weights_out && lengths_out && index,
                   CPPINF_ERR_INVALID_ARGUMENT, "cache_evict received a null pointer.");
    EvictParams p{};
    for (int i = 0; i < 3; ++i) {
        CPPINF_REQUIRE(k_strides[i] >= 0 && v_strides[i] >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                       "cache_evict requires non-negative cache strides.");
        CPPINF_REQUIRE(k_strides[i] * size % 16 == 0 && v_strides[i] * size % 16 == 0, CPPINF_ERR_UNSUPPORTED,
                       "cache_evict requires cache strides in multiples of 16 bytes.");
        p.ks[i] = k_strides[i] * size;
        p.vs[i] = v_strides[i] * size;
    }
    CPPINF_REQUIRE(rt::aligned16(k_cache) && rt::aligned16(v_cache) && rt::aligned16(k_out) && rt::aligned16(v_out),
                   CPPINF_ERR_UNSUPPORTED, "cache_evict requires 16-byte aligned caches.");
    p.k = static_cast<const char*>(k_cache);
    p.v = static_cast<const char*>(v_cache);
    p.weights = weights;
    p.lengths = lengths;
    p.k_out = static_cast<char*>(k_out);
    p.v_out = static_cast<char*>(v_out);
    p.weights_out = weights_out;
    p.lengths_out = lengths_out;
    p.index = index;
    p.batch = batch;
    p.kv_heads = kv_heads;
    p.columns = head_dim * size / 16;
    p.capacity = capacity;
    p.keep = keep;
    p.recent = recent;
    p.sinks = sinks;
    p.out_capacity = out_capacity;
    const cudaStream_t s = rt::as_stream(stream);
    if (const int st = rt::launched(rt::launch(evict_select_kernel, dim3(static_cast<unsigned>(batch * kv_heads)),
                                               dim3(kSelectThreads), s, 1u, p),
                                    "cache_evict selection");
        st != CPPINF_OK) {
        return st;
    }
    const int64_t vectors = 2 * batch * out_capacity * kv_heads * p.columns;
    return rt::launched(rt::launch(evict_copy_kernel, dim3(static_cast<unsigned>(rt::ceil_div(vectors, 256))), dim3(256),
                                   s, 1u, p),
                        "cache_evict copy");
}

}  // extern "C"
