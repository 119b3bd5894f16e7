// Eviction of cached rows by accumulated attention weight: of each sequence's rows, per key-value head, the first
// `sinks`, the last `recent` and the heaviest of the others stay, `keep` in all, in their order.
//
// Two kernels. The first finds the kept rows, one CTA per sequence and head: weights map to unsigned keys of the same
// order (NaN lowest, -0 as +0), which are put into shared memory; a radix select of three digits finds the key of the last
// row that stays and how many rows of that very key do (the lowest rows first; digits of 11 bits, since weights have few
// exponents and the counters of a shorter digit are hit by many threads at once); then each warp counts the kept rows
// of its own stretch of keys, one scan over the warps places them, and their indices are written, 32 keys a step. Its
// time is a chain of a few dozen shared-memory round trips and barriers: 16 sequences of up to 16384 rows and 8 heads of
// 128, cut to 2048, take 57.2 us, of which the copy has about 40 (66.8 us where each pass made the keys anew and each
// thread wrote the kept rows of its own stretch). The second copies the kept rows' weights, K and
// V, one 16-byte vector per thread and step, the source rows of a CTA's share looked up once, and is bound by their bytes.
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

constexpr int kDigits = 2048;       // values of a digit
constexpr int kSharedKeys = 49152;  // keys of a head that fit into shared memory beside the rest

// The kept rows of one head. The keys lie in shared memory, or, where the cache is too long for that, are made again from
// the weights each time.
template <bool kShared>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams p) {
    extern __shared__ uint4 s_fours[];  // the keys, and zeros (the lowest key) up to the next multiple of four
    __shared__ int histogram[kDigits];
    __shared__ int warp_sums[kSelectThreads / 32];
    __shared__ int warp_ties[kSelectThreads / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    grid_dependency_begin();
    const int tid = threadIdx.x;
    const int lane = tid & 31;
    const int warp = tid >> 5;
    const int64_t head = blockIdx.x;  // of all sequences
    const int64_t b = head / p.kv_heads;
    const int len = static_cast<int>(cached_rows(p, b));
    int64_t* index = p.index + head * p.keep;
    const int keep = static_cast<int>(p.keep);
    if (head == b * p.kv_heads && tid == 0) {
        p.lengths_out[b] = len < keep ? len : keep;
    }
    if (len <= keep) {
        for (int i = tid; i < keep; i += kSelectThreads) {
            index[i] = i < len ? i : -1;
        }
        return;
    }
    const int sinks = static_cast<int>(p.sinks);
    const int recent = static_cast<int>(p.recent);
    const int n = len - sinks - recent;  // rows [sinks, sinks + n) are ranked
    const int fours = (n + 3) / 4;
    const float* ranked = p.weights + head * p.capacity + sinks;
    uint32_t* s_keys = reinterpret_cast<uint32_t*>(s_fours);
    for (int i = tid; i < sinks; i += kSelectThreads) {
        index[i] = i;
    }
    for (int i = tid; i < recent; i += kSelectThreads) {
        index[keep - recent + i] = len - recent + i;
    }
    int need = keep - sinks - recent;
    if (need == 0) {
        return;
    }
    if (kShared) {
        constexpr int kBatch = 16;  // loads in flight
        for (int i0 = tid; i0 < fours * 4; i0 += kBatch * kSelectThreads) {
            float x[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int i = i0 + j * kSelectThreads;
                x[j] = i < n ? ranked[i] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int i = i0 + j * kSelectThreads;
                if (i < fours * 4) {
                    s_keys[i] = i < n ? order_key(x[j]) : 0u;
                }
            }
        }
    }
    const auto key_of = [&](int i) { return kShared ? s_keys[i] : order_key(ranked[i]); };
    uint32_t prefix = 0;
    uint32_t known = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
        histogram[tid] = 0;
        histogram[tid + kSelectThreads] = 0;
        __syncthreads();
        const auto count = [&](uint32_t key) {
            if ((key & known) == prefix) {
                atomicAdd(&histogram[(key >> shift) & digits], 1);
            }
        };
        if (kShared) {
#pragma unroll 4
            for (int i = tid; i < fours; i += kSelectThreads) {
                const uint4 keys = s_fours[i];
                count(keys.x);
                count(keys.y);
                count(keys.z);
                count(keys.w);
            }
        } else {
#pragma unroll 4
            for (int i = tid; i < n; i += kSelectThreads) {
                count(order_key(ranked[i]));
            }
        }
        __syncthreads();
        // The digit at which the keys from the highest down reach `need`; a thread has two digits.
        const int digit = kDigits - 1 - 2 * tid;
        const int upper = histogram[digit];
        const int mine = upper + histogram[digit - 1];
        int sum = mine;
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, sum, offset);
            sum += lane >= offset ? other : 0;
        }
        if (lane == 31) {
            warp_sums[warp] = sum;
        }
        __syncthreads();
        const int above = sum - mine + __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0);
        if (above < need && above + mine >= need) {
            const bool first = above + upper >= need;
            s_prefix = prefix | (static_cast<uint32_t>(first ? digit : digit - 1) << shift);
            s_need = need - above - (first ? 0 : upper);
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        known |= digits << shift;
    }
    // Of the rows of key `prefix` the first `need` stay, and all of higher keys. A warp's stretch is whole steps of 32.
    const int stretch = (n + kSelectThreads - 1) / kSelectThreads * 32;
    const int begin = warp * stretch;
    const int end = begin + stretch < n ? begin + stretch : n;
    int higher = 0;
    int ties = 0;
#pragma unroll 4
    for (int i = begin + lane; i < end; i += 32) {
        const uint32_t key = key_of(i);
        higher += key > prefix ? 1 : 0;
        ties += key == prefix ? 1 : 0;
    }
    higher = __reduce_add_sync(0xffffffffu, higher);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) {
        warp_sums[warp] = higher;
        warp_ties[warp] = ties;
    }
    __syncthreads();
    higher = __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0);
    ties = __reduce_add_sync(0xffffffffu, lane < warp ? warp_ties[lane] : 0);  // now those before a step
    const uint32_t lower_lanes = (1u << lane) - 1u;
    int64_t* out = index + sinks + higher + (ties < need ? ties : need);
#pragma unroll 4
    for (int i = begin + lane; i - lane < end; i += 32) {
        const bool inside = i < end;
        const uint32_t key = inside ? key_of(i) : 0u;
        const bool tie = inside && key == prefix;
        bool stays = inside && key > prefix;
        const uint32_t equals = __ballot_sync(0xffffffffu, tie);
        if (equals != 0u) {
            stays = stays || (tie && ties + __popc(equals & lower_lanes) < need);
            ties += __popc(equals);
        }
        const uint32_t all = __ballot_sync(0xffffffffu, stays);
        if (stays) {
            out[__popc(all & lower_lanes)] = sinks + i;
        }
        out += __popc(all);
    }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyRows = 32;  // kept rows of one head that a CTA copies

__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const EvictParams p, FastDiv columns, unsigned blocks) {
    __shared__ int s_from[kCopyRows];
    grid_dependency_begin();
    const unsigned head = blockIdx.x / blocks;  // of all sequences
    const int row0 = static_cast<int>(blockIdx.x % blocks) * kCopyRows;
    const int64_t b = head / static_cast<unsigned>(p.kv_heads);
    const int64_t h = head % static_cast<unsigned>(p.kv_heads);
    const int64_t len = cached_rows(p, b);
    const int left = static_cast<int>(len < p.keep ? len : p.keep);
    if (threadIdx.x < kCopyRows) {
        const int row = row0 + static_cast<int>(threadIdx.x);
        const int64_t from = row < left ? p.index[head * p.keep + row] : -1;
        s_from[threadIdx.x] = static_cast<int>(from);
        if (row < p.out_capacity) {
            p.weights_out[head * p.out_capacity + row] = from >= 0 ? p.weights[head * p.capacity + from] : 0.0f;
        }
    }
    __syncthreads();
    const int rows = p.out_capacity - row0 < kCopyRows ? static_cast<int>(p.out_capacity - row0) : kCopyRows;
    const unsigned vectors = static_cast<unsigned>(rows) * columns.d;
    const char* k = p.k + b * p.ks[0] + h * p.ks[2];
    const char* v = p.v + b * p.vs[0] + h * p.vs[2];
    const int64_t out0 = ((b * p.out_capacity + row0) * p.kv_heads + h) * columns.d;
#pragma unroll 4
    for (unsigned i = threadIdx.x; i < vectors; i += kCopyThreads) {
        const unsigned row = columns.quot(i);
        const int64_t column = i - row * columns.d;
        const int64_t from = s_from[row];
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        uint4 y = x;
        if (from >= 0) {
            x = ld_stream(k + from * p.ks[1] + column * 16);
            y = ld_stream(v + from * p.vs[1] + column * 16);
        }
        const int64_t to = out0 + row * p.kv_heads * columns.d + column;
        st_v4(reinterpret_cast<uint4*>(p.k_out) + to, x);
        st_v4(reinterpret_cast<uint4*>(p.v_out) + to, y);
    }
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
    CPPINF_REQUIRE(batch >= 0 && capacity >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                   "cache_evict requires non-negative sizes.");
    CPPINF_REQUIRE(kv_heads > 0 && head_dim > 0, CPPINF_ERR_INVALID_ARGUMENT,
                   "cache_evict requires non-zero head configuration.");
    CPPINF_REQUIRE(recent >= 0 && sinks >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                   "cache_evict requires non-negative recent and sinks.");
    CPPINF_REQUIRE(keep >= 1 && sinks <= keep && recent <= keep - sinks, CPPINF_ERR_INVALID_ARGUMENT,
                   "cache_evict requires keep to be at least one and to cover recent and sinks.");
    CPPINF_REQUIRE(out_capacity >= keep, CPPINF_ERR_OUT_OF_RANGE, "cache_evict output is too small for the kept rows.");
    const int64_t size = static_cast<int64_t>(rt::dtype_size(dtype));
    CPPINF_REQUIRE(head_dim * size % 16 == 0, CPPINF_ERR_UNSUPPORTED,
                   "cache_evict requires head sizes in multiples of 16 bytes.");
    constexpr int64_t kMost = int64_t{1} << 31;
    CPPINF_REQUIRE(capacity < kMost / 2 && out_capacity < kMost / 2 && batch < (1 << 24) && kv_heads < (1 << 16) &&
                       head_dim < (1 << 16) && batch * kv_heads < kMost &&
                       (batch == 0 || rt::ceil_div(out_capacity, kCopyRows) < kMost / (batch * kv_heads)),
                   CPPINF_ERR_OVERFLOW, "cache_evict sizes exceed the launch range.");
    if (batch == 0) {
        return rt::ok();
    }
    CPPINF_REQUIRE((capacity == 0 || (k_cache && v_cache && weights)) && k_strides && v_strides && lengths && k_out &&
                       v_out && weights_out && lengths_out && index,
                   CPPINF_ERR_INVALID_ARGUMENT, "cache_evict received a null pointer.");
    EvictParams p{};
    for (int i = 0; i < 3; ++i) {
        CPPINF_REQUIRE(k_strides[i] > 0 && v_strides[i] > 0, CPPINF_ERR_INVALID_ARGUMENT,
                       "cache_evict requires positive cache strides.");
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
    p.capacity = capacity;
    p.keep = keep;
    p.recent = recent;
    p.sinks = sinks;
    p.out_capacity = out_capacity;
    const cudaStream_t s = rt::as_stream(stream);
    const unsigned heads = static_cast<unsigned>(batch * kv_heads);
    cudaError_t err = cudaSuccess;
    if (capacity <= kSharedKeys) {
        const std::size_t bytes = static_cast<std::size_t>(rt::ceil_div(capacity, 4)) * sizeof(uint4);
        static rt::SharedMemoryLimit limit;
        CPPINF_CUDA_TRY(limit.raise(evict_select_kernel<true>, kSharedKeys * sizeof(uint32_t)));
        err = rt::launch_smem(evict_select_kernel<true>, dim3(heads), dim3(kSelectThreads), bytes, s, 1u, p);
    } else {
        err = rt::launch(evict_select_kernel<false>, dim3(heads), dim3(kSelectThreads), s, 1u, p);
    }
    if (const int st = rt::launched(err, "cache_evict selection"); st != CPPINF_OK) {
        return st;
    }
    const int64_t blocks = rt::ceil_div(out_capacity, kCopyRows);
    return rt::launched(rt::launch(evict_copy_kernel, dim3(static_cast<unsigned>(blocks * heads)), dim3(kCopyThreads), s,
                                   1u, p, FastDiv(static_cast<uint32_t>(head_dim * size / 16)),
                                   static_cast<unsigned>(blocks)),
                        "cache_evict copy");
}

}  // extern "C"
