// What follows the attention of a drafted tree: the path of drafted tokens that the model agrees with, and the move of
// that path's cache rows behind the committed ones.
//
// tree_accept: node 0 is the token the model produced last; from an accepted node p the walk goes to the child c of p
// with token[c] == predicted[p] (the lowest index where drafts repeat), and ends where there is none; the model's own
// token after the last accepted node is the next one. Whether a node would follow its parent depends on the two alone, so
// one warp per sequence first gives every node its following child, the minimum over its children in shared memory; the
// walk is then one shared-memory load per step. Bound by the latency of two dependent global loads.
//
// tree_commit: cache row len + i takes row len + path[i]. A path ascends from path[i] >= i, so going through it in
// order never overwrites a row that is still to be read; every 16-byte column of a head's rows is one thread's, which
// loads eight rows before it stores them, and the columns of all sequences, heads and both caches run side by side. Bound
// by the latency of a chain of loads: length and count, then a path's entries and their rows for each eight accepted
// nodes (one sequence of two accepted nodes of 8 x 128: 1.8 us; 64 of about 17: 4.9 us).
#include "common.cuh"
#include "runtime.h"

namespace cppinf::device {
namespace {

constexpr int kMaxNodes = 256;

__global__ void __launch_bounds__(32)
    tree_accept_kernel(const int64_t* tokens, const int64_t* parents, const int64_t* predicted, const int64_t* nodes,
                       int64_t* path, int64_t* counts, int64_t* next, int t) {
    __shared__ int64_t s_predicted[kMaxNodes];
    __shared__ int s_following[kMaxNodes];
    grid_dependency_begin();
    const int lane = threadIdx.x;
    const int64_t b = blockIdx.x;
    tokens += b * t;
    parents += b * t;
    predicted += b * t;
    path += b * t;
    int64_t n = nodes == nullptr ? t : nodes[b];
    n = n < 0 ? 0 : (n > t ? t : n);
    int64_t token[kMaxNodes / 32];
    int64_t parent[kMaxNodes / 32];
#pragma unroll
    for (int i = 0; i < kMaxNodes / 32; ++i) {
        const int c = i * 32 + lane;
        if (c < t) {
            token[i] = tokens[c];
            parent[i] = parents[c];
            s_predicted[c] = predicted[c];
            s_following[c] = kMaxNodes;
            path[c] = -1;
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kMaxNodes / 32; ++i) {
        const int c = i * 32 + lane;
        if (c < n && parent[i] >= 0 && parent[i] < c && token[i] == s_predicted[parent[i]]) {
            atomicMin(&s_following[parent[i]], c);
        }
    }
    __syncwarp();
    if (lane == 0) {
        int count = 0;
        int64_t following = -1;
        for (int at = n > 0 ? 0 : kMaxNodes; at < kMaxNodes; at = s_following[at]) {
            path[count++] = at;
            following = s_predicted[at];
        }
        counts[b] = count;
        next[b] = following;
    }
}

struct CommitParams {
    char* k;
    char* v;
    int64_t ks[3];  // byte strides {batch, row, head}
    int64_t vs[3];
    const int64_t* lengths;
    const int64_t* path;    // [B, T]
    const int64_t* counts;  // [B]
    int64_t batch;
    int64_t tokens;
    int64_t kv_heads;
    int64_t columns;  // 16-byte columns of a row
    int64_t capacity;
};

__global__ void __launch_bounds__(128) tree_commit_kernel(const CommitParams p) {
    grid_dependency_begin();
    int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= 2 * p.batch * p.kv_heads * p.columns) {
        return;
    }
    const int64_t column = i % p.columns;
    i /= p.columns;
    const int64_t h = i % p.kv_heads;
    i /= p.kv_heads;
    const bool value = (i & 1) != 0;
    const int64_t b = i >> 1;
    const int64_t* path = p.path + b * p.tokens;
    int64_t len = p.lengths[b];
    int64_t n = p.counts[b];
    len = len < 0 ? 0 : (len > p.capacity ? p.capacity : len);
    const int64_t drafted = p.tokens < p.capacity - len ? p.tokens : p.capacity - len;  // rows inside the cache
    n = n < 0 ? 0 : (n > drafted ? drafted : n);
    const int64_t stride = value ? p.vs[1] : p.ks[1];
    char* rows = value ? p.v + b * p.vs[0] + h * p.vs[2] : p.k + b * p.ks[0] + h * p.ks[2];
    rows += len * stride + column * 16;
    constexpr int kBatch = 8;
    for (int64_t to = 0; to < n; to += kBatch) {
        uint4 x[kBatch];
        bool moves[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int64_t from = to + j < n ? path[to + j] : 0;
            moves[j] = from > to + j && from < drafted;
            if (moves[j]) {
                x[j] = *reinterpret_cast<const uint4*>(rows + from * stride);
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (moves[j]) {
                *reinterpret_cast<uint4*>(rows + (to + j) * stride) = x[j];
            }
        }
    }
}

}  // namespace
}  // namespace cppinf::device

using namespace cppinf::device;
namespace rt = cppinf::runtime;

extern "C" {

int cppinf_tree_accept(const int64_t* tokens, const int64_t* parents, const int64_t* predicted, const int64_t* nodes,
                       int64_t* path, int64_t* counts, int64_t* next, int64_t batch, int64_t tokens_per_sequence,
                       void* stream) {
    CPPINF_REQUIRE(batch >= 0 && tokens_per_sequence >= 0, CPPINF_ERR_INVALID_ARGUMENT,
                   "tree_accept requires non-negative sizes.");
    CPPINF_REQUIRE(tokens_per_sequence <= kMaxNodes, CPPINF_ERR_UNSUPPORTED,
                   "tree_accept supports up to 256 drafted tokens per sequence.");
    CPPINF_REQUIRE(batch < (int64_t{1} << 31), CPPINF_ERR_OVERFLOW, "tree_accept batch exceeds the launch range.");
    if (batch == 0) {
        return rt::ok();
    }
    CPPINF_REQUIRE(counts && next && (tokens_per_sequence == 0 || (tokens && parents && predicted && path)),
                   CPPINF_ERR_INVALID_ARGUMENT, "tree_accept received a null pointer.");
    const cudaError_t err =
        rt::launch(tree_accept_kernel, dim3(static_cast<unsigned>(batch)), dim3(32), rt::as_stream(stream), 1u, tokens,
                   parents, predicted, nodes, path, counts, next, static_cast<int>(tokens_per_sequence));
    return rt::launched(err, "tree_accept");
}

int cppinf_tree_commit(cppinf_dtype dtype, void* k_cache, const int64_t* k_strides, void* v_cache,
                       const int64_t* v_strides, const int64_t* lengths, const int64_t* path, const int64_t* counts,
                       int64_t batch, int64_t tokens, int64_t kv_heads, int64_t head_dim, int64_t capacity,
                       void* stream) {
    CPPINF_REQUIRE(rt::valid_dtype(dtype), CPPINF_ERR_INVALID_ARGUMENT, "tree_commit received an unsupported dtype.");
    CPPINF_REQUIRE(batch >= 0 && tokens >= 0 && kv_heads >= 0 && head_dim >= 0 && capacity >= 0,
                   CPPINF_ERR_INVALID_ARGUMENT, "tree_commit requires non-negative sizes.");
    const int64_t size = static_cast<int64_t>(rt::dtype_size(dtype));
    CPPINF_REQUIRE(head_dim * size % 16 == 0, CPPINF_ERR_UNSUPPORTED,
                   "tree_commit requires head sizes in multiples of 16 bytes.");
    constexpr int64_t kMost = int64_t{1} << 36;
    CPPINF_REQUIRE(batch < (1 << 24) && kv_heads < (1 << 16) && head_dim < (1 << 16) &&
                       batch * kv_heads * (head_dim > 0 ? head_dim : 1) < kMost,
                   CPPINF_ERR_OVERFLOW, "tree_commit sizes exceed the launch range.");
    if (batch == 0 || tokens == 0 || kv_heads == 0 || head_dim == 0 || capacity == 0) {
        return rt::ok();
    }
    CPPINF_REQUIRE(k_cache && v_cache && k_strides && v_strides && lengths && path && counts,
                   CPPINF_ERR_INVALID_ARGUMENT, "tree_commit received a null pointer.");
    CommitParams p{};
    for (int i = 0; i < 3; ++i) {
        CPPINF_REQUIRE(k_strides[i] > 0 && v_strides[i] > 0, CPPINF_ERR_INVALID_ARGUMENT,
                       "tree_commit requires positive cache strides.");
        CPPINF_REQUIRE(k_strides[i] * size % 16 == 0 && v_strides[i] * size % 16 == 0, CPPINF_ERR_UNSUPPORTED,
                       "tree_commit requires cache strides in multiples of 16 bytes.");
        p.ks[i] = k_strides[i] * size;
        p.vs[i] = v_strides[i] * size;
    }
    CPPINF_REQUIRE(rt::aligned16(k_cache) && rt::aligned16(v_cache), CPPINF_ERR_UNSUPPORTED,
                   "tree_commit requires 16-byte aligned caches.");
    CPPINF_REQUIRE(k_cache != v_cache, CPPINF_ERR_INVALID_ARGUMENT, "tree_commit requires K and V caches of their own.");
    p.k = static_cast<char*>(k_cache);
    p.v = static_cast<char*>(v_cache);
    p.lengths = lengths;
    p.path = path;
    p.counts = counts;
    p.batch = batch;
    p.tokens = tokens;
    p.kv_heads = kv_heads;
    p.columns = head_dim * size / 16;
    p.capacity = capacity;
    const int64_t threads = 2 * batch * kv_heads * p.columns;
    const cudaError_t err = rt::launch(tree_commit_kernel, dim3(static_cast<unsigned>(rt::ceil_div(threads, 128))),
                                       dim3(128), rt::as_stream(stream), 1u, p);
    return rt::launched(err, "tree_commit");
}

}  // extern "C"
