// Attention of a batch of cached sequences that takes its sequence lengths from device memory, in two forms:
//  - cppinf_tree_attention: T drafted tokens per sequence behind its committed cache rows, each seeing all committed
//    rows and the drafted ones that a mask names (a tree's ancestors);
//  - cppinf_decoder_attention_weights: T causal tokens per sequence, with the attention weight that each cached row
//    received added to an f32 array (what an eviction ranks rows by).
//
// With s_j = q k_j / sqrt(D) over the rows j that a query sees, M their maximum and l = sum exp(s_j - M):
// ctx = sum exp(s_j - M) v_j / l, and row j's weight is the sum over the queries and the query heads of a key-value
// head of exp(s_j - M) / l. Scores, M, l and both sums are f32; exponentials are taken in base 2 with log2(e) / sqrt(D)
// folded into one factor. Probabilities are rounded to bf16 for their product with V (the tensor cores' operand type;
// the sum l keeps them in f32), contexts once at the end.
//
// Attention on the tensor cores (cache_attention_kernel). The G query heads of a key-value head share its K and V, so
// the rows (token, query head of the group) of one key-value head are packed into tiles of 128, the rows of a
// tcgen05.mma; a warpgroup of four warps owns such a tile's softmax, one thread per row. One pass over the keys, in
// tiles that TMA brings into a ring of shared-memory slots:
//     S = Q K^T (tensor memory) -> running maximum, P = exp2(...) written over S as bf16 -> O += P V (P from tensor
//     memory, V as an MN-major operand straight from its TMA tile).
// Two such chains run side by side and hide each other's softmax behind the other's matrix products: with up to 128
// rows per head, two key tiles in turn for one row tile (their sums are joined at the end); with more, two row tiles
// on the same K and V tiles, which are then read once for 256 rows. Head size 256 has room for one chain.
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time.
//
// All key tiles of all (sequence, row tile, key-value head) items form one line that is cut into equal parts, one per
// CTA (one CTA per SM), so ragged lengths and few sequences load all SMs alike. A CTA that takes only part of an item
// leaves its rows' maximum, sum and unnormalised O in the scratch, and a second kernel joins the parts of the items
// that a cut went through, in the order of their keys.
//
// Rows past a sequence's end and drafted rows that only some queries see may hold anything: scores there are replaced
// before the softmax, and V tiles in which some row is hidden from some query are cleared of such values in shared
// memory before the product (0 * NaN would be NaN); a value that is not finite in a row that a query does see is added
// to its O afterwards, times its probability, so that it counts as in a tile that all queries see.
#include <cmath>

#include "common.cuh"
#include "runtime.h"
#include "tcgen05.cuh"

namespace cppinf::device {
namespace {

using namespace tc;

constexpr int kMaxNodes = 256;  // drafted tokens of a sequence
constexpr int kMaxGroup = 128;  // query heads of a key-value head
constexpr int kMaxKeptRows = 32;  // rows of a head whose scores are kept for the weights
constexpr int64_t kMostScoreBytes = int64_t{1} << 30;  // of kept scores, unless they are few beside K and V

// Where a CTA's part of the line begins, for the kernel that joins the parts.
struct __align__(16) Cut {
    int b;
    int row_tile;
    int h;
    int piece;
    int total;   // pieces of the line
    int set_up;  // pieces of an item before its tiles
    int len;     // of sequence b
    int valid;
};

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
    float* stats;     // [B, Hkv, T, G] M + log2(l) in base 2, infinite for rows of no weight, or null
    float* weights;   // [B, Hkv, capacity]
    int64_t batch;
    int64_t tokens;
    int64_t q_heads;
    int64_t kv_heads;
    int64_t capacity;
    // Tiling (plan()) and scratch.
    int group;            // query heads of a key-value head
    int tile_tokens;      // tokens of a 128-row tile
    FastDiv by_tile_tokens;
    int item_tokens;      // tokens of an item: one or two tiles
    int row_tiles;        // items along the tokens
    int q_box_tokens;     // tokens of one TMA box of q
    bool whole_items;     // the line is cut between items only
    int part_rows;        // rows of a part in the scratch
    Cut* cuts;            // [CTAs]
    float2* part_ml;      // [2 CTAs][part_rows] (M in base 2, l)
    float* part_o;        // [2 CTAs][D / 4][part_rows][4]
    float* scores;          // [B, Hkv][rows][score_stride] S of few rows, kept for the weights, or null
    int64_t score_stride;
    unsigned int* tickets;  // [weight CTAs] parts of a unit that have been left, zeroed by the attention kernel
    float* part_sums;       // [2 weight CTAs][128]
    int weight_ctas;
    unsigned int* error;
    uint32_t poll_limit;
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

// What one item needs to know about its sequence (capacities lie below 2^31).
struct ItemRange {
    int len;       // committed rows
    int valid;     // valid queries
    int first;     // first token of the item
    int full_end;  // keys below are seen by every valid query of the item
    int kv_end;    // keys from here on are seen by none
};

__device__ __forceinline__ ItemRange item_range(const CacheAttentionParams& p, int len, int valid, int row_tile) {
    ItemRange r;
    r.len = len;
    r.valid = valid;
    r.first = row_tile * p.item_tokens;
    if (r.first >= r.valid) {
        r.full_end = 0;
        r.kv_end = 0;
    } else if (p.mask != nullptr) {
        r.full_end = r.len;
        r.kv_end = r.len + r.valid;
    } else {
        const int last = r.first + p.item_tokens;
        r.full_end = r.len + r.first + 1;
        r.kv_end = r.len + (last < r.valid ? last : r.valid);
    }
    return r;
}

// Key tiles of an item; one without visible keys still takes a tile, in which its rows become zeros.
template <int kKeys>
__device__ __forceinline__ int item_tiles(const ItemRange& r) {
    return r.kv_end > 0 ? (r.kv_end + kKeys - 1) / kKeys : 1;
}

// Head size's tiling: keys of a tile, chains side by side, slots of the K/V ring, shared memory.
constexpr int64_t kMostEntries = 1 << 20;  // (sequence, row tile) entries of a call: their groups are counted in the ring

template <int D, bool kPair>
struct Tiling {
    static constexpr int kKeys = D == 256 ? 64 : 128;
    static constexpr int kStreams = D == 256 ? 1 : 2;
    static constexpr int kAtoms = D / 64;
    static constexpr int kQTiles = kPair ? 2 : 1;
    static constexpr int kStep = kPair ? 1 : kStreams;  // a chain takes every kStep-th key tile of a segment
    // Slots for K tiles and as many for V tiles, in rings of their own for each pair of chains that shares tiles, or
    // for each chain that has tiles of its own: whoever waits for a slot's n-th tile has then seen its tile before.
    static constexpr int kRings = kPair ? 1 : kStreams;
    static constexpr int kDepth = (D == 64 ? 4 : 2) / kRings;
    static constexpr int kSlots = 2 * kRings * kDepth;
    static constexpr int kThreads = 128 + 128 * kStreams;
    static constexpr uint32_t kQAtom = 128 * 128;    // [128 rows][64 dims]
    static constexpr uint32_t kKvAtom = kKeys * 128;  // [keys][64 dims]
    static constexpr uint32_t kSlot = kKvAtom * kAtoms;
    static constexpr uint32_t kQ = 0;
    static constexpr uint32_t kRing = kQ + kQTiles * kAtoms * kQAtom;
    static constexpr uint32_t kMask = kRing + kSlots * kSlot;       // [chains][128][9] mask bits
    static constexpr uint32_t kMl = kMask + kStreams * 128 * 9 * 4;  // [128] the second chain's (M, l)
    static constexpr uint32_t kFlags = kMl + 128 * 8;               // [2][16]
    static constexpr uint32_t kBars = kFlags + 2 * 16 * 4;
    static constexpr std::size_t kBytes = 1024 + kBars + 384;
    // Tensor memory columns: the chains' S (P over it), one each or two for a lone chain, then their O.
    static constexpr int kAhead = 128 / kKeys;
    static constexpr int kHalf = kKeys / 2;  // P is handed over in halves
    static constexpr uint32_t kTmemO = kStreams * 128;
    static_assert(kSlots * kSlot >= kMostEntries / 32 * sizeof(int), "the groups' counts");
    static_assert(kDepth >= 1 && kStreams * (128 + D) <= 512, "tensor memory has 512 columns");

    // The slot of a ring's n-th K or V tile, and the parity of its barriers' phase.
    __device__ static __forceinline__ int k_slot(int ring, uint32_t n) { return ring * 2 * kDepth + static_cast<int>(n % kDepth); }
    __device__ static __forceinline__ int v_slot(int ring, uint32_t n) { return k_slot(ring, n) + kDepth; }
    __device__ static __forceinline__ uint32_t parity(uint32_t n) { return n / kDepth & 1u; }

    static_assert(kBytes <= 232448 - 512, "shared memory of a CTA");
};

constexpr uint32_t kTmemAll = 512;

// An item's share of the line: its key tiles, and before them `kSetUp` pieces without any for what an item costs besides
// its tiles (loading Q, the first S, writing the rows: 9000 to 12000 cycles, where a tile takes about 3000). Left out
// where CTAs have few tiles each and a set-up's place would be better taken by a tile. 64 sequences of up to 4000 rows:
// 132 us without, 122 us with 3, 121 us with 6.
constexpr int kSetUp = 3;
constexpr int kSetUpFrom = 8;  // tiles per CTA

// Where a CTA's part of the line is, item by item; every role of the CTA walks it for itself.
struct Walk {
    int b;
    int row_tile;
    int h;
    int piece;       // first piece of the current item that the part has
    int left;        // pieces of the part still to come, those of the current item included
    int set_up;      // pieces of each item before its tiles
    int len;         // of sequence b
    int valid;
    int index;       // segments before the current one
};

__device__ __forceinline__ void advance(const CacheAttentionParams& p, Walk& w, int tiles) {
    w.left -= p.whole_items ? 1 : tiles + w.set_up - w.piece;
    w.piece = 0;
    if (w.left <= 0 || ++w.h < static_cast<int>(p.kv_heads)) {
        return;
    }
    w.h = 0;
    if (++w.row_tile < p.row_tiles) {
        return;
    }
    w.row_tile = 0;
    ++w.b;
    w.len = static_cast<int>(committed_rows(p, w.b));
    w.valid = static_cast<int>(valid_queries(p, w.b));
}

// A line of `total` pieces cut into `parts` that differ by one piece at most.
struct Cuts {
    int each;
    int extra;  // the first `extra` parts have one more

    __device__ __forceinline__ Cuts(int total, int parts) : each(total / parts), extra(total - each * parts) {}
    __device__ __forceinline__ int begin(int part) const { return part * each + (part < extra ? part : extra); }
    __device__ __forceinline__ bool empty(int part) const { return each == 0 && part >= extra; }
    __device__ __forceinline__ int of(int piece) const {  // the part that a piece lies in
        const int longer = extra * (each + 1);
        return piece < longer ? piece / (each + 1) : extra + (piece - longer) / each;
    }
};

// Bounded waits: one that runs out of the poll limit sets the error word and waits again with the default limit; if
// that runs out too, `stop` ends all later waits of the CTA at once, so that it always comes to its end. Its loads end
// then, and it waits for the copies and products in flight, again with the limit, before it frees its tensor memory.
struct Waiter {
    unsigned int* error;
    uint32_t limit;
    volatile uint32_t* stop;

    __device__ __forceinline__ bool stopped() const { return *stop != 0u; }

    __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t phase) const {
        if (limit == 0u || !mbar_try_wait(bar, phase)) {
            slow(bar, phase);
        }
    }

    __device__ __forceinline__ void slow(uint64_t* bar, uint32_t phase) const {
        if (stopped() || mbar_wait_bounded(bar, phase, limit)) {
            return;
        }
        if (error != nullptr) {
            atomicOr(error, 1u);
        }
        if (!mbar_wait_bounded(bar, phase)) {
            *stop = 1u;
        }
    }
};

// Waits until the last of a slot's fills has landed; an odd number of them leaves its bit set in `filled`.
__device__ __forceinline__ void wait_landed(uint64_t* full, uint32_t filled, int slots) {
    for (int i = 0; i < slots; ++i) {
        mbar_wait_bounded(full + i, (filled >> i & 1u) ^ 1u);
    }
}

// Waits for the matrix products that this thread has issued.
__device__ __forceinline__ void wait_products(uint64_t* bar) {
    umma_commit(bar);
    mbar_wait_bounded(bar, 0u);
}

// Visible keys [key, key + 32) of a row as a bit mask. Tree: committed keys, then the row's mask bits (9 words, the last
// empty); causal: keys below `limit`.
__device__ __forceinline__ uint32_t visible_bits(const uint32_t* row, int key, int len, int limit) {
    if (row == nullptr) {
        const int n = limit - key;
        return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
    }
    const int j = key - len;
    if (j <= -32) {
        return 0xffffffffu;
    }
    if (j < 0) {
        return (row[0] << -j) | ((1u << -j) - 1u);
    }
    const int word = j >> 5;
    return word >= 8 ? 0u : __funnelshift_r(row[word], row[word + 1], static_cast<uint32_t>(j & 31));
}

// Scores of keys that the row does not see become -inf; words of 32 keys that every row of the warp sees are left alone.
// Returns whether the warp has other words.
template <int N>
__device__ __forceinline__ bool hide(float (&x)[N], const uint32_t* row, int key, int len, int limit) {
    bool hidden = false;
#pragma unroll
    for (int c = 0; c < N / 32; ++c) {
        const uint32_t see = visible_bits(row, key + c * 32, len, limit);
        if (!__all_sync(0xffffffffu, see == 0xffffffffu)) {
            hidden = true;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                x[c * 32 + j] = (see >> j & 1u) != 0u ? x[c * 32 + j] : -INFINITY;
            }
        }
    }
    return hidden;
}

// Stores N consecutive f32 columns of this thread's tensor-memory lane and waits for the stores.
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t taddr, const float (&x)[N]) {
#pragma unroll
    for (int c = 0; c < N / 16; ++c) {
        uint32_t r[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            r[j] = __float_as_uint(x[c * 16 + j]);
        }
        tmem_store16(taddr + c * 16, r);
    }
    tmem_store_wait();
}

template <int N>
__device__ __forceinline__ void keep(const float (&x)[N], float* to) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
        *reinterpret_cast<float4*>(to + 4 * j) = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
    }
}

template <int N>
__device__ __forceinline__ float largest(const float (&x)[N], float top) {
    float tops[4] = {top, top, top, top};
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        tops[j & 3] = max3(tops[j & 3], x[2 * j], x[2 * j + 1]);
    }
    return fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
}

// P of N keys, 2^(x factor + offset), stored as bf16 pairs at `taddr`; returns their sum in f32.
template <int N>
__device__ __forceinline__ float probabilities(const float (&x)[N], float2 factor, float2 offset, uint32_t taddr) {
    float2 sums[2] = {};
#pragma unroll
    for (int c = 0; c < N / 32; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int k = c * 32 + 2 * j;
            float2 e = __ffma2_rn(make_float2(x[k], x[k + 1]), factor, offset);
            e = make_float2(exp2_approx(e.x), exp2_approx(e.y));
            sums[j & 1] = __fadd2_rn(sums[j & 1], e);
            packed[j] = pack_bf16x2(e.x, e.y);
        }
        tmem_store16(taddr + c * 16, packed);
    }
    return (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
}

// A pair of bf16 values with +0 in the place of each that is not finite.
__device__ __forceinline__ uint32_t finite_pair(uint32_t pair) {
    return ((pair & 0x7f80u) == 0x7f80u ? 0u : pair & 0xffffu) |
           ((pair & 0x7f800000u) == 0x7f800000u ? 0u : pair & 0xffff0000u);
}

// acc + 0 * x for both values of a pair.
__device__ __forceinline__ uint32_t zero_times(uint32_t pair, uint32_t acc) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(pair), "r"(0u), "r"(acc));
    return d;
}

// What a row's probabilities are taken against for the weights: exp2(s - M) / l = exp2(s - (M + log2 l)). Its rounding
// counts for less than that of the scores, whose largest it exceeds by log2(l) at most.
__device__ __forceinline__ float whole_statistic(float top, float sum) {
    return sum == 0.0f ? INFINITY : top + log2f(sum);
}

template <int D, bool kPair>
__global__ void __launch_bounds__(Tiling<D, kPair>::kThreads, 1)
    cache_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const CacheAttentionParams p) {
    using L = Tiling<D, kPair>;
    constexpr int kStreams = L::kStreams;
    constexpr int kKeys = L::kKeys;
    extern __shared__ __align__(16) unsigned char raw[];
    unsigned char* sm = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    uint32_t* s_mask = reinterpret_cast<uint32_t*>(sm + L::kMask);
    float2* s_ml = reinterpret_cast<float2*>(sm + L::kMl);
    uint32_t* s_flags = reinterpret_cast<uint32_t*>(sm + L::kFlags);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBars);
    uint64_t* bar_full = bars;                    // [slots] a K or V tile has landed
    uint64_t* bar_empty = bars + L::kSlots;       // [slots] its products are done
    uint64_t* bar_q_full = bars + 2 * L::kSlots;
    uint64_t* bar_q_empty = bar_q_full + 1;
    uint64_t* bar_s = bar_q_empty + 1;            // [chains][2] S is complete
    uint64_t* bar_pv = bar_s + 2 * kStreams;      // [chains][2] the product of its P with V is complete
    uint64_t* bar_p = bar_pv + 2 * kStreams;      // [chains][2][2] half of P is written
    uint64_t* bar_end = bar_p + 4 * kStreams;     // products in flight at the end of a CTA that gave up
    __shared__ uint32_t s_tmem;
    __shared__ uint32_t s_stop;
    __shared__ Walk s_walk;

    const int tid = threadIdx.x;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int lane = tid & 31;
    if (tid == 0) {
        s_stop = 0u;
        for (int i = 0; i < L::kSlots; ++i) {
            mbar_init(bar_full + i, 1);
            mbar_init(bar_empty + i, 1);
        }
        mbar_init(bar_q_full, 1);
        mbar_init(bar_q_empty, 1);
        for (int w = 0; w < kStreams; ++w) {
            mbar_init(bar_s + 2 * w, 1);
            mbar_init(bar_s + 2 * w + 1, 1);
            for (int i = 0; i < 4; ++i) {
                mbar_init(bar_p + 4 * w + i, 4);
            }
            mbar_init(bar_pv + 2 * w, 1);
            mbar_init(bar_pv + 2 * w + 1, 1);
        }
        mbar_init(bar_end, 1);
    }
    if (warp == 2) {
        tmem_alloc(&s_tmem, kTmemAll);
    }
    grid_dependency_wait();
    if (warp == 2) {  // after its allocation: the next grid could take tensor memory first, and waits for this one to end
        grid_dependency_release();
    }
    // The line's length, and where this CTA's part of it begins. Entries (sequence, row tile) go in groups of 32, a lane
    // each; all warps count the groups' tiles, the first finds its place among them (1024 sequences of up to 300 rows:
    // 425 us against 436 us with one warp). With one group the first warp does without the others.
    const int heads = static_cast<int>(p.kv_heads);
    const int entries = static_cast<int>(p.batch) * p.row_tiles;
    const int groups = (entries + 31) / 32;
    int* s_groups = reinterpret_cast<int*>(sm + L::kRing);  // before the ring is used
    const auto entry = [&](int e) {
        Walk w{};
        w.b = e / p.row_tiles;
        w.row_tile = e - w.b * p.row_tiles;
        if (e < entries) {
            w.len = static_cast<int>(committed_rows(p, w.b));
            w.valid = static_cast<int>(valid_queries(p, w.b));
        }
        return w;
    };
    const auto tiles_of = [&](int e, const Walk& w) {
        const int each = p.whole_items ? 1 : item_tiles<kKeys>(item_range(p, w.len, w.valid, w.row_tile));
        return e < entries ? each * heads : 0;
    };
    if (groups > 1) {
        for (int group = warp; group < groups; group += L::kThreads / 32) {
            const int e = group * 32 + lane;
            const int sum = __reduce_add_sync(0xffffffffu, tiles_of(e, entry(e)));
            if (lane == 0) {
                s_groups[group] = sum;
            }
        }
        __syncthreads();
    }
    if (warp == 0) {
        Walk w = entry(lane);
        int pieces = tiles_of(lane, w);
        int total = groups > 1 ? 0 : pieces;
        for (int group = lane; groups > 1 && group < groups; group += 32) {
            total += s_groups[group];
        }
        total = __reduce_add_sync(0xffffffffu, total);
        const int set_up = !p.whole_items && total / kSetUpFrom >= static_cast<int>(gridDim.x) ? kSetUp : 0;
        total += set_up * heads * entries;
        const Cuts cuts(total, static_cast<int>(gridDim.x));
        const int begin = cuts.begin(static_cast<int>(blockIdx.x));
        const int end = cuts.begin(static_cast<int>(blockIdx.x) + 1);
        if (lane == 0) {
            s_walk = Walk{};  // a part of the line may be empty
        }
        __syncwarp();
        const auto before_lane = [&](int x) {  // sum over the lanes up to this one
            for (int offset = 1; offset < 32; offset <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, x, offset);
                x += lane >= offset ? other : 0;
            }
            return x;
        };
        int before = 0;
        int e = lane;
        for (int group0 = 0; groups > 1 && group0 < groups; group0 += 32) {  // the group that `begin` lies in
            const int left = entries - (group0 + lane) * 32;                 // entries from the lane's group on
            const int mine = left > 0 ? s_groups[group0 + lane] + set_up * heads * (left < 32 ? left : 32) : 0;
            const int sum = before_lane(mine);
            const unsigned reached = __ballot_sync(0xffffffffu, before + sum > begin);
            if (reached != 0u) {
                const int at_lane = __ffs(reached) - 1;
                before += __shfl_sync(0xffffffffu, sum - mine, at_lane);
                e += (group0 + at_lane) * 32;
                w = entry(e);
                pieces = tiles_of(e, w);
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        pieces += e < entries ? set_up * heads : 0;
        const int lo = before + before_lane(pieces) - pieces;
        if (begin < end && begin >= lo && begin < lo + pieces) {
            const int each = pieces / heads;
            w.h = (begin - lo) / each;
            w.piece = (begin - lo) - w.h * each;
            w.left = end - begin;
            w.set_up = set_up;
            s_walk = w;
            if (!p.whole_items) {
                p.cuts[blockIdx.x] = Cut{w.b, w.row_tile, w.h, w.piece, total, set_up, w.len, w.valid};
            }
        }
        if (blockIdx.x == 0) {
            for (int i = lane; i < p.weight_ctas; i += 32) {
                p.tickets[i] = 0u;
            }
        }
    }
    if (groups > 1) {
        fence_proxy_async_smem();  // the ring's loads come after the counts
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(s_tmem);
    const Waiter wait{p.error, p.poll_limit, &s_stop};
    Walk at = s_walk;
    // The current segment: its item, the item's key tiles, the first and the number of those that it takes, the chains at
    // work (a row tile without valid queries has none).
    ItemRange r{};
    int tiles = 0;
    int tile0 = 0;
    int count = 0;
    int chains = 0;
    const auto segment = [&]() {
        for (;; advance(p, at, tiles)) {
            if (at.left <= 0) {
                return false;
            }
            r = item_range(p, at.len, at.valid, at.row_tile);
            tiles = item_tiles<kKeys>(r);
            tile0 = at.piece > at.set_up ? at.piece - at.set_up : 0;
            const int end = p.whole_items ? tiles : at.piece + at.left - at.set_up;
            count = (end < tiles ? end : tiles) - tile0;
            if (count > 0) {
                break;
            }
        }
        chains = kStreams == 1 ? 1 : kPair ? (r.first + p.tile_tokens < r.valid ? 2 : 1) : (count < 2 ? count : 2);
        return true;
    };
    const auto next = [&]() {
        ++at.index;
        advance(p, at, tiles);
    };
    uint32_t filled = 0;  // a bit for each slot of the ring, then Q: whether it was filled an odd number of times
    if (warp < 4) {
        if (warp == 0) {  // ---- loads
            uint32_t k_tiles[L::kRings] = {};  // loaded so far
            uint32_t v_tiles[L::kRings] = {};
            const auto load = [&](const CUtensorMap* map, int slot, uint32_t n, int tile) {
                if (n >= static_cast<uint32_t>(L::kDepth)) {
                    wait(bar_empty + slot, L::parity(n) ^ 1u);
                }
                if (elect_one() && !wait.stopped()) {
                    filled ^= 1u << slot;
                    mbar_arrive_expect_tx(bar_full + slot, L::kSlot);
                    unsigned char* dst = sm + L::kRing + slot * L::kSlot;
#pragma unroll
                    for (int a = 0; a < L::kAtoms; ++a) {
                        tma_load_4d(dst + a * L::kKvAtom, map, a * 64, at.h, tile * kKeys, at.b, bar_full + slot);
                    }
                }
                __syncwarp();
            };
            // Tile i of the segment; a tile that does not exist is left out.
            const auto load_k = [&](int i) {
                const int ring = i % L::kRings;
                if (i < count) {
                    load(&map_k, L::k_slot(ring, k_tiles[ring]), k_tiles[ring], tile0 + i);
                    ++k_tiles[ring];
                }
            };
            const auto load_v = [&](int i) {
                const int ring = i % L::kRings;
                if (i < count) {
                    load(&map_v, L::v_slot(ring, v_tiles[ring]), v_tiles[ring], tile0 + i);
                    ++v_tiles[ring];
                }
            };
            for (; segment(); next()) {
                if (at.index > 0) {
                    wait(bar_q_empty, static_cast<uint32_t>(at.index - 1) & 1u);
                }
                const int q_tiles = kPair ? chains : 1;
                const uint32_t box = static_cast<uint32_t>(p.q_box_tokens * p.group) * 128u;
                if (elect_one() && !wait.stopped()) {
                    filled ^= 1u << L::kSlots;
                    mbar_arrive_expect_tx(bar_q_full, box * L::kAtoms * q_tiles);
                    for (int i = 0; i < q_tiles; ++i) {
#pragma unroll
                        for (int a = 0; a < L::kAtoms; ++a) {
                            tma_load_4d(sm + L::kQ + (i * L::kAtoms + a) * L::kQAtom, &map_q, a * 64, at.h * p.group,
                                        r.first + i * p.tile_tokens, at.b, bar_q_full);
                        }
                    }
                }
                __syncwarp();
                // In the order in which slots come free: a chain's S lets go of its K tile, its O a step later of its V tile.
                for (int i = 0; i < L::kStep; ++i) {
                    load_k(i);
                }
                for (int i = 0; i < L::kStep; ++i) {
                    load_v(i);
                }
                for (int i = L::kStep; i < 2 * L::kStep; ++i) {
                    load_k(i);
                }
                for (int i = L::kStep; i < count; ++i) {
                    load_v(i);
                    load_k(i + L::kStep);
                }
            }
        } else if (warp == 1) {  // ---- matrix products, the chains in turn
            constexpr uint32_t s_idesc = idesc_bf16_f32(kKeys);
            constexpr uint32_t o_idesc = idesc_bf16_f32_bmn(D);
            uint32_t n0 = 0;  // tiles of the chains before the segment
            uint32_t n1 = 0;
            uint32_t p_phase = 0;  // a bit for each S
            const uint64_t q_desc = uniform(smem_desc_sw128(sm + L::kQ, 0));
            const uint64_t k_desc = uniform(smem_desc_sw128(sm + L::kRing, 0));
            const uint64_t v_desc = uniform(smem_desc_sw128_mn(sm + L::kRing, 0, L::kKvAtom));
            for (; segment(); next()) {
                const int mine0 = kPair ? count : (count + kStreams - 1) / kStreams;  // the chains' key tiles
                const int mine1 = chains < 2 ? 0 : kPair ? count : count / 2;
                wait(bar_q_full, static_cast<uint32_t>(at.index) & 1u);
                // Turn i of a chain: O += P V of its i-th key tile, then S of its tile kAhead further on. The loops stay
                // rolled: the code is run once a tile, and what it takes in the instruction cache the softmax misses.
#pragma unroll 1
                for (int i = -L::kAhead; i < mine0; ++i) {
#pragma unroll 1
                    for (int w = 0; w < chains; ++w) {
                        const int mine = w == 0 ? mine0 : mine1;
                        const int ring = kPair ? 0 : w;
                        const int buffer = (i + L::kAhead) % L::kAhead;
                        const uint32_t tile = (w == 0 ? n0 : n1) + static_cast<uint32_t>(i);
                        const uint32_t t_s = uniform(tmem + w * 128 + buffer * kKeys);
                        const uint32_t t_o = uniform(tmem + L::kTmemO + w * D);
                        if (i >= 0 && i < mine) {
                            const int slot = L::v_slot(ring, tile);
                            const uint64_t v = smem_desc_at(v_desc, uniform(slot * L::kSlot));
                            wait(bar_full + slot, L::parity(tile));
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                wait(bar_p + 4 * w + 2 * buffer + half, p_phase >> (2 * w + buffer) & 1u);
                                tc_fence_after();
                                if (elect_one()) {
#pragma unroll
                                    for (int j = half * (L::kHalf / kUmmaK); j < (half + 1) * (L::kHalf / kUmmaK); ++j) {
                                        umma_bf16_ta(t_o, t_s + j * 8, smem_desc_at(v, j * 2048u), o_idesc,
                                                     (i > 0 || j > 0) ? 1u : 0u);
                                    }
                                    if (half == 1) {
                                        umma_commit(bar_pv + 2 * w + buffer);
                                        if (!kPair || w == chains - 1) {
                                            umma_commit(bar_empty + slot);
                                        }
                                    }
                                }
                                __syncwarp();
                            }
                            p_phase ^= 1u << (2 * w + buffer);
                        }
                        if (i + L::kAhead < mine) {
                            const uint32_t ahead = tile + L::kAhead;
                            const int slot = L::k_slot(ring, ahead);
                            const uint64_t q = smem_desc_at(q_desc, uniform(kPair ? w * L::kAtoms * L::kQAtom : 0u));
                            const uint64_t k = smem_desc_at(k_desc, uniform(slot * L::kSlot));
                            wait(bar_full + slot, L::parity(ahead));
                            tc_fence_after();
                            if (elect_one()) {
#pragma unroll
                                for (int j = 0; j < D / kUmmaK; ++j) {
                                    const uint32_t in = static_cast<uint32_t>(j & 3) * 32u;
                                    umma_bf16(t_s, smem_desc_at(q, (j >> 2) * L::kQAtom + in),
                                              smem_desc_at(k, (j >> 2) * L::kKvAtom + in), s_idesc, j > 0 ? 1u : 0u);
                                }
                                umma_commit(bar_s + 2 * w + buffer);
                                if (!kPair || w == chains - 1) {
                                    umma_commit(bar_empty + slot);
                                }
                                // The segment's last S: no chain has another tile.
                                if (w == 0 ? i + L::kAhead >= mine1 && i + L::kAhead == mine0 - 1 : i + L::kAhead == mine0 - 1) {
                                    umma_commit(bar_q_empty);
                                }
                            }
                            __syncwarp();
                        }
                    }
                }
                n0 += static_cast<uint32_t>(mine0);
                n1 += static_cast<uint32_t>(kPair ? count : mine1);
            }
        }
    } else {  // ---- softmax: chain w, one thread per row
        const int w = (warp - 4) >> 2;
        const int row = tid & 127;
        const int g = row % p.group;
        const int token_in_tile = row / p.group;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lanes + w * 128;
        const uint32_t t_o = tmem + lanes + L::kTmemO + w * D;
        const float c2 = 1.4426950408889634f / sqrtf(static_cast<float>(D));
        int masked = -1;       // the entry whose mask bits the chain has in shared memory
        uint32_t s_phase = 0;  // a bit for each of the chain's two S
        uint32_t n = 0;        // tiles of the chain before the segment
        const auto hand_over = [&](uint64_t* bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar);
            }
        };
        // Waits until the product of a tile, the last one whose S has been taken or the one before it, has reached O.
        // With two S each has a barrier for this: its last phase but one is over, since its S was complete after that.
        const auto settled = [&](int i) {
            wait(bar_pv + 2 * w + i % L::kAhead, (s_phase >> (i % L::kAhead) & 1u) ^ 1u);
            tc_fence_after();
        };
        for (; segment(); next()) {
            const int token0 = r.first + (kPair ? w * p.tile_tokens : 0);
            const int t = token0 + token_in_tile;
            const bool inside = token_in_tile < p.tile_tokens && t < p.tokens;  // a row of ctx
            bf16* ctx = p.ctx + ((at.b * p.tokens + t) * p.q_heads + at.h * p.group + g) * D;
            float* stats = p.stats + ((at.b * p.kv_heads + at.h) * p.tokens + t) * p.group + g;
            if (w >= chains) {  // nothing to do in this segment, but for rows of padding
                if (kPair && inside && tile0 == 0) {
                    for (int c = 0; c < D; c += 16) {
                        st_stream32(ctx + c, U8{});
                    }
                    if (p.stats != nullptr) {
                        *stats = INFINITY;
                    }
                }
                n += kPair ? static_cast<uint32_t>(count) : 0u;
                continue;
            }
            const bool valid = inside && t < r.valid;
            // This row's scores, where they are kept.
            float* scores = p.scores + ((at.b * p.kv_heads + at.h) * p.part_rows + row) * p.score_stride;
            const bool busy = __any_sync(0xffffffffu, inside);
            const int limit = valid ? r.len + t + 1 : 0;
            const int part0 = r.full_end / kKeys * kKeys;  // first key of the first tile in which a key may be hidden
            const bool hides = (tile0 + count) * kKeys > r.full_end;  // the segment has such tiles
            const uint32_t* bits_row = nullptr;
            if (hides) {
                if (row < 16) {
                    s_flags[w * 16 + row] = 0u;
                }
                // The tile's mask rows as bits, the same for all heads of an entry. 1024 sequences of up to 300 rows: 425 us
                // where each item makes them, 370 us.
                if (p.mask != nullptr) {
                    uint32_t* words = s_mask + w * 128 * 9;
                    const int tokens = r.valid - token0 < p.tile_tokens ? r.valid - token0 : p.tile_tokens;
                    const int entry = at.b * p.row_tiles + at.row_tile;
                    const bool made = entry == masked;
                    masked = entry;
                    for (int u = row; u < tokens * 9 && !made; u += 128) {  // a thread makes a word of 32 nodes
                        const int token = u / 9;
                        const int node0 = (u - token * 9) * 32;
                        const uint8_t* mask =
                            p.mask + at.b * p.mask_stride + static_cast<int64_t>(token0 + token) * p.tokens + node0;
                        uint32_t word = 0u;
                        if (node0 < r.valid) {
                            const int last = r.valid - 1 - node0;
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const uint32_t on = mask[i < last ? i : last] != 0 ? 1u : 0u;
                                word |= i <= last ? on << i : 0u;
                            }
                        }
                        words[u] = word;
                    }
                    bits_row = words + (token_in_tile < tokens ? token_in_tile : 0) * 9;
                }
                named_barrier(1 + w, 128);
            }
            float top = -INFINITY;  // the maximum that P is taken against, in units of S
            float sum = 0.0f;
            const int mine = kPair ? count : (count - w + kStreams - 1) / kStreams;  // the chain's key tiles
            for (int i = 0; i < mine; ++i) {
                const uint32_t tile = n + static_cast<uint32_t>(i);
                const int buffer = i % L::kAhead;
                const int key0 = (tile0 + (kPair ? 0 : w) + i * L::kStep) * kKeys;
                const bool partial = key0 + kKeys > r.full_end;
                const uint32_t t_x = t_s + buffer * kKeys;
                wait(bar_s + 2 * w + buffer, s_phase >> buffer & 1u);
                s_phase ^= 1u << buffer;
                tc_fence_after();
                if (partial) {
                    // V rows that nobody sees become zeros, values that are not finite are set aside. S is complete, so
                    // the tile before the last of the chain has been multiplied and the slot's tile before has landed.
                    const int slot = L::v_slot(kPair ? 0 : w, tile);
                    wait(bar_full + slot, L::parity(tile));
                    unsigned char* v = sm + L::kRing + slot * L::kSlot;
                    const int sharing = kPair ? chains : 1;  // chains that read this tile
                    for (int u = (sharing == 2 ? w * 128 : 0) + row; u < kKeys * L::kAtoms; u += 128 * sharing) {
                        const int key = u % kKeys;  // this thread's: 64 dims of a row
                        uint4* at16 = reinterpret_cast<uint4*>(v + u / kKeys * L::kKvAtom + key * 128);
                        if (key0 + key >= r.kv_end) {
#pragma unroll
                            for (int ch = 0; ch < 8; ++ch) {
                                at16[ch ^ (key & 7)] = make_uint4(0u, 0u, 0u, 0u);
                            }
                            continue;
                        }
                        uint32_t bad = 0u;  // sum of 0 * x: not zero where some x is not finite
#pragma unroll
                        for (int ch = 0; ch < 8; ++ch) {
                            const uint4 x = at16[ch ^ (key & 7)];
                            bad = zero_times(x.x, zero_times(x.y, zero_times(x.z, zero_times(x.w, bad))));
                        }
                        if ((bad & 0x7fff7fffu) != 0u) {
                            for (int ch = 0; ch < 8; ++ch) {
                                const uint4 x = at16[ch];
                                at16[ch] = make_uint4(finite_pair(x.x), finite_pair(x.y), finite_pair(x.z),
                                                      finite_pair(x.w));
                            }
                            const int bit = key0 + key - part0;
                            atomicOr(&s_flags[w * 16 + (bit >> 5)], 1u << (bit & 31));
                        }
                    }
                    fence_proxy_async_smem();
                    if (kPair && sharing == 2) {
                        named_barrier(3, 256);
                    }
                }
                float2 offset = make_float2(0.0f, 0.0f);
                float x[L::kHalf];
                if (busy) {
                    // The second half first, for its maximum alone: it is read again for its exponentials, which costs
                    // less than a row of registers. Scores that the row does not see are written back as -inf.
                    tmem_load_begin<L::kHalf>(t_x + L::kHalf, x);
                    tmem_load_end<L::kHalf>(x);
                    if (partial && hide(x, bits_row, key0 + L::kHalf, r.len, limit)) {
                        tmem_store(t_x + L::kHalf, x);
                    }
                    if (!kPair && p.scores != nullptr) {
                        if (valid) {
                            keep(x, scores + key0 + L::kHalf);
                        }
                        __syncwarp();
                    }
                    float new_top = largest(x, top);
                    tmem_load_begin<L::kHalf>(t_x, x);
                    tmem_load_end<L::kHalf>(x);
                    if (partial) {
                        hide(x, bits_row, key0, r.len, limit);
                    }
                    if (!kPair && p.scores != nullptr) {
                        if (valid) {
                            keep(x, scores + key0);
                        }
                        __syncwarp();
                    }
                    new_top = largest(x, new_top);
                    const bool grown = i == 0 || (new_top - top) * c2 > 8.0f;
                    if (i > 0 && __any_sync(0xffffffffu, grown)) {
                        if constexpr (L::kAhead > 1) {
                            settled(i - 1);
                        }
                        const float f = grown ? exp2_approx((top - new_top) * c2) : 1.0f;
                        sum *= f;
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_load16(t_o + c * 16, o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            }
                            tmem_store16(t_o + c * 16, o);
                        }
                    }
                    top = grown ? new_top : top;
                    const float shift = top == -INFINITY ? 0.0f : top * c2;
                    offset = make_float2(-shift, -shift);
                    sum += probabilities(x, make_float2(c2, c2), offset, t_x);
                    tmem_store_wait();
                }
                hand_over(bar_p + 4 * w + 2 * buffer);
                if (busy) {
                    tmem_load_begin<L::kHalf>(t_x + L::kHalf, x);
                    tmem_load_end<L::kHalf>(x);
                    sum += probabilities(x, make_float2(c2, c2), offset, t_x + L::kHalf / 2);
                    tmem_store_wait();
                }
                hand_over(bar_p + 4 * w + 2 * buffer + 1);
            }
            n += static_cast<uint32_t>(mine);
            settled(mine - 1);
            if (hides) {
                named_barrier(1 + w, 128);  // the flags of all the chain's threads
                uint32_t flagged = 0u;
                for (int i = 0; i < 16; ++i) {
                    flagged |= s_flags[w * 16 + i] | (kPair && chains == 2 ? s_flags[(1 - w) * 16 + i] : 0u);
                }
                if (flagged != 0u && busy) {
                    // Values that are not finite, added to the O of the rows that see them by what the product makes of
                    // them, infinity or NaN, with their probability formed again: NaN where it is 0.
                    const float shift = top == -INFINITY ? 0.0f : top * c2;
                    const bf16* q = p.q + ((at.b * p.tokens + t) * p.q_heads + at.h * p.group + g) * D;
                    for (int i = 0; i < 16; ++i) {
                        uint32_t word = s_flags[w * 16 + i] | (kPair && chains == 2 ? s_flags[(1 - w) * 16 + i] : 0u);
                        while (word != 0u) {
                            const int key = part0 + i * 32 + __ffs(word) - 1;
                            word &= word - 1u;
                            const bool seen = valid && (visible_bits(bits_row, key, r.len, limit) & 1u) != 0u;
                            const bf16* k = p.k + at.b * p.ks[0] + key * p.ks[1] + at.h * p.ks[2];
                            const bf16* v = p.v + at.b * p.vs[0] + key * p.vs[1] + at.h * p.vs[2];
                            float s = 0.0f;
#pragma unroll 1
                            for (int c = 0; seen && c < D; ++c) {
                                s = __fmaf_rn(__bfloat162float(q[c]), __bfloat162float(k[c]), s);
                            }
                            const float weight = exp2_approx(__fmaf_rn(s, c2, -shift));
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                __syncwarp();
                                tmem_load16(t_o + c, o);
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                    const float x = __bfloat162float(v[c + j]);
                                    if (seen && !(fabsf(x) < INFINITY)) {
                                        o[j] = __float_as_uint(__fmaf_rn(x, weight, __uint_as_float(o[j])));
                                    }
                                }
                                __syncwarp();
                                tmem_store16(t_o + c, o);
                            }
                            tmem_store_wait();
                        }
                    }
                }
            }
            float scaled_top = top == -INFINITY ? -INFINITY : top * c2;
            const bool whole = count == tiles;
            const bool joins = !kPair && chains == 2;  // the second chain's sums and O are the first's to add
            float f0 = 1.0f;
            float f1 = 0.0f;
            if (joins) {
                if (w == 1) {
                    s_ml[row] = make_float2(scaled_top, sum);
                    tc_fence_before();
                }
                named_barrier(3, 256);
                if (w == 0) {
                    tc_fence_after();
                    const float2 other = s_ml[row];
                    const float most = fmaxf(scaled_top, other.x);
                    f0 = scaled_top == -INFINITY ? 0.0f : exp2_approx(scaled_top - most);
                    f1 = other.x == -INFINITY ? 0.0f : exp2_approx(other.x - most);
                    sum = __fmaf_rn(other.y, f1, sum * f0);
                    scaled_top = most;
                }
            }
            if (busy && !(joins && w == 1)) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int64_t part_row = static_cast<int64_t>(kPair ? w * 128 : 0) + row;
                const int64_t part = 2 * static_cast<int64_t>(blockIdx.x) + (at.index == 0 ? 0 : 1);
                float* part_o = p.part_o + part * D * p.part_rows + part_row * 4;
#pragma unroll 1
                for (int c = 0; c < D; c += 64) {
                    float o[64];
                    tmem_load_begin<64>(t_o + c, o);
                    tmem_load_end<64>(o);
                    if (joins) {
                        float o1[64];
                        tmem_load_begin<64>(t_o + D + c, o1);
                        tmem_load_end<64>(o1);
#pragma unroll
                        for (int j = 0; j < 64; ++j) {
                            o[j] = __fmaf_rn(o1[j], f1, o[j] * f0);
                        }
                    }
                    if (inside && whole) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            U8 x;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                x.r[e] = valid ? pack_bf16x2(o[16 * j + 2 * e] * inv, o[16 * j + 2 * e + 1] * inv) : 0u;
                            }
                            st_stream32(ctx + c + 16 * j, x);
                        }
                    } else if (inside) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            st_v4(part_o + (c + 4 * j) * static_cast<int64_t>(p.part_rows),
                                  make_uint4(__float_as_uint(o[4 * j]), __float_as_uint(o[4 * j + 1]),
                                             __float_as_uint(o[4 * j + 2]), __float_as_uint(o[4 * j + 3])));
                        }
                    }
                    __syncwarp();  // the next tensor-memory load is warp-collective
                }
                if (inside && !whole) {
                    p.part_ml[part * p.part_rows + part_row] = make_float2(scaled_top, sum);
                } else if (inside && p.stats != nullptr) {
                    *stats = valid ? whole_statistic(scaled_top, sum) : INFINITY;
                }
            }
            tc_fence_before();
            if (chains == 2 && (joins || (kPair && hides))) {
                named_barrier(3, 256);  // the second chain's O has been read; both are done with the flags
            } else if (hides) {
                named_barrier(1 + w, 128);
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (s_stop != 0u) {
        if (warp == 0 && elect_one()) {
            wait_landed(bar_full, filled, L::kSlots);
            wait_landed(bar_q_full, filled >> L::kSlots, 1);
        } else if (warp == 1 && elect_one()) {
            wait_products(bar_end);
        }
        __syncthreads();
    }
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemAll);
    }
}

// Joins the parts of the items that a cut of the line went through: block (c, i, j) takes rows 32 i to 32 i + 31 of the
// item that cut c + 1 is the first to go through, a lane a row, and columns 32 kPieces j and on, a warp 4 kPieces of
// them. An item has few parts, and a block takes all its columns; or, where few items have the whole line, over a hundred
// of few rows, which blocks of 32 columns then share (one sequence of 32000 rows and one key-value head: 36.6 -> 28.6
// us; but a batch of 66 rows a head would go from 31.0 to 34.3 us).
template <int D, int kKeys, int kPieces>
__global__ void __launch_bounds__(256) cache_attention_join_kernel(const CacheAttentionParams p, int ctas) {
    constexpr int kColumns = kPieces * 8;  // of four elements, of the block
    __shared__ uint2 s_rows[32][kColumns + 1];
    __shared__ int64_t s_places[32];
    grid_dependency_begin();
    const int cut = static_cast<int>(blockIdx.x) + 1;
    const Cut where = p.cuts[cut];
    const int set_up = where.set_up;
    const Cuts cuts(p.cuts[0].total, ctas);  // a cut at the line's end has no record of its own
    const int first = cuts.begin(cut) - where.piece;  // the item's first piece on the line
    if (cuts.empty(cut) || where.piece <= set_up || cuts.begin(cut - 1) > first + set_up) {
        return;
    }
    const ItemRange r = item_range(p, where.len, where.valid, where.row_tile);
    const int last = cuts.of(first + set_up + item_tiles<kKeys>(r) - 1);  // parts before it are not empty
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int row = static_cast<int>(blockIdx.y) * 32 + lane;
    const int in_tile = row & 127;
    const int64_t t = r.first + (row >> 7) * p.tile_tokens + in_tile / p.group;
    const int g = in_tile % p.group;
    const bool inside = row < p.part_rows && in_tile / p.group < p.tile_tokens && t < p.tokens;
    const bool valid = inside && t < r.valid;
    float top = -INFINITY;
    float sum = 0.0f;
    float o[kPieces][4] = {};
    constexpr int kBatch = kPieces == 1 ? 8 : kPieces == 8 ? 2 : 4;  // parts whose loads are in flight together
    const int64_t column = static_cast<int64_t>(blockIdx.z) * kColumns + warp * kPieces;
    for (int c0 = cut - 1; inside && c0 <= last; c0 += kBatch) {
        float2 ml[kBatch];
        float4 x[kBatch][kPieces];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (c0 + j <= last) {
                const int64_t slot = 2 * static_cast<int64_t>(c0 + j) + (cuts.begin(c0 + j) >= first ? 0 : 1);
                ml[j] = p.part_ml[slot * p.part_rows + row];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    x[j][i] = reinterpret_cast<const float4*>(p.part_o)[(slot * (D / 4) + column + i) * p.part_rows + row];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (c0 + j > last) {
                break;
            }
            const float most = fmaxf(top, ml[j].x);
            const float f0 = top == -INFINITY ? 0.0f : exp2_approx(top - most);
            const float f1 = ml[j].x == -INFINITY ? 0.0f : exp2_approx(ml[j].x - most);
            top = most;
            sum = __fmaf_rn(ml[j].y, f1, sum * f0);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                o[i][0] = __fmaf_rn(x[j][i].x, f1, o[i][0] * f0);
                o[i][1] = __fmaf_rn(x[j][i].y, f1, o[i][1] * f0);
                o[i][2] = __fmaf_rn(x[j][i].z, f1, o[i][2] * f0);
                o[i][3] = __fmaf_rn(x[j][i].w, f1, o[i][3] * f0);
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        s_rows[lane][warp * kPieces + i] =
            valid ? make_uint2(pack_bf16x2(o[i][0] * inv, o[i][1] * inv), pack_bf16x2(o[i][2] * inv, o[i][3] * inv))
                  : make_uint2(0u, 0u);
    }
    if (warp == 0) {
        s_places[lane] =
            inside ? ((where.b * p.tokens + t) * p.q_heads + where.h * p.group + g) * D + blockIdx.z * kColumns * 4 : -1;
        if (inside && blockIdx.z == 0 && p.stats != nullptr) {
            p.stats[((where.b * p.kv_heads + where.h) * p.tokens + t) * p.group + g] =
                valid ? whole_statistic(top, sum) : INFINITY;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * kColumns; i += 256) {
        const int64_t place = s_places[i / kColumns];
        if (place >= 0) {
            reinterpret_cast<uint2*>(p.ctx + place)[i % kColumns] = s_rows[i / kColumns][i % kColumns];
        }
    }
}

// ---- weights --------------------------------------------------------------------------------------------------------

// The weight kernel's tiling: S^T = K Q^T, so that a thread owns a key (a row of the product) and adds its
// probabilities over the queries in registers. A key tile of 128 rows is the A operand and stays in shared memory while
// the sequence's query tiles that see any of it pass through a ring; four warpgroups take turns with the products, each
// with a tensor-memory buffer of its own (2 prompts of 2000 tokens, 16 over 8 heads of 128: 88.3 us the whole call, 91.7
// us with two warpgroups). A product's 16384 exponentials take the special-function unit 1024 cycles, its 128 x 128 x 128
// matrix product 256: the first is the bound, and a product takes about 1100 once the line flows. Exponentials of an
// eighth or a quarter of the pairs by a polynomial on the multiply-add units made the call slower by 4 to 10 us.
template <int D>
struct WeightTiling {
    static constexpr int kAtoms = D / 64;
    static constexpr int kKeySlots = D == 256 ? 1 : 2;
    static constexpr int kSlots = D == 64 ? 8 : D == 128 ? 4 : 2;
    static constexpr int kBuffers = 4;
    static constexpr int kGroups = 4;  // warpgroups that turn products into sums; a group keeps to one buffer
    static constexpr int kThreads = 128 + 128 * kGroups;
    static constexpr uint32_t kAtom = 128 * 128;
    static constexpr uint32_t kTile = kAtom * kAtoms;
    static constexpr uint32_t kK = 0;
    static constexpr uint32_t kRing = kK + kKeySlots * kTile;
    static constexpr uint32_t kStats = kRing + kSlots * kTile;     // [groups][2][128]
    static constexpr uint32_t kSum = kStats + kGroups * 2 * 128 * 4;  // [groups - 1][128] the other groups' sums
    static constexpr uint32_t kBars = kSum + (kGroups - 1) * 128 * 4;
    static constexpr std::size_t kBytes = 1024 + kBars + 256;
    static_assert(kBytes <= 232448, "shared memory of a CTA");
};

// A sequence's key tiles: each has the query tiles from its first visible token's on.
struct KeyRange {
    int len;
    int valid;
    int q_tiles;    // query tiles of the sequence
    int key_tiles;

    __device__ __forceinline__ int first(int kt, const FastDiv& tile_tokens) const {  // query tile that sees key tile kt
        const int past = kt * 128 - len;
        return past > 0 ? static_cast<int>(tile_tokens.quot(static_cast<uint32_t>(past))) : 0;
    }
};

__device__ __forceinline__ KeyRange key_range(const CacheAttentionParams& p, int64_t b) {
    KeyRange r;
    r.len = static_cast<int>(committed_rows(p, b));
    r.valid = static_cast<int>(valid_queries(p, b));
    r.q_tiles = static_cast<int>(p.by_tile_tokens.quot(static_cast<uint32_t>(r.valid + p.tile_tokens - 1)));
    r.key_tiles = r.valid > 0 ? (r.len + r.valid + 127) / 128 : 0;
    return r;
}

// A unit's share of the line: its products, and before them kUnitSetUp pieces without any for what it costs besides
// (loading K, the first statistics, joining the groups' sums). The last key tiles of a prompt are seen by few queries, so
// that CTAs there have many units of few products: the same call 98.1 us without, 89.1 us with 2, 88.1 with 3, 88.4 with 4.
constexpr int kUnitSetUp = 3;

// Pieces of key tiles [kt0, kt0 + 32) of a sequence's head, one tile a lane.
__device__ __forceinline__ int lane_pieces(const CacheAttentionParams& p, const KeyRange& r, int kt0) {
    const int kt = kt0 + static_cast<int>(threadIdx.x & 31);
    return kt < r.key_tiles ? r.q_tiles - r.first(kt, p.by_tile_tokens) + kUnitSetUp : 0;
}

// Pieces of one head of a sequence, by a whole warp.
__device__ __forceinline__ int head_pieces(const CacheAttentionParams& p, const KeyRange& r) {
    int sum = 0;
    for (int kt0 = 0; kt0 < r.key_tiles; kt0 += 32) {
        sum += lane_pieces(p, r, kt0);
    }
    return __reduce_add_sync(0xffffffffu, sum);
}

// The range that another lane of the warp holds.
__device__ __forceinline__ KeyRange from_lane(const KeyRange& r, int lane) {
    KeyRange other;
    other.len = __shfl_sync(0xffffffffu, r.len, lane);
    other.valid = __shfl_sync(0xffffffffu, r.valid, lane);
    other.q_tiles = __shfl_sync(0xffffffffu, r.q_tiles, lane);
    other.key_tiles = __shfl_sync(0xffffffffu, r.key_tiles, lane);
    return other;
}

// The line of pieces is cut like the attention's; a unit is one key tile of one head.
struct UnitWalk {
    int b;
    int kt;
    int h;
    int piece;   // the current unit's first piece that the part has
    int left;
    int begin;   // that piece's place on the line
    int total;
    uint32_t products;  // before the current segment
    int index;
};

template <int D>
__global__ void __launch_bounds__(WeightTiling<D>::kThreads, 1)
    cache_weights_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const CacheAttentionParams p) {
    using L = WeightTiling<D>;
    extern __shared__ __align__(16) unsigned char raw[];
    unsigned char* sm = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    float* s_stats = reinterpret_cast<float*>(sm + L::kStats);
    float* s_sum = reinterpret_cast<float*>(sm + L::kSum);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBars);
    uint64_t* bar_full = bars;                    // [slots] a query tile has landed
    uint64_t* bar_empty = bars + L::kSlots;
    uint64_t* bar_k_full = bars + 2 * L::kSlots;  // [key slots]
    uint64_t* bar_k_empty = bar_k_full + L::kKeySlots;
    uint64_t* bar_s = bar_k_empty + L::kKeySlots;  // [buffers] a product is complete
    uint64_t* bar_free = bar_s + L::kBuffers;      // [buffers] and read
    uint64_t* bar_end = bar_free + L::kBuffers;    // products in flight at the end of a CTA that gave up
    __shared__ uint32_t s_tmem;
    __shared__ uint32_t s_stop;
    __shared__ uint32_t s_last[L::kGroups];
    __shared__ UnitWalk s_walk;

    const int tid = threadIdx.x;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int lane = tid & 31;
    const int columns = p.q_box_tokens * p.group;       // rows of a query tile, columns of the product
    const int chunks = (columns + 31) / 32;             // of 32 columns
    if (tid == 0) {
        s_stop = 0u;
        for (int i = 0; i < L::kSlots; ++i) {
            mbar_init(bar_full + i, 1);
            mbar_init(bar_empty + i, 1);
        }
        for (int i = 0; i < L::kKeySlots; ++i) {
            mbar_init(bar_k_full + i, 1);
            mbar_init(bar_k_empty + i, 1);
        }
        for (int i = 0; i < L::kBuffers; ++i) {
            mbar_init(bar_s + i, 1);
            mbar_init(bar_free + i, 4);
        }
        mbar_init(bar_end, 1);
    }
    if (warp == 2) {
        tmem_alloc(&s_tmem, kTmemAll);
    }
    // Rows of the query slots that no tile fills: zeros, so that their columns are finite and count for nothing.
    for (int i = tid; i < L::kSlots * L::kAtoms * (128 - columns) * 8; i += L::kThreads) {
        const int chunk = i & 7;
        const int row = columns + (i >> 3) % (128 - columns);
        const int atom = (i >> 3) / (128 - columns);
        *reinterpret_cast<uint4*>(sm + L::kRing + atom * L::kAtom + row * 128 + chunk * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    grid_dependency_wait();
    if (warp == 2) {  // after its allocation, as in cache_attention_kernel
        grid_dependency_release();
    }
    if (warp == 0) {
        // Sequences in groups of 32, a lane each; each one's products are then counted by the whole warp.
        const int heads = static_cast<int>(p.kv_heads);
        const int batch = static_cast<int>(p.batch);
        const auto ranges_of = [&](int b0) { return b0 + lane < batch ? key_range(p, b0 + lane) : KeyRange{}; };
        KeyRange mine = ranges_of(0);
        int total = 0;
        for (int b = 0; b < batch; ++b) {
            if (b > 0 && b % 32 == 0) {
                mine = ranges_of(b);
            }
            total += head_pieces(p, from_lane(mine, b % 32)) * heads;
        }
        const Cuts cuts(total, static_cast<int>(gridDim.x));
        const int begin = cuts.begin(static_cast<int>(blockIdx.x));
        const int end = cuts.begin(static_cast<int>(blockIdx.x) + 1);
        UnitWalk w{};
        w.total = total;
        if (begin < end) {
            if (batch > 32) {
                mine = ranges_of(0);
            }
            KeyRange r{};
            int rest = begin;
            for (;; ++w.b) {  // the sequence that `begin` lies in
                if (w.b > 0 && w.b % 32 == 0) {
                    mine = ranges_of(w.b);
                }
                r = from_lane(mine, w.b % 32);
                const int here = head_pieces(p, r) * heads;
                if (rest < here) {
                    break;
                }
                rest -= here;
            }
            for (int kt0 = 0;; kt0 += 32) {  // the key tile; order within a sequence: key tile, head, query tile
                const int here = lane_pieces(p, r, kt0) * heads;
                int sum = here;
                for (int offset = 1; offset < 32; offset <<= 1) {
                    const int other = __shfl_up_sync(0xffffffffu, sum, offset);
                    sum += lane >= offset ? other : 0;
                }
                const unsigned reached = __ballot_sync(0xffffffffu, sum > rest);
                if (reached != 0u) {
                    const int at_lane = __ffs(reached) - 1;
                    w.kt = kt0 + at_lane;
                    rest -= __shfl_sync(0xffffffffu, sum - here, at_lane);
                    break;
                }
                rest -= __shfl_sync(0xffffffffu, sum, 31);
            }
            const int each = r.q_tiles - r.first(w.kt, p.by_tile_tokens) + kUnitSetUp;
            w.h = rest / each;
            w.piece = rest - w.h * each;
            w.left = end - begin;
            w.begin = begin;
        }
        if (lane == 0) {
            s_walk = w;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const Waiter wait{p.error, p.poll_limit, &s_stop};
    UnitWalk at = s_walk;
    KeyRange r = at.left > 0 ? key_range(p, at.b) : KeyRange{};
    // The current segment: its unit's first query tile and their number, the first of those that it takes, counted from
    // the unit's first, and how many.
    int q0 = 0;
    int tiles = 0;
    int tile0 = 0;
    int count = 0;
    const auto advance_unit = [&]() {
        const int rest = tiles + kUnitSetUp - at.piece;
        at.left -= rest;
        at.begin += rest;
        at.piece = 0;
        if (at.left <= 0 || ++at.h < static_cast<int>(p.kv_heads)) {
            return;
        }
        at.h = 0;
        if (++at.kt < r.key_tiles) {
            return;
        }
        at.kt = 0;
        while (++at.b < static_cast<int>(p.batch)) {
            r = key_range(p, at.b);
            if (r.key_tiles > 0) {
                break;
            }
        }
    };
    const auto segment = [&]() {
        for (;; advance_unit()) {
            if (at.left <= 0) {
                return false;
            }
            q0 = r.first(at.kt, p.by_tile_tokens);
            tiles = r.q_tiles - q0;
            tile0 = at.piece > kUnitSetUp ? at.piece - kUnitSetUp : 0;
            const int end = at.piece + at.left - kUnitSetUp;
            count = (end < tiles ? end : tiles) - tile0;
            if (count > 0) {
                return true;
            }
        }
    };
    const auto next = [&]() {
        ++at.index;
        at.products += static_cast<uint32_t>(count);
        advance_unit();
    };

    uint32_t filled = 0;  // a bit for each slot of the ring, then of K: whether it was filled an odd number of times
    if (warp == 0) {
        {  // ---- loads
            for (; segment(); next()) {
                const uint32_t ks = static_cast<uint32_t>(at.index) % L::kKeySlots;
                const uint32_t kr = static_cast<uint32_t>(at.index) / L::kKeySlots;
                if (kr > 0) {
                    wait(bar_k_empty + ks, (kr - 1) & 1u);
                }
                if (elect_one() && !wait.stopped()) {
                    filled ^= 1u << (L::kSlots + ks);
                    mbar_arrive_expect_tx(bar_k_full + ks, L::kTile);
#pragma unroll
                    for (int a = 0; a < L::kAtoms; ++a) {
                        tma_load_4d(sm + L::kK + ks * L::kTile + a * L::kAtom, &map_k, a * 64, at.h, at.kt * 128, at.b,
                                    bar_k_full + ks);
                    }
                }
                __syncwarp();
                for (int i = 0; i < count; ++i) {
                    const uint32_t fill = at.products + static_cast<uint32_t>(i);
                    const uint32_t slot = fill % L::kSlots;
                    if (fill >= static_cast<uint32_t>(L::kSlots)) {
                        wait(bar_empty + slot, (fill / L::kSlots - 1) & 1u);
                    }
                    if (elect_one() && !wait.stopped()) {
                        filled ^= 1u << slot;
                        mbar_arrive_expect_tx(bar_full + slot, static_cast<uint32_t>(columns) * 128u * L::kAtoms);
#pragma unroll
                        for (int a = 0; a < L::kAtoms; ++a) {
                            tma_load_4d(sm + L::kRing + slot * L::kTile + a * L::kAtom, &map_q, a * 64, at.h * p.group,
                                        (q0 + tile0 + i) * p.tile_tokens, at.b, bar_full + slot);
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp == 1) {
        {  // ---- matrix products
            const uint32_t idesc = idesc_bf16_f32(chunks * 32);
            for (; segment(); next()) {
                const uint32_t ks = static_cast<uint32_t>(at.index) % L::kKeySlots;
                wait(bar_k_full + ks, static_cast<uint32_t>(at.index) / L::kKeySlots & 1u);
                for (int i = 0; i < count; ++i) {
                    const uint32_t n = at.products + static_cast<uint32_t>(i);
                    const uint32_t slot = n % L::kSlots;
                    const uint32_t buffer = n % L::kBuffers;
                    if (n >= static_cast<uint32_t>(L::kBuffers)) {
                        wait(bar_free + buffer, (n / L::kBuffers - 1) & 1u);
                    }
                    wait(bar_full + slot, n / L::kSlots & 1u);
                    tc_fence_after();
                    const unsigned char* k = sm + L::kK + ks * L::kTile;
                    const unsigned char* q = sm + L::kRing + slot * L::kTile;
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < D / kUmmaK; ++j) {
                            const uint32_t off = (j >> 2) * L::kAtom + static_cast<uint32_t>(j & 3) * 32u;
                            umma_bf16(tmem + buffer * 128, smem_desc_sw128(k, off), smem_desc_sw128(q, off), idesc,
                                      j > 0 ? 1u : 0u);
                        }
                        umma_commit(bar_s + buffer);
                        umma_commit(bar_empty + slot);
                        if (i == count - 1) {
                            umma_commit(bar_k_empty + ks);
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp >= 4) {  // ---- probabilities: one thread per key, the groups' products in turn
        const int w = (warp - 4) >> 2;
        const int row = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const float c2 = 1.4426950408889634f / sqrtf(static_cast<float>(D));
        uint32_t turn = 0;  // which of the group's two copies of the statistics
        // Starts the copy of a query tile's statistics into the group's next place; infinity for columns that count for
        // nothing.
        const auto fetch = [&](int token0) {
            const int inside = r.valid - token0 < p.tile_tokens ? r.valid - token0 : p.tile_tokens;
            float* to = s_stats + (w * 2 + turn) * 128 + row;
            if (row < inside * p.group) {
                cp_async4(to, p.stats + ((at.b * p.kv_heads + at.h) * p.tokens + token0) * p.group + row);
            } else {
                *to = INFINITY;
            }
        };
        for (; segment(); next()) {
            const int key = at.kt * 128 + row;
            const int first = (w - static_cast<int>(at.products)) & (L::kGroups - 1);  // of the segment's products
            float2 part[2] = {};
            if (first < count) {
                fetch((q0 + tile0 + first) * p.tile_tokens);
            }
            for (int i = first; i < count; i += L::kGroups) {
                const uint32_t n = at.products + static_cast<uint32_t>(i);
                const uint32_t buffer = n % L::kBuffers;
                const int token0 = (q0 + tile0 + i) * p.tile_tokens;
                const int inside = r.valid - token0 < p.tile_tokens ? r.valid - token0 : p.tile_tokens;
                const float* stats = s_stats + (w * 2 + turn) * 128;
                turn ^= 1u;
                cp_async_wait_all();
                named_barrier(1 + w, 128);  // the statistics are there, and nobody reads the ones before
                if (i + L::kGroups < count) {
                    fetch(token0 + L::kGroups * p.tile_tokens);
                }
                wait(bar_s + buffer, n / L::kBuffers & 1u);
                tc_fence_after();
                const bool partial = inside < p.tile_tokens || columns < chunks * 32 || at.kt * 128 + 127 - r.len > token0;
                // A committed key lies up to 2^30 rows before the tile's first query: only a later one is multiplied, by
                // less than two tiles of tokens.
                const int later = key - r.len - token0;
                const int low = later > 0 ? later * p.group : 0;  // columns below do not see the key
                const int high = inside * p.group;                // columns from here on count for nothing
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    float x[32];
                    tmem_load_begin<32>(tmem + lanes + buffer * 128 + c * 32, x);
                    tmem_load_end<32>(x);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 top = *reinterpret_cast<const float4*>(stats + c * 32 + j);
                        float2 e0 = __ffma2_rn(make_float2(x[j], x[j + 1]), make_float2(c2, c2), make_float2(-top.x, -top.y));
                        float2 e1 = __ffma2_rn(make_float2(x[j + 2], x[j + 3]), make_float2(c2, c2),
                                               make_float2(-top.z, -top.w));
                        e0 = make_float2(exp2_approx(e0.x), exp2_approx(e0.y));
                        e1 = make_float2(exp2_approx(e1.x), exp2_approx(e1.y));
                        if (partial) {
                            const int column = c * 32 + j;
                            e0.x = column >= low && column < high ? e0.x : 0.0f;
                            e0.y = column + 1 >= low && column + 1 < high ? e0.y : 0.0f;
                            e1.x = column + 2 >= low && column + 2 < high ? e1.x : 0.0f;
                            e1.y = column + 3 >= low && column + 3 < high ? e1.y : 0.0f;
                        }
                        part[0] = __fadd2_rn(part[0], e0);
                        part[1] = __fadd2_rn(part[1], e1);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar_free + buffer);
                }
            }
            float sum = (part[0].x + part[0].y) + (part[1].x + part[1].y);
            bool writes = first < count;
            if (count > 1) {  // several groups had products of the unit: they hand their sums to the first
                if (w > 0) {
                    s_sum[(w - 1) * 128 + row] = sum;
                }
                named_barrier(1 + L::kGroups, 128 * L::kGroups);
                for (int other = 0; w == 0 && other < L::kGroups - 1; ++other) {
                    sum += s_sum[other * 128 + row];
                }
                writes = w == 0;
                named_barrier(1 + L::kGroups, 128 * L::kGroups);
            }
            if (writes) {
                const bool seen = key < r.len + r.valid;
                float* out = p.weights + (at.b * p.kv_heads + at.h) * p.capacity + key;
                if (count == tiles) {
                    if (seen) {
                        *out += sum;
                    }
                } else {
                    // A cut went through the unit: whoever leaves the last of its parts adds them up in their order.
                    const int first = at.begin - at.piece;
                    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (at.index == 0 ? 0 : 1);
                    p.part_sums[slot * 128 + row] = sum;
                    const Cuts cuts(at.total, static_cast<int>(gridDim.x));
                    const int c0 = cuts.of(first + kUnitSetUp);
                    const int c1 = cuts.of(first + kUnitSetUp + tiles - 1);  // parts between them are not empty
                    __threadfence();
                    named_barrier(1 + w, 128);
                    if (row == 0) {
                        s_last[w] = atomicAdd(p.tickets + c0, 1u) == static_cast<unsigned>(c1 - c0) ? 1u : 0u;
                    }
                    named_barrier(1 + w, 128);
                    if (s_last[w] != 0u) {
                        __threadfence();
                        float all = 0.0f;
                        for (int c = c0; c <= c1; ++c) {
                            all += __ldcg(p.part_sums + (2 * int64_t{c} + (cuts.begin(c) >= first ? 0 : 1)) * 128 + row);
                        }
                        if (seen) {
                            *out += all;
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (s_stop != 0u) {
        if (warp == 0 && elect_one()) {
            wait_landed(bar_full, filled, L::kSlots);
            wait_landed(bar_k_full, filled >> L::kSlots, L::kKeySlots);
        } else if (warp == 1 && elect_one()) {
            wait_products(bar_end);
        }
        __syncthreads();
    }
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemAll);
    }
}

// The weights from kept scores: a thread takes four keys of a head and adds their probabilities over the head's rows.
// Scores that a row does not see were kept as -inf.
__global__ void __launch_bounds__(256) cache_weights_kept_kernel(const CacheAttentionParams p, float c2) {
    __shared__ float s_stats[kMaxKeptRows];
    grid_dependency_begin();
    const unsigned blocks = static_cast<unsigned>((p.capacity + 1023) / 1024);  // of a head
    const int64_t head = blockIdx.x / blocks;                                     // of all sequences
    const int block = static_cast<int>(blockIdx.x % blocks);
    const int64_t b = head / p.kv_heads;
    const int valid = static_cast<int>(valid_queries(p, b));
    const int end = valid > 0 ? static_cast<int>(committed_rows(p, b)) + valid : 0;
    const int key = (block * 256 + static_cast<int>(threadIdx.x)) * 4;
    const int rows = valid * p.group;
    if (block * 1024 >= end) {
        return;
    }
    if (static_cast<int>(threadIdx.x) < rows) {
        s_stats[threadIdx.x] = p.stats[head * p.tokens * p.group + threadIdx.x];
    }
    __syncthreads();
    float sum[4] = {};
    if (key < end) {
        const float* scores = p.scores + head * p.part_rows * p.score_stride + key;
#pragma unroll 4
        for (int i = 0; i < rows; ++i) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(scores + i * p.score_stride));
            const float st = s_stats[i];
            sum[0] += exp2_approx(__fmaf_rn(x.x, c2, -st));
            sum[1] += exp2_approx(__fmaf_rn(x.y, c2, -st));
            sum[2] += exp2_approx(__fmaf_rn(x.z, c2, -st));
            sum[3] += exp2_approx(__fmaf_rn(x.w, c2, -st));
        }
    }
    float* out = p.weights + head * p.capacity + key;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (key + j < end) {
            out[j] += sum[j];
        }
    }
}

// The tiling of a call, and where its scratch lies (offsets in bytes; `bytes` in all).
struct Plan {
    bool fits;         // the lines' lengths stay below 2^31
    bool pair;         // two row tiles on each K and V tile
    bool whole_items;  // no item has enough key tiles to be cut
    int ctas;
    int tile_tokens;
    int item_tokens;
    int row_tiles;
    int part_rows;
    int64_t ml;
    int64_t o;
    int64_t stats;
    int64_t sums;
    int64_t scores;
    int64_t score_stride;  // 0: K Q^T is formed again for the weights
    int64_t bytes;
    int weight_ctas;
};

Plan plan(int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t capacity,
          bool with_stats) {
    Plan pl{};
    const int64_t group = q_heads / kv_heads;
    const int64_t keys = head_dim == 256 ? 64 : 128;
    pl.tile_tokens = static_cast<int>(kBM / group);
    pl.pair = head_dim != 256 && tokens > pl.tile_tokens;
    pl.item_tokens = pl.tile_tokens * (pl.pair ? 2 : 1);
    pl.row_tiles = static_cast<int>(runtime::ceil_div(tokens, pl.item_tokens));
    pl.part_rows = pl.pair ? 2 * kBM : static_cast<int>((tokens < pl.tile_tokens ? tokens : pl.tile_tokens) * group);
    const int64_t most = batch * pl.row_tiles * kv_heads * runtime::ceil_div(capacity, keys);  // tiles of the line
    // Items of few key tiles are not cut (a piece of the line is then an item): nothing is left to join, which one
    // sequence of 600 rows gains by (11.6 us against 13.0 us cut) and one of 1000 no longer (13.9 against 10.8). Where
    // there are many items of one length of tokens, longer ones too: 16 sequences of up to 1000 rows 15.4 against 22.8,
    // of up to 1900 rows 22.4 against 25.2.
    const int64_t items = batch * pl.row_tiles * kv_heads;
    const int64_t tiles = runtime::ceil_div(capacity, keys);
    pl.whole_items = tiles <= 6 || (tiles <= 16 && pl.row_tiles == 1 && items >= runtime::sm_count() / 2);
    // A CTA whose two chains share a row tile is given two key tiles at least.
    const int64_t pieces = pl.whole_items ? items : pl.pair || head_dim == 256 ? most : (most + 1) / 2;
    pl.ctas = static_cast<int>(pieces < runtime::sm_count() ? pieces : runtime::sm_count());
    const int64_t products = batch * kv_heads * runtime::ceil_div(capacity, 128) * runtime::ceil_div(tokens, pl.tile_tokens);
    // A line has up to four pieces for each tile or product, its set-up's and itself.
    pl.fits = batch * pl.row_tiles <= kMostEntries && most * (kSetUp + 1) < (int64_t{1} << 31) && products * (kUnitSetUp + 1) < (int64_t{1} << 31);
    const auto up = [](int64_t n) { return (n + 127) / 128 * 128; };
    const int64_t parts = pl.whole_items ? 0 : 2 * pl.ctas;
    pl.ml = pl.whole_items ? 0 : up(pl.ctas * static_cast<int64_t>(sizeof(Cut)));
    pl.o = pl.ml + up(parts * pl.part_rows * static_cast<int64_t>(sizeof(float2)));
    pl.stats = pl.o + parts * pl.part_rows * head_dim * static_cast<int64_t>(sizeof(float));
    pl.bytes = pl.stats;
    if (with_stats) {
        pl.sums = pl.stats + up(batch * tokens * q_heads * static_cast<int64_t>(sizeof(float)));
        // Keeping a key's scores for the weights moves 8 bytes for each row, mostly within L2; forming them again reads
        // the key's 2 * head_dim bytes of K from memory and takes a tile's products. Eight sequences of 16000 rows, 8
        // heads of 128: 106 against 162 us with 2 rows, 125 against 163 with 16, 149 against 164 with 32, 223 against
        // 166 with 64. Scores go by the capacity, not by the lengths: past kMostScoreBytes they are kept only where they
        // take a sixteenth of K and V at most, so that the call needs little memory beside its caches. 32 sequences of 8
        // heads of 128: 1054 us kept and 1063 us formed again with 32 rows (33000 cached, 1.01 GB of scores), 1685 and 2103
        // with 16 (65500, 1.00 GB), 1546 and 2101 with 8, which stay kept.
        const int64_t stride = runtime::ceil_div(capacity, 128) * 128;
        const int64_t score_bytes = batch * kv_heads * pl.part_rows * stride * static_cast<int64_t>(sizeof(float));
        const bool few = score_bytes <= kMostScoreBytes || tokens * group * 16 <= head_dim;
        if (tokens * group <= kMaxKeptRows && few) {
            pl.score_stride = stride;
            pl.scores = pl.sums;
            pl.bytes = pl.scores + score_bytes;
            return pl;
        }
        pl.weight_ctas = static_cast<int>(products < runtime::sm_count() ? products : runtime::sm_count());
        // The parts of the units, then the tickets.
        pl.bytes = pl.sums + up(pl.weight_ctas * static_cast<int64_t>(2 * 128 * sizeof(float) + sizeof(unsigned int)));
    }
    return pl;
}

bool encode_4d(CUtensorMap* map, const void* base, const int64_t (&dims)[4], const int64_t (&strides)[3],
               const int (&box)[4]) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) {
        return false;
    }
    cuuint64_t d[4];
    cuuint64_t s[3];
    cuuint32_t b[4];
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    for (int i = 0; i < 4; ++i) {
        d[i] = static_cast<cuuint64_t>(dims[i]);
        b[i] = static_cast<cuuint32_t>(box[i]);
    }
    for (int i = 0; i < 3; ++i) {
        s[i] = static_cast<cuuint64_t>(strides[i]) * 2;
    }
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), d, s, b, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kPair>
cudaError_t launch_cache_attention(const CacheAttentionParams& p, const Plan& pl, cudaStream_t s) {
    using L = Tiling<D, kPair>;
    CUtensorMap mq{};
    CUtensorMap mk{};
    CUtensorMap mv{};
    if (!encode_4d(&mq, p.q, {D, p.q_heads, p.tokens, p.batch}, {D, p.q_heads * D, p.tokens * p.q_heads * D},
                   {64, p.group, p.q_box_tokens, 1}) ||
        !encode_4d(&mk, p.k, {D, p.kv_heads, p.capacity, p.batch}, {p.ks[2], p.ks[1], p.ks[0]}, {64, 1, L::kKeys, 1}) ||
        !encode_4d(&mv, p.v, {D, p.kv_heads, p.capacity, p.batch}, {p.vs[2], p.vs[1], p.vs[0]}, {64, 1, L::kKeys, 1})) {
        return cudaErrorInvalidValue;
    }
    static runtime::SharedMemoryLimit limit;
    cudaError_t err = limit.raise(cache_attention_kernel<D, kPair>, L::kBytes);
    if (err != cudaSuccess) {
        return err;
    }
    err = runtime::launch_smem(cache_attention_kernel<D, kPair>, dim3(static_cast<unsigned>(pl.ctas)),
                               dim3(L::kThreads), L::kBytes, s, 1u, mq, mk, mv, p);
    if (err != cudaSuccess || pl.ctas == 1 || pl.whole_items) {
        return err;
    }
    runtime::count_launches(1);
    const bool shared = pl.part_rows <= 32 && pl.ctas > 4 * p.batch * p.row_tiles * p.kv_heads;
    return runtime::launch(shared ? cache_attention_join_kernel<D, L::kKeys, 1>
                                  : cache_attention_join_kernel<D, L::kKeys, D / 32>,
                           dim3(static_cast<unsigned>(pl.ctas - 1), (static_cast<unsigned>(p.part_rows) + 31) / 32,
                                shared ? D / 32 : 1),
                           dim3(256), s, 1u, p, pl.ctas);
}

template <int D>
cudaError_t launch_cache_weights(const CacheAttentionParams& p, cudaStream_t s) {
    using L = WeightTiling<D>;
    CUtensorMap mq{};
    CUtensorMap mk{};
    if (!encode_4d(&mq, p.q, {D, p.q_heads, p.tokens, p.batch}, {D, p.q_heads * D, p.tokens * p.q_heads * D},
                   {64, p.group, p.q_box_tokens, 1}) ||
        !encode_4d(&mk, p.k, {D, p.kv_heads, p.capacity, p.batch}, {p.ks[2], p.ks[1], p.ks[0]}, {64, 1, 128, 1})) {
        return cudaErrorInvalidValue;
    }
    static runtime::SharedMemoryLimit limit;
    const cudaError_t err = limit.raise(cache_weights_kernel<D>, L::kBytes);
    if (err != cudaSuccess) {
        return err;
    }
    return runtime::launch_smem(cache_weights_kernel<D>, dim3(static_cast<unsigned>(p.weight_ctas)), dim3(L::kThreads),
                                L::kBytes, s, 1u, mq, mk, p);
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
    CPPINF_REQUIRE(capacity < kMost / 2 && q_heads < (1 << 16) && batch < (1 << 24) && tokens < kMost &&
                       (batch == 0 || tokens == 0 || tokens * q_heads < kMost / batch) &&
                       (batch == 0 || capacity == 0 || kv_heads < kMost * 4 / (batch * capacity)),
                   CPPINF_ERR_OVERFLOW, name + " sizes exceed the kernels' index range.");
    return CPPINF_OK;
}

int check_cache(const char* op, const void* cache, const int64_t* strides, int64_t capacity) {
    const std::string name(op);
    CPPINF_REQUIRE((cache || capacity == 0) && strides, CPPINF_ERR_INVALID_ARGUMENT, name + " received a null pointer.");
    for (int i = 0; i < 3; ++i) {
        CPPINF_REQUIRE(strides[i] > 0, CPPINF_ERR_INVALID_ARGUMENT, name + " requires positive cache strides.");
        CPPINF_REQUIRE(strides[i] % 8 == 0 && strides[i] < (int64_t{1} << 38), CPPINF_ERR_UNSUPPORTED,
                       name + " requires cache strides in multiples of 8 elements, below 2^38.");
    }
    CPPINF_REQUIRE(runtime::aligned16(cache), CPPINF_ERR_UNSUPPORTED, name + " requires 16-byte aligned caches.");
    return CPPINF_OK;
}

int run_attention(const char* op, CacheAttentionParams& p, int64_t head_dim, void* scratch, int64_t scratch_bytes,
                  cudaStream_t s) {
    if (p.capacity == 0) {  // no rows: every query is padding
        const auto bytes = static_cast<std::size_t>(p.batch * p.tokens * p.q_heads * head_dim) * sizeof(bf16);
        CPPINF_CUDA_TRY(cudaMemsetAsync(p.ctx, 0, bytes, s));
        return runtime::ok();
    }
    const std::string name(op);
    const Plan pl = plan(p.batch, p.tokens, p.q_heads, p.kv_heads, head_dim, p.capacity, p.weights != nullptr);
    CPPINF_REQUIRE(pl.fits, CPPINF_ERR_OVERFLOW, name + " sizes exceed the kernels' index range.");
    CPPINF_REQUIRE((scratch || pl.bytes == 0) && scratch_bytes >= pl.bytes, CPPINF_ERR_INVALID_ARGUMENT,
                   name + " requires a scratch of cppinf_cache_attention_scratch_bytes.");
    CPPINF_REQUIRE(runtime::aligned16(scratch), CPPINF_ERR_UNSUPPORTED, name + " requires a 16-byte aligned scratch.");
    char* base = static_cast<char*>(scratch);
    p.group = static_cast<int>(p.q_heads / p.kv_heads);
    p.tile_tokens = pl.tile_tokens;
    p.by_tile_tokens = FastDiv(static_cast<uint32_t>(pl.tile_tokens));
    p.item_tokens = pl.item_tokens;
    p.row_tiles = pl.row_tiles;
    p.q_box_tokens = static_cast<int>(p.tokens < pl.tile_tokens ? p.tokens : pl.tile_tokens);
    p.whole_items = pl.whole_items;
    p.part_rows = pl.part_rows;
    p.cuts = reinterpret_cast<Cut*>(base);
    p.part_ml = reinterpret_cast<float2*>(base + pl.ml);
    p.part_o = reinterpret_cast<float*>(base + pl.o);
    if (p.weights != nullptr) {
        p.stats = reinterpret_cast<float*>(base + pl.stats);
        p.scores = pl.score_stride > 0 ? reinterpret_cast<float*>(base + pl.scores) : nullptr;
        p.score_stride = pl.score_stride;
        p.weight_ctas = pl.weight_ctas;
        p.part_sums = reinterpret_cast<float*>(base + pl.sums);
        p.tickets = reinterpret_cast<unsigned int*>(p.part_sums + pl.weight_ctas * 2 * 128);
    }
    p.poll_limit = runtime::wait_poll_limit();
    cudaError_t err = cudaSuccess;
    if (head_dim == 64) {
        err = pl.pair ? launch_cache_attention<64, true>(p, pl, s) : launch_cache_attention<64, false>(p, pl, s);
    } else if (head_dim == 128) {
        err = pl.pair ? launch_cache_attention<128, true>(p, pl, s) : launch_cache_attention<128, false>(p, pl, s);
    } else {
        err = launch_cache_attention<256, false>(p, pl, s);
    }
    return runtime::launched(err, op);
}

int run_weights(const char* op, const CacheAttentionParams& p, int64_t head_dim, cudaStream_t s) {
    if (p.scores != nullptr) {
        const float c2 = 1.4426950408889634f / std::sqrt(static_cast<float>(head_dim));
        return runtime::launched(runtime::launch(cache_weights_kept_kernel,
                                                 dim3(static_cast<unsigned>(runtime::ceil_div(p.capacity, 1024) *
                                                                            p.batch * p.kv_heads)),
                                                 dim3(256), s, 1u, p, c2),
                                 op);
    }
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
    if (batch == 0 || tokens == 0) {
        return 0;
    }
    const Plan pl = plan(batch, tokens, q_heads, kv_heads, head_dim, capacity, with_weights != 0);
    return pl.fits ? pl.bytes : -1;
}

int cppinf_tree_attention(const void* q, const void* k_cache, const int64_t* k_strides, const void* v_cache,
                          const int64_t* v_strides, const int64_t* lengths, const uint8_t* mask,
                          int64_t mask_batch_stride, const int64_t* nodes, void* ctx, int64_t batch, int64_t tokens,
                          int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t capacity, void* scratch,
                          int64_t scratch_bytes, unsigned int* error, void* stream) {
    constexpr const char* kOp = "tree_attention";
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
    if (const int st = check_cache(kOp, k_cache, k_strides, capacity); st != CPPINF_OK) {
        return st;
    }
    if (const int st = check_cache(kOp, v_cache, v_strides, capacity); st != CPPINF_OK) {
        return st;
    }
    CPPINF_REQUIRE(rt::aligned16(q) && (reinterpret_cast<std::uintptr_t>(ctx) & 31u) == 0, CPPINF_ERR_UNSUPPORTED,
                   "tree_attention requires 16-byte aligned queries and 32-byte aligned contexts.");
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
    p.error = error;
    return run_attention(kOp, p, head_dim, scratch, scratch_bytes, rt::as_stream(stream));
}

int cppinf_decoder_attention_weights(const void* q, const void* k_cache, const int64_t* k_strides, const void* v_cache,
                                     const int64_t* v_strides, const int64_t* lengths, const int64_t* counts, void* ctx,
                                     float* weights, int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                                     int64_t head_dim, int64_t capacity, void* scratch, int64_t scratch_bytes,
                                     unsigned int* error, void* stream) {
    constexpr const char* kOp = "decoder_attention_weights";
    if (const int st = check_sizes(kOp, batch, tokens, q_heads, kv_heads, head_dim, capacity); st != CPPINF_OK) {
        return st;
    }
    if (batch == 0 || tokens == 0) {
        return rt::ok();
    }
    CPPINF_REQUIRE(q && lengths && ctx && (weights || capacity == 0), CPPINF_ERR_INVALID_ARGUMENT,
                   "decoder_attention_weights received a null pointer.");
    if (const int st = check_cache(kOp, k_cache, k_strides, capacity); st != CPPINF_OK) {
        return st;
    }
    if (const int st = check_cache(kOp, v_cache, v_strides, capacity); st != CPPINF_OK) {
        return st;
    }
    CPPINF_REQUIRE(rt::aligned16(q) && (reinterpret_cast<std::uintptr_t>(ctx) & 31u) == 0, CPPINF_ERR_UNSUPPORTED,
                   "decoder_attention_weights requires 16-byte aligned queries and 32-byte aligned contexts.");
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
    p.error = error;
    p.weights = weights;
    p.batch = batch;
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.capacity = capacity;
    if (const int st = run_attention(kOp, p, head_dim, scratch, scratch_bytes, rt::as_stream(stream));
        st != CPPINF_OK || capacity == 0) {
        return st;
    }
    return run_weights(kOp, p, head_dim, rt::as_stream(stream));
}

}  // extern "C"
