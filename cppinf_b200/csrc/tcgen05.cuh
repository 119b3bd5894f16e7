// tcgen05 / TMA building blocks shared by the tensor-core kernels (gemm_tc.cu, attention_tc.cu): 2-D and 3-D TMA
// tile loads, tensor-memory allocation, the bf16 UMMA with its commit, 32-column tensor-memory loads, and the
// shared-memory and instruction descriptors of K-major tiles written by TMA with the 128-byte swizzle.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace cppinf::device::tc {

constexpr int kBM = 128;  // UMMA rows = tensor-memory lanes
constexpr int kBK = 64;   // one 128-byte swizzle row of bf16
constexpr int kUmmaK = 16;

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t* dst_smem, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst_smem)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}

__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T, both K-major; `accumulate` = 0 overwrites D.
__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrives once on `bar` when every tcgen05.mma this thread issued before has completed.
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

// 32 consecutive f32 columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_load32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        v[i] = __uint_as_float(r[i]);
    }
}

// Shared-memory matrix descriptor of a K-major tile written by TMA with the 128-byte swizzle: rows of 64 bf16
// (128 bytes), 8-row groups 1024 bytes apart (stride byte offset), layout type 2 (SWIZZLE_128B) in bits 61-63,
// descriptor version 1 in bits 46-47. The leading byte offset is not used by swizzled K-major layouts. Moving along
// K inside the 128-byte row adds the byte offset to the start address (the swizzle is a function of the address
// bits, and every tile starts 1024-byte aligned).
__device__ __forceinline__ uint64_t smem_desc_sw128(const void* tile, uint32_t k_byte_offset) {
    const uint32_t addr = smem_addr(tile) + k_byte_offset;
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr >> 4) & 0x3fffu);       // start address, bits 0-13
    d |= static_cast<uint64_t>(1u) << 16;                     // leading byte offset (unused), bits 16-29
    d |= static_cast<uint64_t>((1024u >> 4) & 0x3fffu) << 32;  // stride byte offset, bits 32-45
    d |= static_cast<uint64_t>(1u) << 46;                     // version, bits 46-47
    d |= static_cast<uint64_t>(2u) << 61;                     // SWIZZLE_128B, bits 61-63
    return d;
}

// A descriptor `bytes` (a multiple of 16) further on: the start address lies below 2^18 and leaves its field's upper bits
// free, so only the lower word changes.
__device__ __forceinline__ uint64_t smem_desc_at(uint64_t desc, uint32_t bytes) {
    return (desc & 0xffffffff00000000ull) | (static_cast<uint32_t>(desc) + (bytes >> 4));
}

// A value that is the same in all lanes of a converged warp, said so that the compiler knows it: it can then live in a
// uniform register, where the tcgen05 instructions take their operands from.
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
    return __shfl_sync(0xffffffffu, x, 0);
}

__device__ __forceinline__ uint64_t uniform(uint64_t x) {
    return static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32 | uniform(static_cast<uint32_t>(x));
}

// Instruction descriptor of kind::f16 with bf16 A and B, f32 D, both K-major, M = 128, N = n:
// D format bits 4-5 (1 = f32), A format bits 7-9 and B format bits 10-12 (1 = bf16), N >> 3 in bits 17-22,
// M >> 4 in bits 24-28.
__host__ __device__ constexpr uint32_t idesc_bf16_f32(int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((static_cast<uint32_t>(n) >> 3) << 17) |
           ((static_cast<uint32_t>(kBM) >> 4) << 24);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
        : "memory");
}

// umma_bf16 with A in tensor memory: 128 lanes of packed bf16 pairs, 8 columns for each 16 of K.
__device__ __forceinline__ void umma_bf16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 16 consecutive columns of this thread's tensor-memory lane, as bits.
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// N consecutive f32 columns of this thread's tensor-memory lane: the load, and the wait after which (and only then) its
// registers may be read. The wait covers all loads that the thread has begun.
template <int N>
__device__ __forceinline__ void tmem_load_begin(uint32_t taddr, float (&x)[N]);
template <int N>
__device__ __forceinline__ void tmem_load_end(float (&x)[N]);

template <>
__device__ __forceinline__ void tmem_load_begin<32>(uint32_t taddr, float (&x)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, "
        "%31}, [%32];"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]),
          "=f"(x[8]), "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15]),
          "=f"(x[16]), "=f"(x[17]), "=f"(x[18]), "=f"(x[19]), "=f"(x[20]), "=f"(x[21]), "=f"(x[22]),
          "=f"(x[23]), "=f"(x[24]), "=f"(x[25]), "=f"(x[26]), "=f"(x[27]), "=f"(x[28]), "=f"(x[29]),
          "=f"(x[30]), "=f"(x[31])
        : "r"(taddr));
}

template <>
__device__ __forceinline__ void tmem_load_end<32>(float (&x)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]),
                   "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]),
                   "+f"(x[14]), "+f"(x[15]), "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]),
                   "+f"(x[21]), "+f"(x[22]), "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]),
                   "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31])
                 :
                 : "memory");
}

template <>
__device__ __forceinline__ void tmem_load_begin<64>(uint32_t taddr, float (&x)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, "
        "%51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]),
          "=f"(x[8]), "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15]),
          "=f"(x[16]), "=f"(x[17]), "=f"(x[18]), "=f"(x[19]), "=f"(x[20]), "=f"(x[21]), "=f"(x[22]),
          "=f"(x[23]), "=f"(x[24]), "=f"(x[25]), "=f"(x[26]), "=f"(x[27]), "=f"(x[28]), "=f"(x[29]),
          "=f"(x[30]), "=f"(x[31]), "=f"(x[32]), "=f"(x[33]), "=f"(x[34]), "=f"(x[35]), "=f"(x[36]),
          "=f"(x[37]), "=f"(x[38]), "=f"(x[39]), "=f"(x[40]), "=f"(x[41]), "=f"(x[42]), "=f"(x[43]),
          "=f"(x[44]), "=f"(x[45]), "=f"(x[46]), "=f"(x[47]), "=f"(x[48]), "=f"(x[49]), "=f"(x[50]),
          "=f"(x[51]), "=f"(x[52]), "=f"(x[53]), "=f"(x[54]), "=f"(x[55]), "=f"(x[56]), "=f"(x[57]),
          "=f"(x[58]), "=f"(x[59]), "=f"(x[60]), "=f"(x[61]), "=f"(x[62]), "=f"(x[63])
        : "r"(taddr));
}

template <>
__device__ __forceinline__ void tmem_load_end<64>(float (&x)[64]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]),
                   "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]),
                   "+f"(x[14]), "+f"(x[15]), "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]),
                   "+f"(x[21]), "+f"(x[22]), "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]),
                   "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31]), "+f"(x[32]), "+f"(x[33]), "+f"(x[34]),
                   "+f"(x[35]), "+f"(x[36]), "+f"(x[37]), "+f"(x[38]), "+f"(x[39]), "+f"(x[40]), "+f"(x[41]),
                   "+f"(x[42]), "+f"(x[43]), "+f"(x[44]), "+f"(x[45]), "+f"(x[46]), "+f"(x[47]), "+f"(x[48]),
                   "+f"(x[49]), "+f"(x[50]), "+f"(x[51]), "+f"(x[52]), "+f"(x[53]), "+f"(x[54]), "+f"(x[55]),
                   "+f"(x[56]), "+f"(x[57]), "+f"(x[58]), "+f"(x[59]), "+f"(x[60]), "+f"(x[61]), "+f"(x[62]),
                   "+f"(x[63])
                 :
                 : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Stores 16 consecutive columns of this thread's tensor-memory lane; tmem_store_wait() completes the thread's stores.
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_store_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Descriptor of the same kind of tile read with its 64-element rows along M or N (MN-major): a TMA tile [k][64] of
// 128-byte rows holds one 64-wide block of the operand, 8 rows of k lie 1024 bytes apart (stride byte offset), the next
// 64-wide block `block_bytes` on (leading byte offset). 16 rows of k further on is 2048 bytes on.
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(const void* tile, uint32_t k_byte_offset, uint32_t block_bytes) {
    const uint32_t addr = smem_addr(tile) + k_byte_offset;
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr >> 4) & 0x3fffu);
    d |= static_cast<uint64_t>((block_bytes >> 4) & 0x3fffu) << 16;
    d |= static_cast<uint64_t>((1024u >> 4) & 0x3fffu) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// idesc_bf16_f32 with B MN-major (bit 16).
__host__ __device__ constexpr uint32_t idesc_bf16_f32_bmn(int n) {
    return idesc_bf16_f32(n) | (1u << 16);
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Barrier `id` (1..15) of `threads` threads of the block.
__device__ __forceinline__ void named_barrier(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// True in one lane of a converged warp. Code that issues tcgen05 and TMA instructions goes in warps that stay together
// and has one lane picked for the instructions alone: their descriptors then stay in the warp's uniform registers, where
// the instructions take them from, instead of being moved there for each of them.
__device__ __forceinline__ bool elect_one() {
    uint32_t picked;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(picked));
    return picked != 0u;
}

// 2^x of the hardware, within 2 ulp; results below 2^-126 become 0.
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Makes this thread's generic-proxy shared-memory writes visible to the async proxy (tcgen05.mma operands).
__device__ __forceinline__ void fence_proxy_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---- host side ----------------------------------------------------------------------------------------------

using EncodeTiled = PFN_cuTensorMapEncodeTiled_v12000;

// cuTensorMapEncodeTiled from the driver, looked up once through the runtime (no link against libcuda).
inline EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            return static_cast<EncodeTiled>(nullptr);
        }
        return reinterpret_cast<EncodeTiled>(ptr);
    }();
    return fn;
}

}  // namespace cppinf::device::tc
