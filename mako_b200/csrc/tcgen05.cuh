// Thin wrappers over the fifth-generation tensor core instructions of sm_100a and the tiled TMA copies that feed them
// (one CTA, no multicast).
#pragma once
#include <cstdint>
#include <cuda.h>

#include "ptx.cuh"

namespace mk {

// Tiled copy of a 2-d box, global -> this CTA's shared memory. x: the innermost coordinate, in elements (a multiple of 8 of a
// 16-bit type); places outside of the tensor read as zero and count like the others. policy: an L2 cache policy.
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, uint64_t* bar, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

__device__ __forceinline__ uint64_t l2_evict_first()
{
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}

__device__ __forceinline__ uint64_t l2_evict_last()
{
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}

// All 512 columns of tensor memory, by one warp; the address is left at `slot`. The CTA must be alone on its SM.
__device__ __forceinline__ void tmem_alloc_all(uint32_t* slot)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}

__device__ __forceinline__ void tmem_free_all(uint32_t at)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(at));
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A tile in shared memory whose rows are 128 bytes of the contracted dimension, laid down by TMA with the 128-byte swizzle (1024
// bytes from one group of eight rows to the next; 1024-byte aligned). Steps along the contraction add bytes / 16.
__device__ __forceinline__ uint64_t smem_tile_desc(const void* tile)
{
    return (uint64_t)((smem_u32(tile) & 0x3ffffu) >> 4) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// D [128 x n] in tensor memory (+)= A [128 x 16] B [n x 16]^T, 16-bit operands of one type, fp32 sums.
__device__ __forceinline__ uint32_t mma_f16_desc(bool bf16, uint32_t n)
{
    const uint32_t t = bf16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
        : "memory");
}

// An arrival on `bar` once all MMAs that this thread has issued are done.
__device__ __forceinline__ void mma_commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// 16 columns of this warp's 32 lanes (lanes 32 * (warp % 4) on), one lane a thread; the values are there after tmem_wait.
__device__ __forceinline__ void tmem_load16(float (&x)[16], uint32_t at)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]),
          "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
        : "r"(at)
        : "memory");
}

// Takes the values through its operands, so that nothing that uses them is moved ahead of it.
__device__ __forceinline__ void tmem_wait(float (&x)[16], float (&y)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]),
                   "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]),
                   "+f"(x[15]), "+f"(y[0]), "+f"(y[1]), "+f"(y[2]), "+f"(y[3]), "+f"(y[4]), "+f"(y[5]), "+f"(y[6]),
                   "+f"(y[7]), "+f"(y[8]), "+f"(y[9]), "+f"(y[10]), "+f"(y[11]), "+f"(y[12]), "+f"(y[13]),
                   "+f"(y[14]), "+f"(y[15])
                 :
                 : "memory");
}

} // namespace mk
