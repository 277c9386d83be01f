// Fifth-generation tensor core helpers (PTX wrappers): products of 16-bit tiles in shared memory, accumulated in tensor memory.
// The tiles are the blocks of newton_schulz.cu: 64 elements (128 bytes) per row, the 16-byte chunk c of row r at position
// c ^ (r & 7), eight rows after one another (the 128-byte swizzle of the matrix descriptors).
#pragma once

#include "tma.cuh"

namespace sb200 {

#ifdef __CUDACC__
// rows of the tile are rows of the operand, its columns the summation index: groups of eight rows lie 1024 bytes apart
__device__ __forceinline__ uint64_t desc_rows(unsigned addr)
{
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// rows of the tile are the summation index, its columns rows of the operand: eight summation steps lie 1024 bytes apart,
// the next 64 columns `far` bytes
__device__ __forceinline__ uint64_t desc_columns(unsigned addr, unsigned far)
{
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(far >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// fp16 x fp16 -> fp32, M x N; which operands are given by desc_columns
__device__ __forceinline__ uint32_t product_shape(int m, int n, bool a_columns, bool b_columns)
{
    return 1u << 4 | (a_columns ? 1u << 15 : 0u) | (b_columns ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// The operations come for one CTA (CG = 1), or for a cluster of two (CG = 2) whose tensor cores make one product of twice the rows:
// each CTA has half of the first operand's rows and half of the second's, at the same places of its shared memory, and gets
// its own rows of the result.  The first CTA issues it.

// one thread: d (+)= a b, 16 steps of the summation index
template <int CG>
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add)
{
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
            : "memory");
}

// the barrier (of both CTAs) is told when all products that this thread has issued are done
template <int CG>
__device__ __forceinline__ void product_commit(uint64_t *bar)
{
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

// one warp (of each CTA); `columns` a power of two from 32 to 512
template <int CG>
__device__ __forceinline__ void tensor_alloc(uint32_t *where, uint32_t columns)
{
    if constexpr (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}

template <int CG>
__device__ __forceinline__ void tensor_free(uint32_t base, uint32_t columns)
{
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}

__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// one warp reads 32 columns of its 32 lanes (those of quarter warp % 4): lane = row
__device__ __forceinline__ void tensor_read(float (&v)[32], uint32_t addr)
{
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// the same, 16 columns
__device__ __forceinline__ void tensor_read(float (&v)[16], uint32_t addr)
{
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// contiguous copy of global memory into shared memory; both 16-byte aligned, bytes a multiple of 16
__device__ __forceinline__ void bulk_load(void *dst, const void *src, unsigned bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// The barrier at the same place of another CTA of the cluster.  What these arrivals stand for lies in shared or tensor memory, where
// it is by then, so they need none of the ordering of global memory that a release of cluster scope waits for (it and
// the acquire on the other side took 2000 cycles a step where the products take 512).
__device__ __forceinline__ void mbar_arrive_at(uint64_t *bar, unsigned rank)
{
    asm volatile(
        "{\n\t.reg .b32 far;\n\t"
        "mapa.shared::cluster.u32 far, %0, %1;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [far];\n\t}"
        ::"r"(smem_u32(bar)), "r"(rank) : "memory");
}

// the same, and what other threads of the cluster have done before they arrived is seen
__device__ __forceinline__ void mbar_release_at(uint64_t *bar, unsigned rank)
{
    asm volatile(
        "{\n\t.reg .b32 far;\n\t"
        "mapa.shared::cluster.u32 far, %0, %1;\n\t"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [far];\n\t}"
        ::"r"(smem_u32(bar)), "r"(rank) : "memory");
}

__device__ __forceinline__ bool mbar_acquire_bounded(uint64_t *bar, unsigned parity, int limit)
{
    for (int i = 0; i < limit; ++i) {
        unsigned ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
}

// Between plain accesses and asynchronous copies of the same memory, in either order: global and shared, or global alone.
__device__ __forceinline__ void fence_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void fence_async_global() { asm volatile("fence.proxy.async.global;" ::: "memory"); }

// a barrier of `threads` threads of the CTA, which says whether all of them came with `value`
__device__ __forceinline__ bool all_agree(int barrier, int threads, bool value)
{
    unsigned all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %3, 0;\n\t"
        "barrier.cta.red.and.pred p, %1, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all) : "r"(barrier), "r"(threads), "r"((unsigned)value) : "memory");
    return all != 0;
}

// A count that the CTAs of a grid which is resident as a whole arrive at.
__device__ __forceinline__ void grid_arrive(unsigned *count) { asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(count) : "memory"); }

__device__ __forceinline__ bool grid_wait_bounded(const unsigned *count, unsigned target, int limit)
{
    for (int i = 0; i < limit; ++i) {
        unsigned now;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(count) : "memory");
        if (now >= target) return true;
    }
    return false;
}

__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ unsigned cluster_size()
{
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

// all threads of all CTAs of the cluster
__device__ __forceinline__ void cluster_wait_all()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void write_at(void *p, unsigned rank, float4 v)
{
    asm volatile(
        "{\n\t.reg .b32 far;\n\t"
        "mapa.shared::cluster.u32 far, %0, %1;\n\t"
        "st.shared::cluster.v4.f32 [far], {%2, %3, %4, %5};\n\t}"
        ::"r"(smem_u32(p)), "r"(rank), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// 16 bytes at the same place of another CTA's shared memory
__device__ __forceinline__ float4 read_at(const void *p, unsigned rank)
{
    float4 v;
    asm volatile(
        "{\n\t.reg .b32 far;\n\t"
        "mapa.shared::cluster.u32 far, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [far];\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_u32(p)), "r"(rank) : "memory");
    return v;
}

__device__ __forceinline__ void write_at(void *p, unsigned rank, uint32_t a, uint32_t b)
{
    asm volatile(
        "{\n\t.reg .b32 far;\n\t"
        "mapa.shared::cluster.u32 far, %0, %1;\n\t"
        "st.shared::cluster.v2.b32 [far], {%2, %3};\n\t}"
        ::"r"(smem_u32(p)), "r"(rank), "r"(a), "r"(b) : "memory");
}

__device__ __forceinline__ double read_double_at(const void *p, unsigned rank)
{
    double v;
    asm volatile(
        "{\n\t.reg .b32 far;\n\t"
        "mapa.shared::cluster.u32 far, %1, %2;\n\t"
        "ld.shared::cluster.f64 %0, [far];\n\t}"
        : "=d"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
    return v;
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
#endif

}  // namespace sb200
