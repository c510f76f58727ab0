// Instructions of the tensor cores and of the copies that feed them, as the softmax kernels use them (sm_100a).
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace gtm_readout {

__device__ __forceinline__ unsigned smem_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// The same place in the shared memory of the pair's first thread block.
__device__ __forceinline__ unsigned in_leader(unsigned address)
{
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(address));
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void barrier_init(unsigned barrier, unsigned count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_expect(unsigned barrier, unsigned bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}

// Behind loads from tensor memory that have been waited for and `tmem_before_sync`, which order them; nothing else is told by it.  With .release the
// arrival waited for the thread's stores too, 2,300 cycles.
__device__ __forceinline__ void barrier_arrive_leader(unsigned barrier_in_leader)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(barrier_in_leader) : "memory");
}

__device__ __forceinline__ bool barrier_try(unsigned barrier, unsigned parity)
{
    unsigned done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(barrier), "r"(parity) : "memory");
    return done;
}

// Whether a phase of a barrier is over, without a wait.
__device__ __forceinline__ bool barrier_test(unsigned barrier, unsigned parity)
{
    unsigned done;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(barrier), "r"(parity) : "memory");
    return done;
}

__device__ __forceinline__ unsigned long long nanoseconds()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Waits for a phase of a barrier, `limit` nanoseconds at most.  The clock is asked only once a usual wait is over.
__device__ __forceinline__ bool barrier_wait(unsigned barrier, unsigned parity, unsigned long long limit)
{
#pragma unroll 1
    for (int i = 0; i < 64; i++)
        if (barrier_try(barrier, parity)) return true;
    const unsigned long long began = nanoseconds();
    while (nanoseconds() - began < limit)
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (barrier_try(barrier, parity)) return true;
    return false;
}

// A box of a tensor map to shared memory; its bytes count on a barrier of the pair's first block.
__device__ __forceinline__ void load_box(const CUtensorMap *map, unsigned to, unsigned barrier_in_leader, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to), "l"(map),
                 "r"(barrier_in_leader), "r"(x), "r"(y), "r"(z)
                 : "memory");
}

__device__ __forceinline__ void tmem_allocate(unsigned to, unsigned columns)
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}

__device__ __forceinline__ void tmem_free(unsigned address, unsigned columns)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}

__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Operand tile in shared memory, rows of 128 bytes swizzled by 128; strides in bytes.
__device__ __forceinline__ unsigned long long operand(unsigned address, unsigned leading, unsigned stride)
{
    return (unsigned long long)((address & 0x3ffff) >> 4) | (unsigned long long)(leading >> 4) << 16 | (unsigned long long)(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Products of two 16-bit types (0: fp16, 1: bf16) in 32 bits, 256 rows over the pair.  `a_rows`: operand A's rows (and not its
// sum's index) lie next to each other in memory.
__host__ __device__ constexpr unsigned product(int type, int columns, bool a_rows)
{
    return 1u << 4 | (unsigned)type << 7 | (unsigned)type << 10 | (unsigned)a_rows << 15 | (unsigned)(columns / 8) << 17 | (256u / 16) << 24;
}

__device__ __forceinline__ void multiply(unsigned to, unsigned long long a, unsigned long long b, unsigned what, bool add)
{
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(to), "l"(a), "l"(b), "r"(what), "r"((unsigned)add) : "memory");
}

// Arrival on a barrier of both blocks once all products issued so far are done.
__device__ __forceinline__ void commit_to_pair(unsigned barrier)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(barrier), "h"((unsigned short)3) : "memory");
}

// Columns of the warp's 32 rows: column i in v[i].
__device__ __forceinline__ void tmem_load32_begin(unsigned from, float *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
                   "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
                   "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
                   "=f"(v[31])
                 : "r"(from));
}

// Waits for the warp's loads.  The registers are operands, so that nothing is done with them before.
__device__ __forceinline__ void tmem_load32_end(float *v)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                 "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]),
                 "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_load32(unsigned from, float (&v)[32])
{
    tmem_load32_begin(from, v);
    tmem_load32_end(v);
}

__device__ __forceinline__ void tmem_load64(unsigned from, float (&v)[64])
{
    tmem_load32_begin(from, v);
    tmem_load32_begin(from + 32, v + 32);
    tmem_load32_end(v);
    tmem_load32_end(v + 32);
}

// 2^x by the hardware, off by up to 2^-22 of the value; zero below 2^-126.  As exact as the 32-bit logits and sums around it, and one instruction.
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace gtm_readout
