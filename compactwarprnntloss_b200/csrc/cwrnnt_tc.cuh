// The fifth-generation tensor cores' plumbing, as thin wrappers of PTX: mbarriers with bounded waits, tiled TMA loads,
// TMEM allocation, tcgen05.mma / commit / ld and the two descriptors. Internal.
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace cwrnnt {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_init_fence()
{
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// The same barrier of another CTA of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank)
{
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void mbar_arrive_peer(uint32_t addr)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.b32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}
__device__ __forceinline__ uint64_t now_ns()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// How long a wait has lasted: two seconds of the CTA's own time. The timer runs on while a CTA is off its SM (another
// process's turn on the GPU, a debugger), and a wait that such a break alone made long is not to run out: of what passes between
// two looks at the timer, 20 ms count at most. The waits end all the same, as every look counts what has passed.
struct Patience {
    static constexpr uint64_t kLimit = 2000000000ull, kMostAtOnce = 20000000ull;  // ns
    uint64_t last, waited;
    __host__ __device__ explicit Patience(uint64_t now) : last(now), waited(0) {}
    __host__ __device__ bool spent(uint64_t now)
    {
        const uint64_t step = now - last;
        waited += step < kMostAtOnce ? step : kMostAtOnce;
        last = now;
        return waited > kLimit;
    }
};
// Waits for a phase, as long as its patience lasts. `gave_up` is the CTA's flag (shared memory): whoever runs out of time
// sets it, and everyone else stops waiting then. Returns whether the phase came.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, volatile int *gave_up)
{
    if (mbar_try(bar, parity)) return true;
    Patience patience(now_ns());
    for (;;) {
        for (int i = 0; i < 32; ++i)
            if (mbar_try(bar, parity)) return true;
        if (*gave_up) return false;
        if (patience.spent(now_ns())) {
            *gave_up = 1;
            return false;
        }
    }
}
// The same for what has to come before the CTA's memory goes, whether others have given up or not.
__device__ __forceinline__ void mbar_drain(uint64_t *bar, uint32_t parity)
{
    Patience patience(now_ns());
    while (!mbar_try(bar, parity) && !patience.spent(now_ns())) {
    }
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void load_2d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
                 "[%2];" ::"r"(smem_addr(dst)),
                 "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y)
                 : "memory");
}

// One CTA of a pair loads into its own memory and signals a barrier of the pair's first CTA.
__device__ __forceinline__ void load_2d_pair(void *dst, const CUtensorMap *map, uint32_t bar, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                 "[%1, {%3, %4}], [%2];" ::"r"(smem_addr(dst)),
                 "l"(map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap *map, const void *src, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                 "r"(smem_addr(src)), "r"(x), "r"(y)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// This thread's stores have read their shared memory.
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
// Shared memory written by this thread is visible to the copies issued behind the next barrier.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// PAIR: two CTAs of a cluster on neighbouring SMs share the product (cta_group::2).
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t columns)
{
    if (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)),
                     "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)),
                     "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns)
{
    if (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D[tmem] (+)= A * B, operands described in shared memory; `accumulate` 0 starts a new sum. Of a pair, the first CTA
// issues for both: each gives half the rows of A and half of B, each keeps the sums of its rows of A.
template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    if (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                     "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                     "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
}
// The same with D scaled first: D = A * B + D * 2^-SHIFT, SHIFT at most 15.
template <bool PAIR, int SHIFT>
__device__ __forceinline__ void mma_f16_scaled(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc)
{
    if (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, %4;\n\t}" ::"r"(tmem),
                     "l"(a), "l"(b), "r"(idesc), "n"(SHIFT)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, %4;\n\t}" ::"r"(tmem),
                     "l"(a), "l"(b), "r"(idesc), "n"(SHIFT)
                     : "memory");
}
// The barrier (of a pair: that of both CTAs) completes when every mma issued so far by this thread has.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t *bar)
{
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::
                         "r"(smem_addr(bar)), "h"(uint16_t(3))
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                     : "memory");
}
// 32 consecutive columns of this warp's 32 TMEM lanes: register i of lane t is column i of lane t.
__device__ __forceinline__ void tmem_load32(uint32_t tmem, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(tmem));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory operand of an mma, 128-byte swizzle. K-major: rows of 64 elements along the sum, `sbo` = 1024 bytes from
// one group of eight rows to the next. MN-major: rows of 64 elements along the output, one row per element of the sum;
// `sbo` = 1024 bytes from one group of eight such rows to the next, `lbo` from one 64 outputs to the next.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lbo, uint32_t sbo)
{
    return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(lbo >> 4) << 16) | (uint64_t(sbo >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor of kind::f16 with float sums: type 0 = f16, 1 = bf16 (of both operands).
__host__ __device__ constexpr uint32_t instruction(int type, bool a_mn, bool b_mn, int m, int n)
{
    return (1u << 4) | (uint32_t(type) << 7) | (uint32_t(type) << 10) | (uint32_t(a_mn) << 15) |
           (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

}  // namespace tc
}  // namespace cwrnnt
