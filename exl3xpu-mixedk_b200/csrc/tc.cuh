// tc.cuh -- mbarrier, TMA and tcgen05 wrappers of the forward kernels.  Every wait is
// bounded.  A wait for another role's handover gives up after the library's wait limit
// (exl3b_set_wait_limit_ms), or when another role of the CTA has; the CTA then drains
// what it has in flight, whatever that limit is, and ends.  No wait spans more than one
// handover or drain, so a long product does not come near the limit.
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace exl3b {

__device__ __forceinline__ uint32_t shared_addr(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}

__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                 :: "r"(bar), "r"(bytes) : "memory");
}

// The limit of a wait, in SM cycles, and how long one try may sleep, in ns.
struct WaitLimit {
    long long cycles;
    uint32_t sleep;
    WaitLimit() = default;
    __host__ __device__ explicit WaitLimit(long long c)
        : cycles(c), sleep(c < 40000 ? (uint32_t)(c / 2) : 20000u) {}
};

__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity, uint32_t sleep) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(sleep) : "memory");
    return ok != 0;
}

// Wait for a handover; false when the wait ran out or `fail` (shared memory) is set.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const int* fail,
                                         const WaitLimit& limit) {
    if (bar_try(bar, parity, limit.sleep)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (bar_try(bar, parity, limit.sleep)) return true;
        if (*(const volatile int*)fail || clock64() - t0 > limit.cycles) return false;
    }
}

// Wait for what is in flight already (copies, MMAs); false after some two seconds.
__device__ __forceinline__ bool bar_drain(uint32_t bar, uint32_t parity) {
    const int never = 0;
    return bar_wait(bar, parity, &never, WaitLimit(4000000000LL));
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];"
        :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// Shared-memory operand descriptor: K-major rows of 128 bytes, 128-byte swizzle, atoms
// of 8 rows 1 KB apart.  A k step of 16 fp16 inside the row adds 32 bytes.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Instruction descriptor: fp32 accumulators, fp16 operands, both K-major.
__host__ __device__ constexpr uint32_t mma_desc_f16(int m, int n) {
    return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Count bytes at a barrier that no copy will bring any more.
__device__ __forceinline__ void bar_forgo(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;"
                 :: "r"(bar), "r"(bytes) : "memory");
}

// Arrive at `bar` when every MMA this thread has issued is done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 :: "r"(bar) : "memory");
}

// 32 columns of this warp's 32 lanes; wait for them with tc_wait_ld.
__device__ __forceinline__ void tc_load32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_wait_ld() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ------------------------------------------------------------ pairs of CTAs
// Address of a shared-memory location in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ void cluster_store(uint32_t addr, int v) {
    asm volatile("st.shared::cluster.s32 [%0], %1;" :: "r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Arrive at a barrier given by its cluster address.  What these arrivals order is tensor
// memory, by the tcgen05 fences around them; a release at cluster scope would make the
// warp wait for its copies in flight.
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(bar) : "memory");
}

// A load into this CTA's shared memory, counted at a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];"
        :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// Arrive at `bar` of both CTAs of the pair when every MMA issued so far is done.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        :: "r"(bar), "h"((uint16_t)3) : "memory");
}

// All 512 columns of tensor memory, for both CTAs of a pair.  A warp of each.
__device__ __forceinline__ void tc_alloc_pair(uint32_t slot) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_free_pair(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
}

}  // namespace exl3b
