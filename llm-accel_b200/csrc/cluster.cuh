// Exchange between the CTAs of a thread-block cluster.  A value goes to another CTA's
// shared memory with its arrival counted by a barrier there (st_async), so that the
// receiver waits for the values alone: a cluster barrier with release would first
// drain whatever the CTAs have on its way to memory.  For launches with clusters only: in
// one without, an asynchronous store faults, also one to the CTA itself.
#pragma once
#include <cstdint>

#include "gemv_common.cuh"

namespace llmx {

static __device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Address of p's place in the shared memory of the cluster's CTA `rank`.
static __device__ __forceinline__ uint32_t remote(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// For the exchange's start: barriers are set up before cluster_arrive (after
// fence.mbarrier_init), nothing is sent before cluster_wait.
static __device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
static __device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Time for what nobody waits for any more to land: some 100 us, hundreds of times what it takes.
static __device__ __forceinline__ void let_land() {
    for (const long long t = clock64(); clock64() - t < 200000;) {
    }
}
// The exchange's end, after a cluster_arrive by every thread of the cluster once it sends nothing
// more and every thread of its CTA has passed the cluster_wait before: no CTA's shared memory
// goes while another may still address it.  came: this thread got all that it waited for; if
// not, something may have been sent just now.
static __device__ __forceinline__ void cluster_leave(bool came) {
    __syncwarp();
    cluster_wait();
    if (!came) let_land();
}
// The receiver's barrier expects the bytes of all values (mbar_expect_tx).
static __device__ __forceinline__ void st_async(uint32_t to, uint64_t v, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u64 [%0], %1, [%2];" ::"r"(to), "l"(v), "r"(bar)
                 : "memory");
}
static __device__ __forceinline__ void st_async(uint32_t to, int32_t v, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.s32 [%0], %1, [%2];" ::"r"(to), "r"(v), "r"(bar)
                 : "memory");
}
// An arrival on another CTA's barrier, once everything this thread did before is seen there.
static __device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Whether the phase is complete now; try_wait would stay for a microsecond where it is not.
static __device__ __forceinline__ bool mbar_test_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
static __device__ __forceinline__ bool mbar_wait_cluster(uint64_t *bar, uint32_t parity, uint32_t polls) {
#pragma unroll 1
    for (uint32_t i = 0; i < polls; i++) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}

}  // namespace llmx
