// glm_tc.cuh -- mbarriers, clusters, TMEM and descriptors shared by the
// tcgen05 kernels (glm_dense.cu, glm_ortho.cu, glm_q4.cu).
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "glm_common.cuh"

namespace glmb {

constexpr long long kWaitCycles = 4ll << 30;  // ~2 s at 1.9 GHz

__device__ __forceinline__ uint32_t saddr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(unsigned long long* b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* b, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(saddr(b)),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool mbar_test(unsigned long long* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(saddr(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Arrive on the barrier at the same shared-memory offset in CTA `rank` of
// this cluster (default semantics: release at CTA scope).  What the arrival
// publishes is either tensor-core input in this CTA's shared memory, made
// visible to the async proxy by fence.proxy.async beforehand, or the end of
// this CTA's TMEM reads, ordered by tcgen05.fence::before_thread_sync.
// (A release at cluster scope measured 750-1200 cycles per arrival here.)
__device__ __forceinline__ void mbar_arrive_rank(unsigned long long* b, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(saddr(b)), "r"(rank));
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Both CTAs of the pair reach this point (every thread of both).
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Bounded wait: false when the clock limit ran out (which sets *failed) or, with
// `failed` given, as soon as another role has failed.  Teardown waits pass
// failed == nullptr and only give up on the limit.
__device__ __forceinline__ bool mbar_wait(unsigned long long* b, uint32_t parity, volatile int* failed) {
    const long long t0 = clock64();
    while (!mbar_test(b, parity)) {
        if (failed != nullptr && *failed) return false;
        if (clock64() - t0 > kWaitCycles) {
            if (failed != nullptr) *failed = 1;
            return false;
        }
    }
    return true;
}

// The same for a whole warp, which comes out of it converged (what follows -- TMEM loads, an arrival for the
// warp -- needs that) and of one mind.
__device__ __forceinline__ bool mbar_wait_warp(unsigned long long* b, uint32_t parity, volatile int* failed) {
    if (__all_sync(0xffffffffu, mbar_test(b, parity))) return true;
    const bool ok = mbar_wait(b, parity, failed);
    return __all_sync(0xffffffffu, ok) != 0;
}

// The warp of this thread as a value that the compiler knows to be the same in all its lanes.  A role that
// branches on it and loops as a whole warp keeps its descriptors in uniform registers, which the MMA reads; with
// one lane of a divergent branch every operand of every MMA went through a move first, and issuing one took 100
// to 170 clocks.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0); }
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor (tcgen05 "version 1").
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo, uint32_t layout) {
    uint64_t d = 0;
    d |= uint64_t((addr >> 4) & 0x3FFF);
    d |= uint64_t((lbo >> 4) & 0x3FFF) << 16;
    d |= uint64_t((sbo >> 4) & 0x3FFF) << 32;
    d |= uint64_t(1) << 46;  // descriptor version for sm_100
    d |= uint64_t(layout & 7) << 61;
    return d;
}

// The two words of such a descriptor apart: the one with the address, which a loop can add to (in units of 16
// bytes), and the one that stays.  One thread issues all MMAs, so every instruction it spends on a descriptor
// is on the path: building whole descriptors per MMA took longer than the MMAs of N < 256.
// (A shared-memory address carries the CTA's rank in its cluster above the bits a descriptor takes.)
__device__ __forceinline__ uint32_t desc_address(uint32_t addr, uint32_t lbo) {
    return ((addr >> 4) & 0x3FFF) | ((lbo >> 4) << 16);
}
constexpr uint32_t desc_rest(uint32_t sbo, uint32_t layout) { return (sbo >> 4) | (1u << 14) | (layout << 29); }
__device__ __forceinline__ uint64_t desc_join(uint32_t address, uint32_t rest) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(address), "r"(rest));
    return d;
}

// 16 consecutive 32-bit columns of this warp's 32 TMEM lanes; the values
// are valid after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// Waits for this thread's outstanding TMEM loads.  The registers pass through
// the statement so that no use of them is scheduled ahead of the wait.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15])
                 :
                 : "memory");
}
// Orders later uses of r after the preceding volatile statement (a wait).
__device__ __forceinline__ void reg_after(uint32_t (&r)[16]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]));
}

// Every thread of the cluster has come this far; nothing it wrote is published (a release waits for every
// store in flight, about 2000 clocks behind a tile's output).
__device__ __forceinline__ void cluster_sync_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// The address in CTA `rank` of this cluster of what is at `addr` here, and loads from there.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_cluster_f32(const float* p, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa(saddr(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ double ld_cluster_f64(const double* p, uint32_t rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa(saddr(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ int ld_cluster_s32(const int* p, uint32_t rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa(saddr(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// cuTensorMapEncodeTiled, fetched through the runtime; nullptr without a driver (glm_dense.cu).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

}  // namespace glmb
