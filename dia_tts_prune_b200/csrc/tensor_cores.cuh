// tensor_cores.cuh - PTX of the 5th-generation tensor cores (tcgen05, TMEM, TMA tiles, pairs of SMs) shared by the kernels that multiply.
#pragma once

#include <cuda.h>
#include <math_constants.h>

#include "common.cuh"

namespace dia {

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
                 : "memory");
}
// K-major, 128-byte swizzle: rows of 128 B, 8-row groups 1024 B apart (stride byte offset), version 1 (sm_100)
__device__ __forceinline__ uint64_t umma_desc(uint32_t smem_addr) {
    const uint32_t lo = ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ uint32_t at_rank(const void* local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ bool pair_wait(uint64_t* bar, uint32_t parity, unsigned polls) {       // one answer for a converged warp
    for (unsigned i = 0; i < polls; ++i)
        if (__any_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return false;
}
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity, unsigned polls) {
    for (unsigned i = 0; i < polls; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}
// a load of this CTA that counts on a barrier of the pair's leader
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void umma_bf16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {                // the barrier at this place in both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- how a kernel leaves: nothing that it issued arrives behind it, whichever of its waits ran out ----
// Looks at a barrier for what the kernel has issued itself and what therefore comes, in microseconds: tens of milliseconds, whatever limit its other waits have.
constexpr unsigned kDrainPolls = 1u << 16;

// one thread: the copies of a ring's last uses have landed, where this CTA armed its barriers for all of them (`issued` uses in turn, `stages` of them at a time)
__device__ __forceinline__ void copies_landed(uint64_t* full, unsigned stages, unsigned issued) {
    for (unsigned j = issued > stages ? issued - stages : 0; j < issued; ++j) (void)lane_wait(&full[j % stages], (j / stages) & 1u, kDrainPolls);
}
// the warp that issued them: its MMAs have ended, and what they committed has arrived (done: a barrier of one arrival that nothing else uses)
template <bool PAIR>
__device__ __forceinline__ void mmas_ended(uint64_t* done) {
    if (elect_one_sync()) {
        if constexpr (PAIR) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(done)) : "memory");
        else umma_commit(done);
    }
    __syncwarp();
    (void)pair_wait(done, 0u, kDrainPolls);
}

// A pair's copies count on the leader's barriers, and either CTA's loader may be the one that gives up.  Both say how many uses of the ring they filled; where a wait ran out,
// the leader stands in for what the other one did not do.
struct PairEnd {
    uint64_t done;                                            // see mmas_ended
    uint32_t issued[2];                                       // the leader's: uses of the ring that either CTA has filled
    uint32_t gave_up;                                         // in both
};
__device__ __forceinline__ void store_remote(const uint32_t* local, uint32_t rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at_rank(local, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void pair_begin(PairEnd* end) {    // one thread, in front of a cluster barrier
    mbar_init(&end->done, 1);
    end->gave_up = 0;
}
__device__ __forceinline__ void pair_issued(PairEnd* end, uint32_t rank, unsigned issued) { store_remote(&end->issued[rank], 0, issued); }      // the loader, behind its last copy
__device__ __forceinline__ void pair_gave_up(PairEnd* end) {                                // any thread, in front of pair_end
    store_remote(&end->gave_up, 0, 1u);
    store_remote(&end->gave_up, 1, 1u);
}
// Every thread of both CTAs, converged.  (A use beyond the other's last one lies less than a ring ahead: the slot was free, so both had filled it before.)
__device__ __forceinline__ void pair_end(PairEnd* end, uint32_t rank, uint64_t* full, unsigned stages, uint32_t bytes) {
    cluster_sync_all();
    if (!*reinterpret_cast<volatile uint32_t*>(&end->gave_up)) return;
    if (rank == 0 && threadIdx.x == 0) {
        const unsigned mine = end->issued[0], other = end->issued[1], most = max(mine, other);
        for (unsigned j = most > stages ? most - stages : 0; j < most; ++j) {
            uint64_t* const bar = &full[j % stages];
            if (j >= mine) mbar_arrive_expect_tx(bar, bytes);                                // (armed for one CTA's bytes)
            else if (j >= other) asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
            (void)lane_wait(bar, (j / stages) & 1u, kDrainPolls);
        }
    }
    __syncwarp();
    cluster_sync_all();
}

__device__ __forceinline__ void tmem_columns16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr)
        : "memory");
}

__device__ __forceinline__ void tmem_columns32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr)
        : "memory");
}

__device__ __forceinline__ float load_remote(const float* local, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_remote4(const float* local, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// (The driver encodes maps on threads that have a context, which the runtime gives a thread with its first call that needs one: a thread of the caller's, or the one that a
// backward pass begins on, may not have made any.)
static EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    static thread_local bool bound = false;
    if (!bound) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return nullptr;
        bound = true;
    }
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

}  // namespace dia
