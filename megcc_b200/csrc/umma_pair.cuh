// Inline-PTX building blocks of kernels in which a pair of CTAs, one per SM, works on one tile
// (cta_group::2): cluster addresses and barriers, TMA loads that report to the other CTA, MMAs and commits.
#pragma once
#include "umma_ptx.cuh"

namespace mb200 {
namespace umma {

__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_id_x() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t num_clusters_x() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%nclusterid.x;" : "=r"(r));
    return r;
}
// the shared::cluster address of `local` (an address in this CTA's shared memory) in CTA `rank`
__device__ __forceinline__ uint32_t map_to_cta(uint32_t local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
                 : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
            : "memory");
    return ok != 0;
}
// bounded wait on a barrier that the other CTA of the pair (or a commit issued there) arrives on
__device__ __forceinline__ bool mbar_wait_cluster(
        uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
        if (mbar_try_wait_cluster(bar, parity))
            return true;
    const long long t0 = clock64();
    for (int spin = 0;; ++spin) {
        if (mbar_try_wait_cluster(bar, parity))
            return true;
        if (spin > 256)
            __nanosleep(128);
        if ((spin & 63) == 63) {
            if (*abort_flag)
                return false;
            if (clock64() - t0 > kWaitCycles)
                return false;
        }
    }
}
// TMA loads of a CTA pair: the data lands in THIS CTA's shared memory, the byte count is
// reported to the barrier at `mbar_cluster_addr`, which may belong to the other CTA
__device__ __forceinline__ void tma_pair_load_2d(
        void* smem, const CUtensorMap* map, uint32_t mbar_cluster_addr, int c0, int c1) {
    asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(smem)),
            "l"((uint64_t)map), "r"(mbar_cluster_addr), "r"(c0), "r"(c1)
            : "memory");
}
__device__ __forceinline__ void tma_pair_load_im2col_4d(
        void* smem, const CUtensorMap* map, uint32_t mbar_cluster_addr, int c, int w, int h, int n,
        uint16_t off_w, uint16_t off_h) {
    asm volatile(
            "cp.async.bulk.tensor.4d.im2col.cta_group::2.shared::cluster.global"
            ".mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2], {%7, %8};" ::"r"(
                    smem_u32(smem)),
            "l"((uint64_t)map), "r"(mbar_cluster_addr), "r"(c), "r"(w), "r"(h), "r"(n), "h"(off_w),
            "h"(off_h)
            : "memory");
}
__device__ __forceinline__ void umma_pair_s8(
        uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
}
// arrives (once) on the barrier at a shared::cluster address when the pair's MMAs issued so
// far have retired
__device__ __forceinline__ void umma_pair_commit(uint32_t bar_cluster_addr) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                         bar_cluster_addr)
                 : "memory");
}

}  // namespace umma
}  // namespace mb200
