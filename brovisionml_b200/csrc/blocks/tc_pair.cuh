// Tensor-core primitives of the feed-forward operators beside those of
// tc_common.cuh: 2-D TMA loads, CTA pairs (cta_group::2), clusters, and the
// descriptors of operands stored with the rows' axis contiguous.
//
// Descriptors (fields as in tc_common.cuh). An operand stored (k, rows), rows
// contiguous, is copied as boxes of 64 rows x 64 k in the 128-byte swizzle: the
// rows run along the 128-byte lines, eight lines (eight k) are one swizzle atom
// of 1024 bytes. The leading byte offset is then the distance between boxes
// (64 rows on), the stride byte offset the distance between atoms (8 k on), and the
// instruction descriptor's transpose bit (15 for A, 16 for B) is set.
#pragma once

#include "../bvml_common.cuh"
#include "../tc_common.cuh"

namespace bvml {
namespace tc {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Every thread of the cluster, whole warps. The warps are together before (the aligned
// forms want that) and after: tcgen05's .sync.aligned instructions and the uniform
// datapath must not meet a warp whose lanes left a barrier one by one.
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    __syncwarp();
}
// The address, in CTA `rank` of the cluster, of this CTA's shared address a.
__device__ __forceinline__ uint32_t map_to(uint32_t a, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
// Arrive on a barrier of another CTA of the cluster, relaxed: for hand-backs of
// tensor memory, whose loads have completed (tcgen05.wait::ld). A release would wait
// until this thread's earlier global stores are visible to the whole cluster.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t remote) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote)
                 : "memory");
}

__device__ __forceinline__ void st_cluster(uint32_t remote, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
// Counts bytes on a barrier of this CTA as if a copy had brought them.
__device__ __forceinline__ void mbar_complete_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
// A wait of teardown after another wait gave up: what is in flight lands within
// microseconds, and some 10 ms are waited for at most.
__device__ __forceinline__ bool mbar_wait_landed(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < 1 << 16; ++i) {
        if (mbar_wait_pipe(bar, parity, 1)) return true;
        __nanosleep(100);
    }
    return false;
}

// Checked builds (-DBVML_CHECKED): a copy whose innermost coordinate or shared-memory
// address is off its alignment, or a store at a negative coordinate, is recorded and left
// out. `inner`: bytes of an element.
__device__ __forceinline__ bool copy_ok(uint32_t smem, int x, int inner, bool store, int y) {
    return check_ok((smem & 127) == 0 && (x * inner) % 16 == 0 && (!store || (x >= 0 && y >= 0)),
                    kChkConvTma);
}

// One lane of the warp, chosen by the hardware. The loops that feed the tensor
// cores are walked by the whole warp, and only the instructions below are
// carried out by this lane (`on`): in a branch that one lane takes, every
// descriptor and address goes through vector registers first (130 cycles for an
// MMA, 580 a K step of which the tensor cores need 512 or fewer).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t on;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(on));
    return on;
}
__device__ __forceinline__ void mbar_expect_tx_on(uint32_t on, uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.u32 q, %2, 0;\n\t"
        "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
        "r"(bytes), "r"(on)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t on, uint32_t dst, const CUtensorMap* map,
                                            uint32_t bar, int c0, int c1) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.u32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(on)
        : "memory");
}
// Towards L2 only: nothing waits for it, and what another kernel writes there
// meanwhile is seen by the load that follows.
__device__ __forceinline__ void tma_prefetch_2d(uint32_t on, const CUtensorMap* map, int c0,
                                                int c1) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.u32 q, %3, 0;\n\t"
        "@q cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n\t}" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(c0), "r"(c1), "r"(on)
        : "memory");
}
// The same, its bytes counted on a barrier of either CTA of the pair (`bar` a
// shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t on, uint32_t dst,
                                                 const CUtensorMap* map, uint32_t bar, int c0,
                                                 int c1) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.u32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(on)
        : "memory");
}

// Tiled store of a box from this CTA's shared memory (bulk-group completion).
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(c0), "r"(c1)
                 : "memory");
}

// Operand stored (k, rows): boxes of 64 rows `box_bytes` apart.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t box_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFF);
    d |= (uint64_t)(box_bytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// ------------------------------------------------------- tcgen05, CTA pairs
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}
// D (256 rows, 128 in each CTA) (+)= A B^T: each CTA holds its 128 rows of A and
// half of B's rows; K = 32 bytes of each row. F8: e4m3 operands.
#define BVML_UMMA(group, kind)                                                                \
    asm volatile(                                                                             \
        "{\n\t.reg .pred p, q;\n\t"                                                           \
        "setp.ne.b32 p, %4, 0;\n\t"                                                           \
        "setp.ne.b32 q, %5, 0;\n\t"                                                           \
        "@q tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(   \
            tmem_d),                                                                          \
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate), "r"(on)              \
        : "memory")
template <bool F8>
__device__ __forceinline__ void umma_pair(uint32_t on, uint32_t tmem_d, uint64_t a_desc,
                                          uint64_t b_desc, uint32_t idesc, bool accumulate) {
    if constexpr (F8) BVML_UMMA("2", "f8f6f4");
    else BVML_UMMA("2", "f16");
}
// ... and one CTA's: D (128 rows), K = 32 bytes.
template <bool F8>
__device__ __forceinline__ void umma_single(uint32_t on, uint32_t tmem_d, uint64_t a_desc,
                                            uint64_t b_desc, uint32_t idesc, bool accumulate) {
    if constexpr (F8) BVML_UMMA("1", "f8f6f4");
    else BVML_UMMA("1", "f16");
}
#undef BVML_UMMA
// Arrive on the barrier at this offset in both CTAs of the pair once every MMA
// issued before by this thread has completed.
__device__ __forceinline__ void umma_commit_pair(uint32_t on, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .b16 m;\n\t.reg .pred q;\n\t"
        "mov.b16 m, 3;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], m;\n\t}" ::"r"(bar), "r"(on)
        : "memory");
}
// ... on this CTA's barrier alone.
__device__ __forceinline__ void umma_commit_pair_local(uint32_t on, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
            bar),
        "r"(on)
        : "memory");
}
// ... and one CTA's MMAs.
__device__ __forceinline__ void umma_commit_on(uint32_t on, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
            bar),
        "r"(on)
        : "memory");
}
// 16 consecutive fp32 columns of this warp's 32 TMEM lanes, one lane per thread.
__device__ __forceinline__ void tmem_ld_16cols(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

// v[0 .. 31] of an array
__device__ __forceinline__ void tmem_ld_32cols(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
        "%28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

}  // namespace tc
}  // namespace bvml
