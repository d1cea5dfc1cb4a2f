// The tensor-core side of the MXFP4 products: descriptors, scale copies, block-scaled multiplications and accumulator reads.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace mps {

// Shared-memory operand: rows of 128 bytes, 8-row groups of 1024 bytes one after the other, 16-byte pieces XORed with the row
// (the 128-byte swizzle), columns innermost.
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem) {
    return (uint64_t)((smem >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 512 bytes of scales, 32 rows of 16 bytes, not swizzled.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem) {
    return (uint64_t)((smem >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// E2M1 x E2M1, E8M0 scales, FP32 accumulator of m x n; `sf` says which two of a scale word's four blocks a step of 64 columns uses.
__device__ __forceinline__ uint32_t mx4_instruction(uint32_t m, uint32_t n, uint32_t sf) {
    return sf << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | 1u << 23 | (m >> 7) << 27 | sf << 29;
}

// A CTA that may still allocate keeps others of its SM from it, so the permit goes back at once.
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, uint32_t columns) {
    if (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
    if (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
// What issues to the tensor core runs as a whole warp, and the lane that `lead` (elect_one, taken once) names issues: without a branch around the
// instructions their addresses and descriptors, the same in all lanes, stay in uniform registers, where they are taken from.  Measured with a branch
// around them: some 80 cycles an instruction, twice what a stage's multiplications take.

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
// 128 rows' scales of 128 columns into four columns of tensor memory, the same in each of its four lane quarters.
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t lead, uint32_t tmem, uint64_t desc) {
    if (CTAS == 1)
        asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %2, 0;\n\t@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}"
                     ::"r"(tmem), "l"(desc), "r"(lead) : "memory");
    else
        asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %2, 0;\n\t@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}"
                     ::"r"(tmem), "l"(desc), "r"(lead) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mx4_multiply(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t sfa, uint32_t sfb, uint32_t add) {
    if (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %6, 0;\n\tsetp.ne.u32 e, %7, 0;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(sfa), "r"(sfb), "r"(add), "r"(lead) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %6, 0;\n\tsetp.ne.u32 e, %7, 0;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(sfa), "r"(sfb), "r"(add), "r"(lead) : "memory");
}
// The barrier gets an arrival when everything that lane has issued to the tensor core is done.
__device__ __forceinline__ void tensor_commit(uint32_t lead, uint32_t bar) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %1, 0;\n\t@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// The same for a pair of CTAs: at this place in the shared memory of those that CTAS, a bit each, names.
template <int CTAS = 3>
__device__ __forceinline__ void tensor_commit_pair(uint32_t lead, uint32_t bar) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %2, 0;\n\t"
                 "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
                 ::"r"(bar), "h"((uint16_t)CTAS), "r"(lead) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Arrival at the first CTA's barrier of this place, from either: what this thread did or has seen done before (copies that have come, the accumulator
// read) is done for the thread of the other CTA that waits there.  Without a scope it would be so for this CTA's threads alone.
__device__ __forceinline__ void arrive_at_first(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar) : "memory");
}
// A poll of a barrier that is arrived at, or whose bytes are sent, from another CTA.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Another CTA's shared memory, at the place that has this address in one's own.
__device__ __forceinline__ uint32_t peer_address(uint32_t smem, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 load_peer(uint32_t address) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ void add4(float4& a, const float4& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }
// A box of a tensor map, from its first column and `row` on, into this CTA's shared memory; the bytes count at a barrier of either CTA of the pair, which
// gets them as a release at cluster scope (an untiled bulk copy counts at its own CTA's barriers only).
__device__ __forceinline__ void tiled_g2s_pair(uint32_t dst, const CUtensorMap* map, int row, uint32_t pair_bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(pair_bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// One value into another CTA's shared memory; the barrier there counts its four bytes once they are there.
__device__ __forceinline__ void send_to(uint32_t address, uint32_t bar, float v) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(address), "r"(__float_as_uint(v)), "r"(bar) : "memory");
}
// The cluster's barrier in two halves.  An arrival orders nothing; who has waited knows that all have arrived.  Who leaves after it, or reads what was
// written before it, needs cluster_sync: behind an arrival that orders nothing, a read of another CTA's memory or an arrival there may still be on its way.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Sixteen columns of the accumulator, a lane of tensor memory per thread; the whole warp takes part.  Load and wait are one
// statement: the compiler knows nothing of the wait and might use a register before it.
__device__ __forceinline__ void tmem_load16(uint32_t tmem, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(tmem) : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Thirty-two columns, as above.
__device__ __forceinline__ void tmem_load32(uint32_t tmem, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(tmem) : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

}  // namespace mps
