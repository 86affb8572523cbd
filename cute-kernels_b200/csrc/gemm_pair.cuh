// Pieces shared by the kernels that run on CTA pairs (gemm_tc2.cu, gemm_fp8.cu, gemm_wgrad.cu): cluster addressing, barriers across
// the pair, paired loads, MMAs and commits, and the epilogue's staging patch.
#pragma once

#include "gemm_tc.cuh"

namespace fmab {

// Address of the 16-byte piece (row, piece) of a per-warp staging patch: 32 rows x 128 bytes, pieces
// XOR-swizzled by the row.  Both ways the epilogues touch a patch are then free of bank conflicts:
//   row form   lane = row, one piece per access (how tensor memory hands out an accumulator: a row per lane);
//   line form  one access covers 4 rows x 8 pieces, i.e. four whole 128-byte rows (what global memory likes):
//              step `it` (0..7) gives lane the piece (row it*4 + lane/8, piece lane%8).
__device__ __forceinline__ uint32_t patch_addr(uint32_t patch, int row, int piece) {
    return patch + row * 128 + ((static_cast<uint32_t>(piece) ^ (static_cast<uint32_t>(row) & 7u)) << 4);
}

__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// shared::cluster address of the same shared-memory offset in the CTA of rank `rank`
__device__ __forceinline__ uint32_t map_to_rank(uint32_t smem_addr, uint32_t rank) {
    uint32_t out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_addr), "r"(rank));
    return out;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The same arrive without release semantics.  A releasing arrive at cluster scope has to wait until every
// global store the thread has issued is visible cluster-wide, i.e. until the epilogue's output has drained to
// L2 - a microsecond or two per tile during which the tensor memory it frees stays blocked.  What an epilogue
// warp hands back is tensor memory it has finished reading (tcgen05.wait::ld has returned and a
// tcgen05.fence::before_thread_sync precedes the arrive); its global stores need no ordering with the barrier.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void st_shared_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// Bounded wait with cluster-scope acquire, for barriers that a thread of the OTHER CTA arrives on after
// writing ordinary shared memory of this CTA.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
    const uint64_t t0 = global_timer();
    while (true) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        if (global_timer() - t0 > 1000000000ull) {
            *abort_flag = 1;
            atomicExch(status, STATUS_GEMM_TIMEOUT);
            return false;
        }
    }
}
// With one answer for a whole converged warp (see mbar_wait_warp).
__device__ __forceinline__ bool mbar_wait_cluster_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
    return __all_sync(0xffffffffu, mbar_wait_cluster(bar, parity, abort_flag, status));
}
// TMA load into this CTA's shared memory whose completion bytes are counted on the LEADER's mbarrier.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t leader_bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t leader_bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tc_mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives (once the MMAs issued so far have completed) on the barrier at this offset in BOTH CTAs:
// one commit on the leader's own barrier, one on the peer's (its shared::cluster address).
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    const uint32_t peer_bar = map_to_rank(bar, 1);
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(peer_bar) : "memory");
}

// The same with one commit, issued by an elected lane of a converged warp.
__device__ __forceinline__ void tc_commit_both(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
        ::"r"(bar), "h"(static_cast<uint16_t>(3))
        : "memory");
}
// Bytes [batch, outer, inner] with row pitch `pitch`, boxes of box_outer rows x 128 bytes, 128-byte swizzle.  Boxes that
// reach beyond `outer` read zeros there, not the next batch.
inline int encode_bytes_3d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer, uint64_t batch, uint64_t pitch, uint32_t box_outer,
                           uint32_t rank = 3) {
    EncodeTiledFn fn = encode_fn();
    FMAB_REQUIRE(fn != nullptr, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {inner, outer, batch};
    const cuuint64_t strides[2] = {pitch, outer * pitch};
    const cuuint32_t box[3] = {128, box_outer, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FMAB_REQUIRE(r == CUDA_SUCCESS, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled (8-bit operand) failed with CUresult %d", (int)r);
    return FMA_B200_OK;
}
inline int encode_bytes(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer, uint64_t pitch, uint32_t box_outer) {
    return encode_bytes_3d(map, base, inner, outer, 1, pitch, box_outer, 2);
}

}  // namespace fmab
