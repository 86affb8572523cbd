// Weight gradient of a linear map, plain or per expert, in 16 bits on CTA pairs:
//   dW[e][o, i] = sum over the rows r of expert e of dY[r, o] * X[r, i]
// Both operands are read as they lie (rows of features): MN-major tiles of 64 features x 64 rows, 128-byte swizzle.
//
// The reduction of a tile is as long as its expert has rows, a few hundred for experts, so what a tile costs besides its
// MMAs counts.  Hence 256 x 256 pair tiles with two accumulators that fill tensor memory: reading and storing a result
// overlaps the next tile's main loop whole.  Ring stages of 128 rows make it eight MMAs per commit, and the whole issuing
// warp walks the loop (gemm_fp8.cu says what these two are worth); the MMAs start when half a stage has landed (experts of
// 256 / 1024 rows 231 / 619 -> 225 / 606 us).  Results leave through the copy engine, in boxes of 32 rows x 64 columns that
// end with their expert (128 rows per expert, where writing the result is most of the work: 195 us with stores from
// registers, 175 so).
// Measured, bfloat16: 128 experts of 1536 x 2048 with 512 rows each on average 348 us (417 with the 256 x 512 tiles of
// gemm_tc2.cu, whose single accumulator waits for its epilogue), 14336 x 4096 over 8192 rows 631 us, 1.53 PFLOP/s (651
// there; the library takes 608).  What bounds it now is the tensor pipe, and with short reductions writing the result.
#include "fp8.cuh"
#include "gemm_pair.cuh"

namespace fmab {

constexpr int WG_HALF_ROWS = BK;                        // token rows of one load: 64
constexpr int WG_SLAB = 2 * 64 * WG_HALF_ROWS * 2;      // this CTA's 128 features x 64 rows: 16 KB
constexpr int WG_STAGE_BYTES = 4 * WG_SLAB;             // both operands, two halves of 64 rows
constexpr int WG_STAGES = 3;
constexpr int WG_EPI_WARPS = 8;
constexpr int WG_THREADS = 32 * (2 + WG_EPI_WARPS);
constexpr int WG_PATCH_BYTES = 32 * 128;             // 32 rows x 64 columns of the result per epilogue warp
constexpr size_t WG_SMEM = static_cast<size_t>(WG_STAGES) * WG_STAGE_BYTES + WG_EPI_WARPS * WG_PATCH_BYTES + 1024;
constexpr int WG_SUPER = 8;                             // tiles along OUT walked together (operand reuse in L2)

struct WgradParams {
    CUtensorMap map_a, map_b, map_out;
    const int32_t* offsets;  // [E + 1] first row of each expert; null: one expert, all rows
    const int32_t* counts;   // rows to reduce over per expert; null: up to the next offset
    int32_t* status;
    int64_t rows;
    int32_t E, OUT, IN, m_tiles, n_tiles, f16;
};

struct WgradTile {
    int32_t expert, m0, n0, row0, halves;  // halves: 64-row steps of the reduction
};
__device__ __forceinline__ WgradTile wgrad_decode(const WgradParams& p, int tile) {
    const int per_expert = p.m_tiles * p.n_tiles;
    WgradTile t;
    t.expert = tile / per_expert;
    const int in = tile - t.expert * per_expert, per_super = WG_SUPER * p.n_tiles, super = in / per_super;
    const int m_first = super * WG_SUPER, m_span = min(WG_SUPER, p.m_tiles - m_first), r = in - super * per_super;
    const int nt = r / m_span;
    t.m0 = (m_first + (r - nt * m_span)) * 256;
    t.n0 = nt * 256;
    int64_t first = 0, end = p.rows;
    if (p.offsets != nullptr) {
        first = __ldg(p.offsets + t.expert);
        end = min(p.rows, static_cast<int64_t>(__ldg(p.offsets + t.expert + 1)));
    }
    int64_t len = end > first ? end - first : 0;
    if (p.counts != nullptr) len = min(len, static_cast<int64_t>(max(0, __ldg(p.counts + t.expert))));
    t.row0 = static_cast<int32_t>(first);
    t.halves = static_cast<int32_t>((len + WG_HALF_ROWS - 1) / WG_HALF_ROWS);
    return t;
}

__device__ __forceinline__ void tc_mma_pair_elected(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The result [E, OUT, IN]: boxes of 32 rows x 64 columns that end with their expert, 128-byte swizzle.
static int encode_result(CUtensorMap* map, void* base, uint64_t E, uint64_t OUT, uint64_t IN, bool f16) {
    EncodeTiledFn fn = encode_fn();
    FMAB_REQUIRE(fn != nullptr, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {IN, OUT, E};
    const cuuint64_t strides[2] = {IN * 2, OUT * IN * 2};
    const cuuint32_t box[3] = {64, 32, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FMAB_REQUIRE(r == CUDA_SUCCESS, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled (weight gradient) failed with CUresult %d", (int)r);
    return FMA_B200_OK;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(WG_THREADS, 1) linear_wgrad_kernel(const __grid_constant__ WgradParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[WG_STAGES][2];  // per half of 64 rows; used in the leader only
    __shared__ __align__(8) uint64_t empty_bar[WG_STAGES];  // each CTA waits on its own copy
    __shared__ __align__(8) uint64_t acc_full_bar[2];       // each CTA waits on its own copy
    __shared__ __align__(8) uint64_t acc_empty_bar[2];      // used in the leader only
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t patches = ring + WG_STAGES * WG_STAGE_BYTES;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < WG_STAGES; ++s) {
            mbar_init(smem_u32(&full_bar[s][0]), 1);
            mbar_init(smem_u32(&full_bar[s][1]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&acc_full_bar[b]), 1);
            mbar_init(smem_u32(&acc_empty_bar[b]), 2 * WG_EPI_WARPS);  // every epilogue warp of both CTAs
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {  // the same warp of both CTAs takes part in the paired allocation
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the peer's barriers exist before anything is signalled across CTAs
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    volatile int* abort_ptr = &abort_flag;
    const int total_tiles = p.E * p.m_tiles * p.n_tiles;
    const int pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

    if (warp == 0) {
        // ------------------------------ TMA producer (both CTAs) ------------------------------
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool alive = true;
            for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
                const WgradTile t = wgrad_decode(p, tile);
                const int am = t.m0 + static_cast<int>(rank) * 128, bn = t.n0 + static_cast<int>(rank) * 128;
                for (int h0 = 0; h0 < t.halves; h0 += 2) {
                    if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    const int n_halves = min(2, t.halves - h0);
                    const uint32_t sa = ring + stage * WG_STAGE_BYTES, sb = sa + 2 * WG_SLAB;
                    for (int h = 0; h < n_halves; ++h) {
                        const uint32_t leader_bar = map_to_rank(smem_u32(&full_bar[stage][h]), 0);
                        if (leader) mbar_arrive_expect_tx(smem_u32(&full_bar[stage][h]), 2 * 2 * WG_SLAB);
                        const int row = t.row0 + (h0 + h) * WG_HALF_ROWS;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            tma_load_2d_pair(sa + h * WG_SLAB + j * (WG_SLAB / 2), &p.map_a, leader_bar, am + 64 * j, row);
                            tma_load_2d_pair(sb + h * WG_SLAB + j * (WG_SLAB / 2), &p.map_b, leader_bar, bn + 64 * j, row);
                        }
                    }
                    if (++stage == WG_STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!alive) {
                for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land
            }
        }
    } else if (warp == 1) {
        // ------------------------------ MMA issuer (leader CTA only) ------------------------------
        if (leader) {
            const uint32_t fmt = p.f16 ? 0u : 1u;  // operand format: IEEE half or bfloat16
            const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) |
                                   (static_cast<uint32_t>(256 >> 3) << 17) | (static_cast<uint32_t>(256 >> 4) << 24);
            int stage = 0;
            uint32_t phases[2] = {0, 0};  // of the halves' barriers, a bit per stage
            uint32_t n_done = 0;  // tiles with MMAs so far: accumulator n_done % 2
            bool alive = true;
            for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
                const WgradTile t = wgrad_decode(p, tile);
                if (t.halves == 0) continue;
                if (n_done >= 2 && !mbar_wait_warp(smem_u32(&acc_empty_bar[n_done & 1u]), ((n_done >> 1) - 1) & 1u, abort_ptr, p.status)) break;
                tc_fence_after();
                const uint32_t acc = tmem_base + (n_done & 1u) * 256;
                for (int h0 = 0; h0 < t.halves && alive; h0 += 2) {
                    const uint32_t sa = ring + stage * WG_STAGE_BYTES;
                    const uint64_t a_desc = make_smem_desc<true>(sa), b_desc = make_smem_desc<true>(sa + 2 * WG_SLAB);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h0 + h >= t.halves || !alive) continue;
                        alive = mbar_wait_warp(smem_u32(&full_bar[stage][h]), (phases[h] >> stage) & 1u, abort_ptr, p.status);
                        if (!alive) continue;
                        phases[h] ^= 1u << stage;
                        tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < WG_HALF_ROWS / UMMA_K; ++ks) {
                            const uint32_t at = (h * WG_SLAB + ks * desc_k_step<true>()) / 16;
                            tc_mma_pair_elected(acc, a_desc + at, b_desc + at, idesc, (h0 | h | ks) != 0);
                        }
                    }
                    tc_commit_both(smem_u32(&empty_bar[stage]));
                    if (++stage == WG_STAGES) stage = 0;
                }
                // published last: once the epilogues have seen it no other signal of the tile is outstanding
                if (alive) tc_commit_both(smem_u32(&acc_full_bar[n_done & 1u]));
                ++n_done;
            }
        }
    } else {
        // ------------------------------ epilogue (both CTAs) ------------------------------
        const int quad = warp & 3;         // tensor-memory lanes this warp may read
        const int half = (warp - 2) >> 2;  // columns 0-127 or 128-255 of the tile
        const uint32_t patch = patches + (warp - 2) * WG_PATCH_BYTES;
        const bool f16 = p.f16 != 0;
        uint32_t n_done = 0;
        for (int tile = pair_id; tile < total_tiles; tile += n_pairs) {
            const WgradTile t = wgrad_decode(p, tile);
            const uint32_t acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + (n_done & 1u) * 256;
            if (t.halves > 0) {
                if (!mbar_wait_warp(smem_u32(&acc_full_bar[n_done & 1u]), (n_done >> 1) & 1u, abort_ptr, p.status)) break;
                tc_fence_after();
            }
            const int first_row = t.m0 + static_cast<int>(rank) * 128 + quad * 32;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {  // 32 columns each; two make a box
                const int c0 = half * 128 + i * 32;
                float v[32];
                if (t.halves > 0) {
                    tc_load_32(acc + c0, v);
                    if (i == 3) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_rank(smem_u32(&acc_empty_bar[n_done & 1u]), 0));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0.f;
                }
                if ((i & 1) == 0) {
                    if (lane == 0) bulk_wait_read_all();  // the previous box has left the patch
                    __syncwarp();
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) st_shared_16(patch_addr(patch, lane, (i & 1) * 4 + q), pack8(v + 8 * q, f16));
                if ((i & 1) == 1) {
                    fence_smem_to_async();
                    __syncwarp();
                    const int col = t.n0 + c0 - 32;
                    if (lane == 0 && first_row < p.OUT && col < p.IN) {
                        tma_store_3d(&p.map_out, patch, col, first_row, t.expert);
                        bulk_commit();
                    }
                }
            }
            if (t.halves > 0) ++n_done;
        }
        if (lane == 0) bulk_wait_all();
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA touches the pair's tensor memory or barriers after this point
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

}  // namespace fmab

extern "C" {

int fma_b200_linear_wgrad(const void* dY, const void* X, void* dW, int32_t dtype, int64_t rows, int32_t E, int32_t OUT,
                          int32_t IN, const int32_t* seg_offsets, const int32_t* seg_rows, void* stream) {
    using namespace fmab;
    FMAB_REQUIRE(dtype == FMA_B200_BF16 || dtype == FMA_B200_F16, FMA_B200_ERR_UNSUPPORTED, "dtype %d", dtype);
    FMAB_REQUIRE(rows >= 1 && rows < (1LL << 31) - 256, FMA_B200_ERR_BAD_ARG, "rows=%lld", (long long)rows);
    FMAB_REQUIRE(E >= 1 && E <= 1024, FMA_B200_ERR_BAD_ARG, "E=%d not in [1,1024]", E);
    FMAB_REQUIRE(OUT >= 8 && IN >= 8 && OUT % 8 == 0 && IN % 8 == 0 && OUT < (1 << 30) && IN < (1 << 30), FMA_B200_ERR_BAD_ARG,
                 "OUT=%d and IN=%d must be positive multiples of 8", OUT, IN);
    FMAB_REQUIRE(dW && dY && X && (seg_offsets || (E == 1 && !seg_rows)), FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(dY) && aligned16(X) && aligned16(dW), FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    WgradParams p;
    memset(&p, 0, sizeof(p));
    p.status = device_status_ptr();
    FMAB_REQUIRE(p.status != nullptr, FMA_B200_ERR_LAUNCH, "no device status word");
    p.f16 = dtype == FMA_B200_F16 ? 1 : 0;
    if (int rc = encode_2d(&p.map_a, dY, OUT, rows, OUT, 64, WG_HALF_ROWS, p.f16 != 0)) return rc;
    if (int rc = encode_2d(&p.map_b, X, IN, rows, IN, 64, WG_HALF_ROWS, p.f16 != 0)) return rc;
    if (int rc = encode_result(&p.map_out, dW, E, OUT, IN, p.f16 != 0)) return rc;
    p.offsets = seg_offsets;
    p.counts = seg_rows;
    p.rows = rows;
    p.E = E;
    p.OUT = OUT;
    p.IN = IN;
    p.m_tiles = (OUT + 255) / 256;
    p.n_tiles = (IN + 255) / 256;
    const int64_t total = static_cast<int64_t>(E) * p.m_tiles * p.n_tiles;
    FMAB_REQUIRE(total < (1LL << 31), FMA_B200_ERR_BAD_ARG, "too many tiles");
    static bool configured[64] = {false};  // per device: the attribute applies to the current device only
    const int dev = current_device_slot();
    FMAB_REQUIRE(dev >= 0, FMA_B200_ERR_LAUNCH, "no current CUDA device with an ordinal below 64");
    if (!configured[dev]) {
        FMAB_CUDA(cudaFuncSetAttribute(linear_wgrad_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WG_SMEM));
        configured[dev] = true;
    }
    const int64_t max_pairs = sm_count() >= 2 ? sm_count() / 2 : 1;
    const int pairs = static_cast<int>(total < max_pairs ? total : max_pairs);
    return launch_kernel("linear weight gradient", linear_wgrad_kernel, dim3(2 * pairs), WG_THREADS, WG_SMEM, 0,
                          static_cast<cudaStream_t>(stream), p);
}

}  // extern "C"
