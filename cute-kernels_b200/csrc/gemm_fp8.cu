// Grouped product of 8-bit operands with power-of-two block scales, on CTA pairs:
//   out[r, n] = sum over k-blocks b of sa[r, b] * sw[n, b] * sum_{k in b} a[r, k] * w[e(r), n, k]
// with a in e4m3 with a scale per (row, 128 columns) and w in e4m3 with a scale per 128 x 128 block (fp8.cuh).  Scaling,
// products and sums happen in the tensor core (tcgen05.mma kind::mxf8f6f4 with block scaling, fp32 accumulators in
// tensor memory); the result is rounded once, to bfloat16 or half.
//
// The instruction wants one scale per 32 columns and row; it picks one of the four bytes of a 32-bit tensor-memory
// word by an index in its descriptor.  With one scale per 128 columns the four bytes hold four consecutive k-blocks:
// all four MMAs of k-block b use byte b % 4, so scales enter shared memory and tensor memory once per 512 columns
// (512 bytes per 128 rows) and are never replicated along k.
//
// Structure as in gemm_tc2.cu: cluster of two CTAs, one persistent pair per two SMs, warp 0 = TMA producer, warp 1 of
// the leader = MMA issuer, warps 2-9 = epilogue.  What bounds it is the traffic from L2 to the SMs (an 8-bit MMA
// consumes its operands in half the time of a 16-bit one), so the pair tile is as wide as tensor memory allows next to
// the scales: 256 rows x 384 columns (a 256-column and a 128-column accumulator), 80 KB of operands per 25 MFLOP
// instead of 64 KB per 17 MFLOP with 256 x 256.
#include "fp8.cuh"
#include "gemm_pair.cuh"

namespace fmab {

constexpr int BK8 = 128;                          // reduction elements per stage = one 128-byte swizzle row
constexpr int UMMA_K8 = 32;
constexpr int F8_THREADS = 320;
constexpr int F8_EPI_WARPS = 8;
constexpr int F8_A_BYTES = 128 * BK8;             // this CTA's 128 rows
constexpr int F8_SCALE_SLOT = 2048;               // per stage: 512 bytes for A, 512 per 128 columns for B
constexpr int F8_PATCH_BYTES = 32 * 128;
constexpr int F8_SUPER = 8;                       // pair m-tiles walked together (operand reuse in L2)

// PARTS accumulators: 256 columns, and with two parts 128 more.
template <int PARTS>
struct F8Tile {
    static constexpr int N = PARTS == 2 ? 384 : 256;
    static constexpr int B_BYTES = N / 2 * BK8;   // this CTA's half of every part
    static constexpr int STAGE_BYTES = F8_A_BYTES + B_BYTES;
    static constexpr int STAGES = PARTS == 2 ? 4 : 5;
    static constexpr int SCALE_TILES = N / 128;
    static constexpr int SCALE_BYTES = 512 * (1 + SCALE_TILES);
    static constexpr size_t SMEM = static_cast<size_t>(STAGES) * (STAGE_BYTES + F8_SCALE_SLOT) +
                                   F8_EPI_WARPS * F8_PATCH_BYTES + 1024;
};
constexpr int F8_SCALE_COL = 384;                 // tensor-memory column of the first scale buffer
constexpr int F8_SCALE_COLS = 16;                 // A: 4 columns, B: 4 per 128 columns
// A scale buffer is written again four 512-column groups later.  The MMAs that read it last have completed by then:
// the copy follows a wait for a refilled ring stage (at most 5 k-blocks back) or for an empty accumulator.
constexpr int F8_SCALE_BUFFERS = 4;

struct GemmFp8Params {
    CUtensorMap map_a, map_b0, map_b1, map_sa, map_sb;
    void* out;
    const int32_t* tile_expert;  // per 128-row tile: expert, -1 = unused, -2 = rows of no expert (zeros); null: one expert
    const int32_t* tile_row;     // per 128-row tile: first output row; null: tile * 128
    const int32_t* tile_rows;    // per 128-row tile: output rows; null: up to out_rows
    const int32_t* rows_used;    // rows of the layout in use (device); null: layout_rows
    int32_t* status;
    int64_t out_rows;
    int64_t ldd;
    int64_t layout_rows;
    int32_t n_cols, k_blocks, n_ntiles;
    int32_t b_rows;              // rows of w per expert
    int32_t sa_tiles;            // scale tiles per quad of A, and of w; of w per expert
    int32_t sb_tiles, sb_tiles_expert;
    int32_t f16;
};

__device__ __forceinline__ uint64_t f8_operand_desc(uint32_t addr) {  // K-major, 128-byte swizzle
    return make_smem_desc<false>(addr);
}
// 32 rows x 16 bytes without swizzle: 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t f8_scale_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (8ull << 16) | (8ull << 32) | (1ull << 46);
}
__device__ __forceinline__ void tc_copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
// M = 256, e4m3 operands, ue8m0 scales; scale_byte = which byte of the scale words.
__device__ __forceinline__ uint32_t f8_instr_desc(int n, uint32_t scale_byte) {
    return (scale_byte << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(256 >> 4) << 24) |
           (scale_byte << 29);
}

struct F8PairTile {
    int32_t expert;
    int32_t a_row;       // this CTA's first row of A
    int32_t n0;
    int32_t parts;       // parts with columns
    int32_t rows;        // output rows of this CTA
    int64_t out_row;
};

template <int PARTS>
__device__ __forceinline__ bool f8_decode(const GemmFp8Params& p, int tile, int n_pairs_m, uint32_t rank, F8PairTile& t) {
    const int per_super = F8_SUPER * p.n_ntiles;
    const int super = tile / per_super;
    const int m_first = super * F8_SUPER;
    const int m_span = min(F8_SUPER, n_pairs_m - m_first);
    const int r = tile - super * per_super;
    const int nt = r / m_span;
    const int pm = m_first + (r - nt * m_span);
    const int mt = 2 * pm + static_cast<int>(rank);
    t.expert = p.tile_expert != nullptr ? __ldg(p.tile_expert + 2 * pm) : 0;
    if (t.expert == -1) return false;
    t.a_row = mt * 128;
    t.n0 = nt * F8Tile<PARTS>::N;
    t.parts = (PARTS == 2 && t.n0 + 256 < p.n_cols) ? 2 : 1;
    t.out_row = p.tile_row != nullptr ? __ldg(p.tile_row + mt) : static_cast<int64_t>(mt) * 128;
    const int64_t left = p.tile_rows != nullptr ? __ldg(p.tile_rows + mt) : p.out_rows - t.out_row;
    t.rows = static_cast<int32_t>(left < 0 ? 0 : (left > 128 ? 128 : left));
    return true;
}

template <int PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F8_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ GemmFp8Params p) {
    using Tile = F8Tile<PARTS>;
    constexpr int STAGES = Tile::STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES];      // used in the leader only
    __shared__ __align__(8) uint64_t empty_bar[STAGES];     // each CTA waits on its own copy
    __shared__ __align__(8) uint64_t acc_full_bar[PARTS];   // each CTA waits on its own copy
    __shared__ __align__(8) uint64_t acc_empty_bar[PARTS];  // used in the leader only
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t scale_ring = ring + STAGES * Tile::STAGE_BYTES;
    const uint32_t patches = scale_ring + STAGES * F8_SCALE_SLOT;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int b = 0; b < PARTS; ++b) {
            mbar_init(smem_u32(&acc_full_bar[b]), 1);
            mbar_init(smem_u32(&acc_empty_bar[b]), 2 * F8_EPI_WARPS);  // every epilogue warp of both CTAs
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

    const int64_t rows_used = p.rows_used != nullptr ? min(p.layout_rows, static_cast<int64_t>(__ldg(p.rows_used))) : p.layout_rows;
    const int n_pairs_m = static_cast<int>((rows_used + 255) / 256);
    const int total_tiles = n_pairs_m * p.n_ntiles;
    const int pair_id = blockIdx.x >> 1;
    const int n_pairs = gridDim.x >> 1;

    if (warp == 0) {
        // ------------------------------ TMA producer (both CTAs) ------------------------------
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool alive = true;
            for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
                F8PairTile t;
                if (!f8_decode<PARTS>(p, tile, n_pairs_m, rank, t) || t.expert < 0) continue;
                const int b_row = t.expert * p.b_rows + t.n0;
                const int sb_tile = t.expert * p.sb_tiles_expert + t.n0 / 128;
                const uint32_t operand_bytes = F8_A_BYTES + (t.parts == 2 ? Tile::B_BYTES : 128 * BK8);
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    const bool scales = (kb & 3) == 0;
                    const uint32_t leader_bar = map_to_rank(smem_u32(&full_bar[stage]), 0);
                    const uint32_t sa = ring + stage * Tile::STAGE_BYTES;
                    const uint32_t sb = sa + F8_A_BYTES;
                    if (leader)
                        mbar_arrive_expect_tx(smem_u32(&full_bar[stage]), 2 * (operand_bytes + (scales ? Tile::SCALE_BYTES : 0)));
                    if (scales) {
                        const uint32_t ss = scale_ring + stage * F8_SCALE_SLOT;
                        tma_load_2d_pair(ss, &p.map_sa, leader_bar, 0, (kb >> 2) * p.sa_tiles + t.a_row / 128);
                        tma_load_2d_pair(ss + 512, &p.map_sb, leader_bar, 0, (kb >> 2) * p.sb_tiles + sb_tile);
                    }
                    tma_load_2d_pair(sa, &p.map_a, leader_bar, kb * BK8, t.a_row);
                    tma_load_2d_pair(sb, &p.map_b0, leader_bar, kb * BK8, b_row + static_cast<int>(rank) * 128);
                    if (t.parts == 2)
                        tma_load_2d_pair(sb + 128 * BK8, &p.map_b1, leader_bar, kb * BK8, b_row + 256 + static_cast<int>(rank) * 64);
                    if (++stage == STAGES) {
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
        if (leader && lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            uint32_t acc_phase = 0;
            uint32_t part1_phase = 0;
            int group = 0;  // 512-column groups so far: scale buffer
            bool alive = true;
            for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
                F8PairTile t;
                if (!f8_decode<PARTS>(p, tile, n_pairs_m, rank, t) || t.expert < 0) continue;
                uint32_t scales = 0;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait(smem_u32(&full_bar[stage]), phase, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    if (kb == 0) {
                        if (!mbar_wait(smem_u32(&acc_empty_bar[0]), acc_phase ^ 1u, abort_ptr, p.status)) {
                            alive = false;
                            break;
                        }
                        tc_fence_after();
                    }
                    if ((kb & 3) == 0) {
                        scales = tmem_base + F8_SCALE_COL + (group % F8_SCALE_BUFFERS) * F8_SCALE_COLS;
                        ++group;
                        const uint32_t ss = scale_ring + stage * F8_SCALE_SLOT;
#pragma unroll
                        for (int i = 0; i < 1 + Tile::SCALE_TILES; ++i)
                            tc_copy_scales_pair(scales + 4 * i, f8_scale_desc(ss + 512 * i));
                    }
                    const uint32_t sa = ring + stage * Tile::STAGE_BYTES;
                    const uint64_t a_desc = f8_operand_desc(sa);
                    const uint64_t b_desc = f8_operand_desc(sa + F8_A_BYTES);
                    const uint32_t byte = kb & 3;
#pragma unroll
                    for (int ks = 0; ks < BK8 / UMMA_K8; ++ks)
                        tc_mma_f8_pair(tmem_base, a_desc + ks * (UMMA_K8 >> 4), b_desc + ks * (UMMA_K8 >> 4),
                                       f8_instr_desc(256, byte), scales, scales + 4, (kb | ks) != 0);
                    const bool last = kb == p.k_blocks - 1;
                    if (last && t.parts == 2) tc_commit_pair(smem_u32(&acc_full_bar[0]));
                    if (PARTS == 2 && t.parts == 2) {
                        if (kb == 0) {
                            if (!mbar_wait(smem_u32(&acc_empty_bar[PARTS - 1]), part1_phase ^ 1u, abort_ptr, p.status)) {
                                alive = false;
                                break;
                            }
                            tc_fence_after();
                        }
                        const uint64_t b1_desc = f8_operand_desc(sa + F8_A_BYTES + 128 * BK8);
#pragma unroll
                        for (int ks = 0; ks < BK8 / UMMA_K8; ++ks)
                            tc_mma_f8_pair(tmem_base + 256, a_desc + ks * (UMMA_K8 >> 4), b1_desc + ks * (UMMA_K8 >> 4),
                                           f8_instr_desc(128, byte), scales, scales + 12, (kb | ks) != 0);
                    }
                    tc_commit_pair(smem_u32(&empty_bar[stage]));
                    // the accumulator that is finished last is published last: no signal of this tile is outstanding
                    // once the epilogues have seen it
                    if (last) tc_commit_pair(smem_u32(&acc_full_bar[t.parts - 1]));
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                acc_phase ^= 1u;
                if (t.parts == 2) part1_phase ^= 1u;
            }
        }
    } else {
        // ------------------------------ epilogue (both CTAs) ------------------------------
        const int quad = warp & 3;               // tensor-memory lanes this warp may read
        const int half = (warp - 2) >> 2;        // half of a part's columns
        const uint32_t patch = patches + (warp - 2) * F8_PATCH_BYTES;
        const bool f16 = p.f16 != 0;
        uint16_t* const out = static_cast<uint16_t*>(p.out);
        uint32_t acc_phase[2] = {0, 0};
        bool alive = true;
        for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
            F8PairTile t;
            if (!f8_decode<PARTS>(p, tile, n_pairs_m, rank, t)) continue;
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                if (part >= t.parts) continue;
                constexpr int kMaxLoads = 4;
                const int loads = part == 0 ? 4 : 2;                 // 32-column loads per warp
                const int c_first = part * 256 + half * loads * 32;  // accumulator column of this warp's first
                uint32_t packed[kMaxLoads * 16];
                if (t.expert >= 0) {
                    if (!mbar_wait(smem_u32(&acc_full_bar[part]), acc_phase[part], abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    acc_phase[part] ^= 1u;
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < kMaxLoads; ++j) {
                        if (j >= loads) continue;
                        float v[32];
                        tc_load_32(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + c_first + j * 32, v);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 w = pack8(v + 8 * i, f16);
                            packed[j * 16 + 4 * i] = w.x;
                            packed[j * 16 + 4 * i + 1] = w.y;
                            packed[j * 16 + 4 * i + 2] = w.z;
                            packed[j * 16 + 4 * i + 3] = w.w;
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster_relaxed(map_to_rank(smem_u32(&acc_empty_bar[part]), 0));
                } else {
#pragma unroll
                    for (int i = 0; i < kMaxLoads * 16; ++i) packed[i] = 0;
                }
#pragma unroll
                for (int j = 0; j < kMaxLoads; j += 2) {  // 64 columns at a time through the patch
                    if (j >= loads) continue;
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        st_shared_16(patch_addr(patch, lane, i), make_uint4(packed[j * 16 + 4 * i], packed[j * 16 + 4 * i + 1],
                                                                            packed[j * 16 + 4 * i + 2], packed[j * 16 + 4 * i + 3]));
                    __syncwarp();
                    const int col = t.n0 + c_first + j * 32 + (lane & 7) * 8;
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int row = it * 4 + (lane >> 3);
                        const uint4 w = ld_shared_16(patch_addr(patch, row, lane & 7));
                        if (quad * 32 + row < t.rows && col < p.n_cols)
                            st_global_16(out + (t.out_row + quad * 32 + row) * p.ldd + col, w);
                    }
                }
            }
        }
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

// ---- host side -------------------------------------------------------------------------------------
// Bytes [outer, inner] with row pitch `pitch`, boxes of box_outer rows x 128 bytes, 128-byte swizzle.
static int encode_bytes(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer, uint64_t pitch, uint32_t box_outer) {
    EncodeTiledFn fn = encode_fn();
    FMAB_REQUIRE(fn != nullptr, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {inner, outer};
    const cuuint64_t strides[1] = {pitch};
    const cuuint32_t box[2] = {BK8, box_outer};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FMAB_REQUIRE(r == CUDA_SUCCESS, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled (8-bit operand) failed with CUresult %d", (int)r);
    return FMA_B200_OK;
}
// Scale tiles as rows of 128 words, boxes of `tiles` rows.
static int encode_scales(CUtensorMap* map, const void* base, uint64_t n_tiles, uint32_t tiles) {
    EncodeTiledFn fn = encode_fn();
    FMAB_REQUIRE(fn != nullptr, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {FP8_TILE_BYTES / 4, n_tiles};
    const cuuint64_t strides[1] = {FP8_TILE_BYTES};
    const cuuint32_t box[2] = {FP8_TILE_BYTES / 4, tiles};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FMAB_REQUIRE(r == CUDA_SUCCESS, FMA_B200_ERR_LAUNCH, "cuTensorMapEncodeTiled (scales) failed with CUresult %d", (int)r);
    return FMA_B200_OK;
}

template <int PARTS>
static int launch_fp8(GemmFp8Params& p, cudaStream_t s) {
    using Tile = F8Tile<PARTS>;
    static bool configured[64] = {false};  // per device: the attribute applies to the current device only
    auto kernel = gemm_fp8_kernel<PARTS>;
    const int dev = current_device_slot();
    FMAB_REQUIRE(dev >= 0, FMA_B200_ERR_LAUNCH, "no current CUDA device with an ordinal below 64");
    if (!configured[dev]) {
        FMAB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Tile::SMEM));
        configured[dev] = true;
    }
    p.n_ntiles = (p.n_cols + Tile::N - 1) / Tile::N;
    const int64_t total = (p.layout_rows + 255) / 256 * p.n_ntiles;
    FMAB_REQUIRE(total < (1LL << 31), FMA_B200_ERR_BAD_ARG, "too many tiles");
    const int64_t max_pairs = sm_count() / 2;
    const int pairs = static_cast<int>(total < max_pairs ? total : max_pairs);
    kernel<<<2 * pairs, F8_THREADS, Tile::SMEM, s>>>(p);
    return check_launch("8-bit grouped GEMM");
}

}  // namespace fmab

extern "C" {

int fma_b200_fp8_gemm(const void* a, const void* a_scales, int64_t layout_rows, const void* w, const void* w_scales,
                      int32_t E, int32_t N, int32_t K, void* out, int32_t dtype, int64_t out_rows,
                      const int32_t* tile_expert, const int32_t* tile_row, const int32_t* tile_rows,
                      const int32_t* rows_used, void* stream) {
    using namespace fmab;
    FMAB_REQUIRE(dtype == FMA_B200_BF16 || dtype == FMA_B200_F16, FMA_B200_ERR_UNSUPPORTED,
                 "dtype %d: the 8-bit product returns bfloat16 or half", dtype);
    FMAB_REQUIRE(layout_rows >= 0 && layout_rows < (1LL << 31) - 256 && out_rows >= 0, FMA_B200_ERR_BAD_ARG,
                 "layout_rows=%lld, out_rows=%lld", (long long)layout_rows, (long long)out_rows);
    FMAB_REQUIRE(E >= 1 && E <= 1024, FMA_B200_ERR_BAD_ARG, "E=%d not in [1,1024]", E);
    FMAB_REQUIRE(N >= 8 && K >= 8 && N % 8 == 0 && K % 8 == 0 && N < (1 << 30) && K < (1 << 30), FMA_B200_ERR_BAD_ARG,
                 "N=%d and K=%d must be positive multiples of 8", N, K);
    FMAB_REQUIRE(static_cast<int64_t>(E) * N < (1LL << 31) - 1024, FMA_B200_ERR_BAD_ARG, "E*N overflows");
    FMAB_REQUIRE(E == 1 || tile_expert != nullptr, FMA_B200_ERR_BAD_ARG, "several experts need tile_expert");
    if (layout_rows == 0 || out_rows == 0) return FMA_B200_OK;
    FMAB_REQUIRE(a && a_scales && w && w_scales && out, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(a) && aligned16(a_scales) && aligned16(w) && aligned16(w_scales) && aligned16(out),
                 FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    GemmFp8Params p;
    memset(&p, 0, sizeof(p));
    p.status = device_status_ptr();
    FMAB_REQUIRE(p.status != nullptr, FMA_B200_ERR_LAUNCH, "no device status word");
    p.out = out;
    p.tile_expert = tile_expert;
    p.tile_row = tile_row;
    p.tile_rows = tile_rows;
    p.rows_used = rows_used;
    p.out_rows = out_rows;
    p.ldd = N;
    p.layout_rows = layout_rows;
    p.n_cols = N;
    p.k_blocks = (K + BK8 - 1) / BK8;
    p.b_rows = N;
    p.sa_tiles = static_cast<int32_t>(fp8_row_tiles(layout_rows));
    p.sb_tiles_expert = static_cast<int32_t>(fp8_row_tiles(N));
    p.sb_tiles = E * p.sb_tiles_expert;
    p.f16 = dtype == FMA_B200_F16 ? 1 : 0;
    const int64_t quads = fp8_quads(K);
    if (int rc = encode_bytes(&p.map_a, a, K, layout_rows, fp8_pitch(K), 128)) return rc;
    if (int rc = encode_bytes(&p.map_b0, w, K, static_cast<uint64_t>(E) * N, fp8_pitch(K), 128)) return rc;
    if (int rc = encode_bytes(&p.map_b1, w, K, static_cast<uint64_t>(E) * N, fp8_pitch(K), 64)) return rc;
    if (int rc = encode_scales(&p.map_sa, a_scales, quads * p.sa_tiles, 1)) return rc;
    const bool wide = N > 256;
    if (int rc = encode_scales(&p.map_sb, w_scales, quads * p.sb_tiles, wide ? 3 : 2)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return wide ? launch_fp8<2>(p, s) : launch_fp8<1>(p, s);
}

}  // extern "C"
