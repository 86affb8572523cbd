// Grouped product of 8-bit operands with power-of-two block scales, on CTA pairs:
//   out[r, n] = sum over k-blocks b of sa[r, b] * sw[n, b] * sum_{k in b} a[r, k] * w[e(r), n, k]
// with a in e4m3 with a scale per (row, 128 columns) and w in e4m3 with a scale per 128 x 128 block (fp8.cuh).  Scaling,
// products and sums happen in the tensor core (tcgen05.mma kind::mxf8f6f4 with block scaling, fp32 accumulators in
// tensor memory); the result is rounded once, to bfloat16 or half.
//
// The instruction wants one scale per 32 columns and row; it picks one of the four bytes of a 32-bit tensor-memory
// word by an index in its descriptor.  With one scale per 128 columns the four bytes hold four consecutive k-blocks:
// all four MMAs of k-block b use byte b % 4, so scales enter tensor memory once per 512 columns (512 bytes per 128
// rows) and are never replicated along k.
//
// Structure as in gemm_tc2.cu: cluster of two CTAs, one persistent pair per two SMs, warp 0 = TMA producer, warp 1 of
// the leader = MMA issuer, warps 2-9 = epilogue; and warps 10-13 bring the scales from global memory straight into
// tensor memory (16 bytes per lane are the four rows whose words its lane holds).
//
// What bounds it is the tensor pipe, and what the pipe loses it loses to its command stream rather than to loads (the
// loads alone run at 3.5 PFLOP/s worth of operands).  Measured at 8192 x 4096 x 14336, one change after the other:
//   scales copied from shared memory with tcgen05.cp, which drains the pipe around it, two accumulators of 256 and 128
//   columns so that the operands are read least often, no overlap of the epilogue        486 us  1.98 PFLOP/s
//   one 256 x 256 accumulator (128-column MMAs run below the rate of 256-column ones)     444 us  2.17
//   scales through tcgen05.st, overlapping accumulators                                    436 us  2.21
//   one commit for both CTAs' barriers instead of two                                      418 us  2.30
//   the whole warp walks the loop and an elected lane issues                               365 us  2.64
//   ring stages of 256 columns: eight MMAs per wait and commit instead of four             324 us  2.97
// The library's 8-bit product without block scales takes 322 us on the same GPU.
//
// The pair tile is 256 rows x up to 256 columns.  Two 256-column accumulators and the scales do not fit into the 512
// columns of tensor memory, so the accumulators overlap by 32 columns: the epilogue reads the overlap first and hands
// it back at once, and the next tile's main loop starts while the rest is still being read and stored.
#include "fp8.cuh"
#include "gemm_pair.cuh"

namespace fmab {

// fp8_few.cu: the product by 128 weight rows and up to 128 rows of x
int fp8_some_rows(const void* x, const void* x_scales, int64_t layout_rows, const void* w, const void* w_scales, int32_t E, int32_t N,
                  int32_t K, void* out, int32_t dtype, int64_t out_rows, const int32_t* tile_expert, const int32_t* tile_row,
                  const int32_t* tile_rows, const int32_t* rows_used, int64_t active, cudaStream_t s);
bool fp8_some_rows_fits(int32_t K);

constexpr int BK8 = 128;                          // reduction elements per stage = one 128-byte swizzle row
constexpr int UMMA_K8 = 32;
constexpr int F8_EPI_WARPS = 8;
constexpr int F8_SCALE_WARPS = 4;
constexpr int F8_THREADS = 32 * (2 + F8_EPI_WARPS + F8_SCALE_WARPS);
constexpr int F8_TILE_N = 256;                    // widest tile
constexpr int F8_A_BYTES = 128 * BK8;             // this CTA's 128 rows
constexpr int F8_B_BYTES = F8_TILE_N / 2 * BK8;   // its half of the tile's columns
constexpr int F8_STAGE_KB = 2;                    // k-blocks per ring stage
constexpr int F8_STAGE_BYTES = F8_STAGE_KB * (F8_A_BYTES + F8_B_BYTES);
constexpr int F8_STAGES = 3;
constexpr int F8_PATCH_BYTES = 32 * 64;  // 32 rows x 32 columns of 16 bits per epilogue warp
constexpr size_t F8_SMEM = static_cast<size_t>(F8_STAGES) * F8_STAGE_BYTES + F8_EPI_WARPS * F8_PATCH_BYTES + 1024;
constexpr int F8_SUPER = 8;                       // pair m-tiles walked together (operand reuse in L2)
// tensor memory: accumulator 0 in columns 0-255, accumulator 1 in 224-479, two scale buffers of 12 columns (A: 4,
// B: 8) from 480 on
constexpr int F8_ACC1_COL = 224;
constexpr int F8_SCALE_COL = 480;
constexpr int F8_SCALE_COLS = 16;
constexpr int F8_SCALE_BUFFERS = 2;

struct GemmFp8Params {
    CUtensorMap map_a, map_b;
    const uint8_t* a_scales;
    const uint8_t* b_scales;
    void* out;
    const int32_t* tile_expert;  // per 128-row tile: expert, -1 = unused, -2 = rows of no expert (zeros); null: one expert
    const int32_t* tile_row;     // per 128-row tile: first output row; null: tile * 128
    const int32_t* tile_rows;    // per 128-row tile: output rows; null: up to out_rows
    const int32_t* rows_used;    // rows of the layout in use (device); null: layout_rows
    int32_t* status;
    int64_t out_rows;
    int64_t layout_rows;
    int32_t n_cols, k_blocks, n_ntiles;
    int32_t tile_n;              // columns per tile: a multiple of 32, at most 256
    int32_t a_tiles;             // scale tiles per quad of a
    int32_t b_tiles, b_tiles_expert;  // scale tiles per quad of w, and of one expert
    int32_t f16;
};

// Issued by one elected lane of a converged warp.
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
// M = 256, e4m3 operands, ue8m0 scales; scale_byte = which byte of the scale words.
__device__ __forceinline__ uint32_t f8_instr_desc(int n, uint32_t scale_byte) {
    return (scale_byte << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(256 >> 4) << 24) |
           (scale_byte << 29);
}
__device__ __forceinline__ void tc_store_4(uint32_t taddr, uint4 v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(taddr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}

struct F8PairTile {
    int32_t expert;
    int32_t a_row;       // this CTA's first row of A
    int32_t n0;
    int32_t rows;        // output rows of this CTA
    int64_t out_row;
};

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
    t.n0 = nt * p.tile_n;
    t.out_row = p.tile_row != nullptr ? __ldg(p.tile_row + mt) : static_cast<int64_t>(mt) * 128;
    const int64_t left = p.tile_rows != nullptr ? __ldg(p.tile_rows + mt) : p.out_rows - t.out_row;
    t.rows = static_cast<int32_t>(left < 0 ? 0 : (left > 128 ? 128 : left));
    return true;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F8_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ GemmFp8Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[F8_STAGES];            // used in the leader only
    __shared__ __align__(8) uint64_t empty_bar[F8_STAGES];           // each CTA waits on its own copy
    __shared__ __align__(8) uint64_t acc_full_bar[2];                // each CTA waits on its own copy
    __shared__ __align__(8) uint64_t acc_empty_bar;                  // used in the leader only
    __shared__ __align__(8) uint64_t scale_full_bar[F8_SCALE_BUFFERS];  // used in the leader only
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t patches = ring + F8_STAGES * F8_STAGE_BYTES;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < F8_STAGES; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        mbar_init(smem_u32(&acc_full_bar[0]), 1);
        mbar_init(smem_u32(&acc_full_bar[1]), 1);
        mbar_init(smem_u32(&acc_empty_bar), 2 * F8_EPI_WARPS);  // every epilogue warp of both CTAs
        for (int b = 0; b < F8_SCALE_BUFFERS; ++b) mbar_init(smem_u32(&scale_full_bar[b]), 2 * F8_SCALE_WARPS);
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
    allow_next();
    wait_for_previous();
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
            const uint32_t kb_bytes = F8_A_BYTES + p.tile_n / 2 * BK8;
            for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
                F8PairTile t;
                if (!f8_decode(p, tile, n_pairs_m, rank, t) || t.expert < 0) continue;
                const int b_row = t.expert * p.n_cols + t.n0 + static_cast<int>(rank) * (p.tile_n / 2);
                for (int kb = 0; kb < p.k_blocks; kb += F8_STAGE_KB) {
                    if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    const int n_kb = min(F8_STAGE_KB, p.k_blocks - kb);
                    const uint32_t leader_bar = map_to_rank(smem_u32(&full_bar[stage]), 0);
                    const uint32_t sa = ring + stage * F8_STAGE_BYTES;
                    const uint32_t sb = sa + F8_STAGE_KB * F8_A_BYTES;
                    if (leader) mbar_arrive_expect_tx(smem_u32(&full_bar[stage]), 2 * n_kb * kb_bytes);
                    for (int j = 0; j < n_kb; ++j) {
                        tma_load_2d_pair(sa + j * F8_A_BYTES, &p.map_a, leader_bar, (kb + j) * BK8, t.a_row);
                        tma_load_2d_pair(sb + j * F8_B_BYTES, &p.map_b, leader_bar, (kb + j) * BK8, b_row);
                    }
                    if (++stage == F8_STAGES) {
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
        // The whole warp walks the loop and one elected lane issues: descriptors then live in uniform registers.
        if (leader) {
            int stage = 0;
            uint32_t phase = 0;
            uint32_t sbuf = 0, sphase = 0;
            uint32_t n_done = 0;  // tiles so far: accumulator n_done % 2
            bool alive = true;
            for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
                F8PairTile t;
                if (!f8_decode(p, tile, n_pairs_m, rank, t) || t.expert < 0) continue;
                // the epilogues have read the columns that this accumulator shares with the previous one
                if (n_done > 0 && !mbar_wait(smem_u32(&acc_empty_bar), (n_done - 1) & 1u, abort_ptr, p.status)) break;
                tc_fence_after();
                const uint32_t acc = tmem_base + (n_done & 1u) * F8_ACC1_COL;
                for (int kb = 0; kb < p.k_blocks; kb += F8_STAGE_KB) {
                    if ((kb & 3) == 0 && !mbar_wait(smem_u32(&scale_full_bar[sbuf]), sphase, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    if (!mbar_wait(smem_u32(&full_bar[stage]), phase, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t scales = tmem_base + F8_SCALE_COL + sbuf * F8_SCALE_COLS;
                    const uint32_t sa = ring + stage * F8_STAGE_BYTES;
                    const uint64_t a_desc = make_smem_desc<false>(sa);
                    const uint64_t b_desc = make_smem_desc<false>(sa + F8_STAGE_KB * F8_A_BYTES);
#pragma unroll
                    for (int j = 0; j < F8_STAGE_KB; ++j) {
                        if (kb + j >= p.k_blocks) continue;
                        const uint32_t idesc = f8_instr_desc(p.tile_n, (kb + j) & 3);
#pragma unroll
                        for (int ks = 0; ks < BK8 / UMMA_K8; ++ks)
                            tc_mma_f8_pair(acc, a_desc + (j * F8_A_BYTES + ks * UMMA_K8) / 16,
                                           b_desc + (j * F8_B_BYTES + ks * UMMA_K8) / 16, idesc, scales, scales + 4,
                                           (kb | j | ks) != 0);
                    }
                    tc_commit_both(smem_u32(&empty_bar[stage]));
                    if ((kb & 3) == 4 - F8_STAGE_KB || kb + F8_STAGE_KB >= p.k_blocks) {
                        if (++sbuf == F8_SCALE_BUFFERS) {
                            sbuf = 0;
                            sphase ^= 1u;
                        }
                    }
                    if (++stage == F8_STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                // published last: once the epilogues have seen it no other signal of the tile is outstanding
                if (alive) tc_commit_both(smem_u32(&acc_full_bar[n_done & 1u]));
                ++n_done;
            }
        }
    } else if (warp < 2 + F8_EPI_WARPS) {
        // ------------------------------ epilogue (both CTAs) ------------------------------
        const int quad = warp & 3;               // tensor-memory lanes this warp may read
        const int half = (warp - 2) >> 2;        // columns 0-127 or 128-255 of the tile
        const uint32_t patch = patches + (warp - 2) * F8_PATCH_BYTES;
        const bool f16 = p.f16 != 0;
        uint16_t* const out = static_cast<uint16_t*>(p.out);
        uint32_t n_done = 0;
        for (int tile = pair_id; tile < total_tiles; tile += n_pairs) {
            F8PairTile t;
            if (!f8_decode(p, tile, n_pairs_m, rank, t)) continue;
            const uint32_t acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + (n_done & 1u) * F8_ACC1_COL;
            // the 32 columns of the overlap come first: the last ones of accumulator 0, the first ones of 1
            const bool backwards = half == 1 && (n_done & 1u) == 0;
            if (t.expert >= 0) {
                if (!mbar_wait(smem_u32(&acc_full_bar[n_done & 1u]), (n_done >> 1) & 1u, abort_ptr, p.status)) break;
                tc_fence_after();
            }
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                const int c0 = half * 128 + (backwards ? 3 - i : i) * 32;
                float v[32];
                if (t.expert >= 0) {
                    if (c0 < p.tile_n) tc_load_32(acc + c0, v);  // columns from tile_n on are never stored
                    if (i == 0) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_rank(smem_u32(&acc_empty_bar), 0));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0.f;
                }
                if (c0 >= p.tile_n) continue;
                // through the patch: 32 rows x 64 bytes, written a row per lane, read four lanes to a row
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    st_shared_16(patch + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4), pack8(v + 8 * q, f16));
                __syncwarp();
                const int cw = c0 + (lane & 3) * 8;
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const int row = it * 8 + (lane >> 2);
                    const uint4 w = ld_shared_16(patch + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4));
                    if (quad * 32 + row < t.rows && cw < p.tile_n && t.n0 + cw < p.n_cols)
                        st_global_16(out + (t.out_row + quad * 32 + row) * p.n_cols + t.n0 + cw, w);
                }
            }
            if (t.expert >= 0) ++n_done;
        }
    } else {
        // ------------------------------ scales (both CTAs) ------------------------------
        // All four warps bring the same words, each into its 32 lanes: word j of lane l is row j * 32 + l.  Rows of a
        // weight block share one word, so a tile may start anywhere in it.
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        // A buffer is free again when the MMAs of two groups ago are complete, which the release of the last ring
        // stage of that group tells: these warps follow the stage numbers and watch that barrier.  It cannot run a
        // phase ahead of them, since the MMAs of this group wait for them.
        constexpr int kStagesPerGroup = 4 / F8_STAGE_KB;
        uint32_t buf = 0;
        uint32_t n_stages = 0;              // ring stages up to the end of the previous group
        uint32_t ends[F8_SCALE_BUFFERS] = {0, 0};  // the same up to the end of the group that used each buffer last
        bool alive = true;
        for (int tile = pair_id; tile < total_tiles && alive; tile += n_pairs) {
            F8PairTile t;
            if (!f8_decode(p, tile, n_pairs_m, rank, t) || t.expert < 0) continue;
            const int a_tile = t.a_row / 128;
            for (int kb = 0; kb < p.k_blocks; kb += 4) {
                const int q = kb >> 2;
                const uint32_t one = 0x01010101u * FP8_SCALE_ONE;
                uint4 wa = make_uint4(one, one, one, one);
                if (a_tile < p.a_tiles)
                    wa = __ldg(reinterpret_cast<const uint4*>(p.a_scales + (static_cast<int64_t>(q) * p.a_tiles + a_tile) * FP8_TILE_BYTES) + lane);
                uint32_t wb[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int block = (t.n0 + j * 32 + lane) / FP8_BLOCK;
                    wb[j] = one;
                    if (block < p.b_tiles_expert)
                        wb[j] = __ldg(reinterpret_cast<const uint32_t*>(
                            p.b_scales + (static_cast<int64_t>(q) * p.b_tiles + t.expert * p.b_tiles_expert + block) * FP8_TILE_BYTES));
                }
                if (ends[buf] > 0) {
                    const uint32_t last = ends[buf] - 1;
                    if (!mbar_wait(smem_u32(&empty_bar[last % F8_STAGES]), (last / F8_STAGES) & 1u, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                }
                n_stages += min(kStagesPerGroup, (p.k_blocks - kb + F8_STAGE_KB - 1) / F8_STAGE_KB);
                ends[buf] = n_stages;
                tc_fence_after();
                __syncwarp();
                const uint32_t at = tmem_base + lanes + F8_SCALE_COL + buf * F8_SCALE_COLS;
                tc_store_4(at, wa);
                tc_store_4(at + 4, make_uint4(wb[0], wb[1], wb[2], wb[3]));
                tc_store_4(at + 8, make_uint4(wb[4], wb[5], wb[6], wb[7]));
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(map_to_rank(smem_u32(&scale_full_bar[buf]), 0));
                buf ^= 1u;
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
// Columns per tile.  Few wide tiles read A least often; but the launch takes as long as its fullest pair of SMs, so
// where the number of row tiles is known (no experts) the width that makes waves * (width + 24) smallest is taken, 24
// columns standing for what a tile costs besides its columns: a prompt of up to 256 rows spreads over all SMs (256 x
// 4096 x 4096: 13.7 us, with 256 columns 15.7; 2048 x 2048 x 1536: 10.7 and 11.6; no difference from two waves on).
// With experts only the waste at the right edge is known: the tiles share it (520 columns: three tiles of 192, not
// 256 + 256 + 8).
static int tile_columns(int64_t layout_rows, int N, bool experts) {
    const int64_t pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1, m = (layout_rows + 255) / 256;
    const int fewest = (N + F8_TILE_N - 1) / F8_TILE_N;
    int best = 0;
    int64_t best_cost = 0;
    for (int n = fewest; n <= N / 64 + 1; ++n) {
        const int width = ((N + n - 1) / n + 31) / 32 * 32;  // paired MMAs take whole 32 columns
        const int64_t tiles = (N + width - 1) / width;
        const int64_t cost = (m * tiles + pairs - 1) / pairs * (width + 24);
        if (best == 0 || cost < best_cost) {
            best = width;
            best_cost = cost;
        }
        if (experts || m * n > 16 * pairs) break;  // many waves: the widest tile
    }
    return best;
}

// Whether tiles of 128 weight rows and up to 128 rows of x, spread over clusters along k, are the faster way.  Measured,
// x quantised in both: 4096 x 4096, 32 / 64 / 96 rows 8.7 / 10.1 / 11.3 us against 14.7 / 15.1 / 15.3 with pair tiles;
// 14336 x 4096 (many tiles, little to split) 18.4 / 19.9 / 22.0 against 19.3 / 19.6 / 19.9; 4096 x 14336 18.2 / 20.1 / 22.6
// and 25.1 for 128 rows against 36.2 to 37.3; 128 experts of 1536 x 2048, 16 / 32 / 64 rows each 95 / 100 / 116 against
// 105 / 107 / 115.
static bool some_rows_suit(int64_t layout_rows, int64_t out_rows, int32_t E, int32_t N, int32_t K, bool experts, bool tile_rows) {
    if (!fp8_some_rows_fits(K)) return false;
    if (!experts) return layout_rows <= 64 || (layout_rows <= 96 && K >= N) || (layout_rows <= 128 && K >= 2LL * N);
    return tile_rows && out_rows <= 48LL * E;  // without tile_rows the rows of a layout are not known here
}

static int launch_fp8(GemmFp8Params& p, cudaStream_t s) {
    static bool configured[64] = {false};  // per device: the attribute applies to the current device only
    const int dev = current_device_slot();
    FMAB_REQUIRE(dev >= 0, FMA_B200_ERR_LAUNCH, "no current CUDA device with an ordinal below 64");
    if (!configured[dev]) {
        FMAB_CUDA(cudaFuncSetAttribute(gemm_fp8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F8_SMEM));
        configured[dev] = true;
    }
    const int64_t total = (p.layout_rows + 255) / 256 * p.n_ntiles;
    FMAB_REQUIRE(total < (1LL << 31), FMA_B200_ERR_BAD_ARG, "too many tiles");
    const int64_t max_pairs = sm_count() >= 2 ? sm_count() / 2 : 1;
    const int pairs = static_cast<int>(total < max_pairs ? total : max_pairs);
    return launch_chained("8-bit grouped GEMM", gemm_fp8_kernel, dim3(2 * pairs), F8_THREADS, F8_SMEM, 0, s, p);
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
    if (some_rows_suit(layout_rows, out_rows, E, N, K, tile_expert != nullptr, tile_rows != nullptr))
        return fp8_some_rows(a, a_scales, layout_rows, w, w_scales, E, N, K, out, dtype, out_rows, tile_expert, tile_row, tile_rows,
                             rows_used, tile_expert != nullptr ? (E < out_rows ? E : out_rows) : 1, static_cast<cudaStream_t>(stream));
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
    p.layout_rows = layout_rows;
    p.n_cols = N;
    p.k_blocks = (K + BK8 - 1) / BK8;
    p.tile_n = tile_columns(layout_rows, N, tile_expert != nullptr);
    p.n_ntiles = (N + p.tile_n - 1) / p.tile_n;
    p.a_scales = static_cast<const uint8_t*>(a_scales);
    p.b_scales = static_cast<const uint8_t*>(w_scales);
    p.a_tiles = static_cast<int32_t>(fp8_row_tiles(layout_rows));
    p.b_tiles_expert = static_cast<int32_t>(fp8_row_tiles(N));
    p.b_tiles = E * p.b_tiles_expert;
    p.f16 = dtype == FMA_B200_F16 ? 1 : 0;
    if (int rc = encode_bytes(&p.map_a, a, K, layout_rows, fp8_pitch(K), 128)) return rc;
    if (int rc = encode_bytes(&p.map_b, w, K, static_cast<uint64_t>(E) * N, fp8_pitch(K), p.tile_n / 2)) return rc;
    return launch_fp8(p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
