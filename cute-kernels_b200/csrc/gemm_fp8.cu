// Grouped product of 8-bit operands with power-of-two block scales, on CTA pairs:
//   out[r, n] = sum over k-blocks b of sa[r, b] * sw[n, b] * sum_{k in b} a[r, k] * w[e(r), n, k]
// with a in e4m3 with a scale per (row, 128 columns) and w in e4m3 with a scale per 128 x 128 block (fp8.cuh).  Scaling,
// products and sums happen in the tensor core (tcgen05.mma kind::mxf8f6f4 with block scaling, fp32 accumulators in
// tensor memory); the result is rounded once, to bfloat16 or half.  And its input gradient, where the sum runs over the
// weights' rows: the instruction takes that operand as it lies (TURNED: 128 columns x 128 rows per k-block, MN-major), with
// scale words put together from four scale tiles.  Measured against a transposed copy of the weights, 8192 x 14336 x
// 4096: 346 us and 348, 128 experts of 1536 x 2048 with 64 / 256 / 512 / 1024 rows 92 / 145 / 217 / 393 and 89 / 142 / 216 / 391;
// without the copy, quantising those 128 experts' weights writes 0.4 GB less.
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
// The pair tile is 256 weight rows (the instruction's rows) x up to 256 rows of a (its columns, in steps of 32): an
// expert's last tile is as high as it has rows left.  With the operands the other way round every expert's rows were
// padded to 256; 128 experts of 1536 x 2048 with 52 / 128 / 512 rows each on average took 104 / 108 / 201 us so and take
// 94 / 100 / 193 now, 8 of 14336 x 4096 with 1024 rows 381 and 367; plain products are the same both ways.  A low tile
// saves less than its MMAs: it loads 128 weight rows per CTA all the same, and a full one already loads near L2's rate.
//
// The result lies in tensor memory a weight row per lane.  It is read as fragments of 8 x 8 matrices, turned by the matrix
// store into shared memory and leaves through the copy engine in boxes of 32 rows x 32 columns; only where an expert ends
// inside a box the rows are stored one by one.  128 experts of 2048 x 768 (short sums, so the way out counts) with 512 / 2048
// rows each: 150 / 487 us with two-byte stores into the patch, 135 / 437 with matrix stores, 128 / 415 with the copy engine;
// 1536 x 2048 193 / 658 and 189 / 642.
//
// Two 256-column accumulators and the scales do not fit into the 512 columns of tensor memory, so the accumulators
// overlap by 32 columns: the epilogue reads the overlap first and hands it back at once, and the next tile's main loop
// starts while the rest is still being read and stored.
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
constexpr int F8_TILE_ROWS = 256;                 // most rows of a per tile
constexpr int F8_W_BYTES = 128 * BK8;             // this CTA's 128 weight rows
constexpr int F8_X_BYTES = F8_TILE_ROWS / 2 * BK8;  // its half of the tile's rows of a
constexpr int F8_STAGE_KB = 2;                    // k-blocks per ring stage
constexpr int F8_STAGE_BYTES = F8_STAGE_KB * (F8_W_BYTES + F8_X_BYTES);
constexpr int F8_STAGES = 3;
constexpr int F8_PATCH_BYTES = 32 * 64;           // 32 rows of a x 32 weight rows, 16 bits; two per epilogue warp
constexpr size_t F8_SMEM = static_cast<size_t>(F8_STAGES) * F8_STAGE_BYTES + 2 * F8_EPI_WARPS * F8_PATCH_BYTES + 1024;
constexpr int F8_SUPER = 8;                       // tiles of rows of a walked together (operand reuse in L2)
constexpr int F8_BOXES = 4;                       // rows of a come in boxes of 16, 32, 64 or 128
// tensor memory: accumulator 0 in columns 0-255, accumulator 1 in 224-479, two scale buffers of 12 columns (weights 4,
// rows of a 8) from 480 on
constexpr int F8_ACC1_COL = 224;
constexpr int F8_SCALE_COL = 480;
constexpr int F8_SCALE_COLS = 16;
constexpr int F8_SCALE_BUFFERS = 2;

struct GemmFp8Params {
    CUtensorMap map_w;            // TURNED: [expert, reduction, columns], so that a box does not reach into the next expert
    CUtensorMap map_a[F8_BOXES];
    CUtensorMap map_out;          // boxes of 32 rows x 32 columns
    const uint8_t* a_scales;
    const uint8_t* w_scales;
    void* out;
    const int32_t* tile_expert;  // per 128 rows of a: expert, -1 = unused, -2 = rows of no expert (zeros); null: one expert
    const int32_t* tile_row;     // per 128 rows of a: first output row; null: the same row
    const int32_t* tile_rows;    // per 128 rows of a: output rows; null: up to out_rows
    const int32_t* rows_used;    // rows of the layout in use (device); null: layout_rows
    const int32_t* row_offsets;  // first row and number of rows of each expert in the layout, instead of tile_row and
    const int32_t* row_counts;   // tile_rows: rows up to a multiple of 64 are computed; null: not known
    int32_t* status;
    int64_t out_rows;
    int64_t layout_rows;
    int32_t n_cols, k_blocks, w_ntiles;
    int32_t tile_rows_most;      // rows of a per tile: a multiple of 32, at most 256; 256 where any tile_* is given
    int32_t a_tiles;             // scale tiles per quad of a
    int32_t w_tiles, w_tiles_expert;  // scale tiles per quad of w, and of one expert
    int32_t w_blocks;            // blocks of 128 along the weights' output dimension
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
template <bool TURNED>
__device__ __forceinline__ uint32_t f8_instr_desc(int n, uint32_t scale_byte) {
    return (scale_byte << 4) | ((TURNED ? 1u : 0u) << 15) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(256 >> 4) << 24) |
           (scale_byte << 29);
}
// 32 tensor-memory lanes x 32 columns in the fragments of 8 x 8 matrices: v[16 h + 4 i ..] = (lane 16 h + l/4: columns
// 8 i + 2 (l%4) and the next; lane 16 h + l/4 + 8: the same), l = lane of the warp.
__device__ __forceinline__ void tc_load_32x32_fragments(uint32_t taddr, float* v) {
    uint32_t u[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n\t"
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
          "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
          "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr), "r"(taddr + (16u << 16))
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(u[i]);
}
// Four matrices of 8 x 8 values of 16 bits, turned: thread l holds of matrix m (word m) row l / 4, columns 2 (l % 4) and the
// next; lane 8 m + c gives the address of the 16 bytes that column c becomes.
__device__ __forceinline__ void st_matrix_turned(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared::cta.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tc_store_4(uint32_t taddr, uint4 v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(taddr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}

struct F8PairTile {
    int32_t expert;
    int32_t w0;      // first weight row = output column of the pair
    int32_t a_row;   // first row of a
    int32_t n;       // rows of a in the MMAs: a multiple of 32
    int32_t rows;    // output rows of this half of the tile (128 rows of a)
    int64_t out_row; // and the first of them
};

__device__ __forceinline__ void f8_rows(const GemmFp8Params& p, int32_t expert, int32_t a_row, int half, int64_t& out_row, int32_t& rows) {
    const int mt = a_row / 128 + half;  // used where tiles start at multiples of 256
    out_row = p.tile_row != nullptr ? __ldg(p.tile_row + mt) : a_row + 128LL * half;
    const int64_t most = min(128, p.tile_rows_most - 128 * half);
    int64_t left = p.tile_rows != nullptr ? __ldg(p.tile_rows + mt) : p.out_rows - out_row;
    if (p.row_counts != nullptr && expert >= 0)
        left = min(left, __ldg(p.row_offsets + expert) + (static_cast<int64_t>(__ldg(p.row_counts + expert)) + 63) / 64 * 64 - out_row);
    rows = static_cast<int32_t>(left < 0 || most < 0 ? 0 : (left > most ? most : left));
}

// false: nothing to do for this tile
__device__ __forceinline__ bool f8_decode(const GemmFp8Params& p, int tile, int a_ntiles, int half, F8PairTile& t) {
    const int per_super = F8_SUPER * p.w_ntiles;
    const int super = tile / per_super;
    const int first = super * F8_SUPER;
    const int span = min(F8_SUPER, a_ntiles - first);
    const int r = tile - super * per_super;
    const int wt = r / span;
    t.w0 = wt * 256;
    t.a_row = (first + (r - wt * span)) * p.tile_rows_most;
    t.expert = p.tile_expert != nullptr ? __ldg(p.tile_expert + t.a_row / 128) : 0;
    if (t.expert == -1) return false;
    int64_t other_row;
    int32_t other;
    f8_rows(p, t.expert, t.a_row, half, t.out_row, t.rows);
    f8_rows(p, t.expert, t.a_row, half ^ 1, other_row, other);
    const int32_t lower = half == 0 ? t.rows : other, upper = half == 0 ? other : t.rows;
    t.n = ((upper > 0 ? 128 + upper : lower) + 31) / 32 * 32;
    return t.n > 0;
}

// TURNED: out = a . w (w [E, reduction, n_cols]) instead of a . w^T
template <bool TURNED>
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
    const uint32_t tmem_base = tmem_slot;
    volatile int* abort_ptr = &abort_flag;

    const int64_t rows_used = p.rows_used != nullptr ? min(p.layout_rows, static_cast<int64_t>(__ldg(p.rows_used))) : p.layout_rows;
    const int a_ntiles = static_cast<int>((rows_used + p.tile_rows_most - 1) / p.tile_rows_most);
    const int total_tiles = a_ntiles * p.w_ntiles;
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
                if (!f8_decode(p, tile, a_ntiles, 0, t) || t.expert < 0) continue;
                const int w_row = (TURNED ? 0 : t.expert * p.n_cols) + t.w0 + static_cast<int>(rank) * 128;
                const int a_row = t.a_row + static_cast<int>(rank) * (t.n / 2);
                const int box = t.n > 128 ? 3 : (t.n > 64 ? 2 : (t.n > 32 ? 1 : 0));  // the smallest that holds n / 2 rows
                const uint32_t kb_bytes = F8_W_BYTES + (16 << box) * BK8;
                for (int kb = 0; kb < p.k_blocks; kb += F8_STAGE_KB) {
                    if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    const int n_kb = min(F8_STAGE_KB, p.k_blocks - kb);
                    const uint32_t leader_bar = map_to_rank(smem_u32(&full_bar[stage]), 0);
                    const uint32_t sa = ring + stage * F8_STAGE_BYTES;
                    const uint32_t sb = sa + F8_STAGE_KB * F8_W_BYTES;
                    if (leader) mbar_arrive_expect_tx(smem_u32(&full_bar[stage]), 2 * n_kb * kb_bytes);
                    for (int j = 0; j < n_kb; ++j) {
                        if (TURNED)
                            tma_load_3d_pair(sa + j * F8_W_BYTES, &p.map_w, leader_bar, w_row, (kb + j) * BK8, t.expert);
                        else
                            tma_load_2d_pair(sa + j * F8_W_BYTES, &p.map_w, leader_bar, (kb + j) * BK8, w_row);
                        tma_load_2d_pair(sb + j * F8_X_BYTES, &p.map_a[box], leader_bar, (kb + j) * BK8, a_row);
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
                if (!f8_decode(p, tile, a_ntiles, 0, t) || t.expert < 0) continue;
                // the epilogues have read the columns that this accumulator shares with the previous one
                if (n_done > 0 && !mbar_wait_warp(smem_u32(&acc_empty_bar), (n_done - 1) & 1u, abort_ptr, p.status)) break;
                tc_fence_after();
                const uint32_t acc = tmem_base + (n_done & 1u) * F8_ACC1_COL;
                for (int kb = 0; kb < p.k_blocks; kb += F8_STAGE_KB) {
                    if ((kb & 3) == 0 && !mbar_wait_warp(smem_u32(&scale_full_bar[sbuf]), sphase, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    if (!mbar_wait_warp(smem_u32(&full_bar[stage]), phase, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t scales = tmem_base + F8_SCALE_COL + sbuf * F8_SCALE_COLS;
                    const uint32_t sa = ring + stage * F8_STAGE_BYTES;
                    const uint64_t w_desc = make_smem_desc<TURNED>(sa);
                    const uint64_t a_desc = make_smem_desc<false>(sa + F8_STAGE_KB * F8_W_BYTES);
#pragma unroll
                    for (int j = 0; j < F8_STAGE_KB; ++j) {
                        if (kb + j >= p.k_blocks) continue;
                        const uint32_t idesc = f8_instr_desc<TURNED>(t.n, (kb + j) & 3);
#pragma unroll
                        for (int ks = 0; ks < BK8 / UMMA_K8; ++ks)
                            tc_mma_f8_pair(acc, w_desc + (j * F8_W_BYTES + ks * (TURNED ? UMMA_K8 * 128 : UMMA_K8)) / 16,
                                           a_desc + (j * F8_X_BYTES + ks * UMMA_K8) / 16, idesc, scales, scales + 4,
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
        const int half = (warp - 2) >> 2;        // rows 0-127 or 128-255 of the tile
        uint32_t n_chunks = 0;
        const bool f16 = p.f16 != 0;
        uint16_t* const out = static_cast<uint16_t*>(p.out);
        uint32_t n_done = 0;
        for (int tile = pair_id; tile < total_tiles; tile += n_pairs) {
            F8PairTile t;
            if (!f8_decode(p, tile, a_ntiles, half, t)) continue;
            const uint32_t acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + (n_done & 1u) * F8_ACC1_COL;
            // the 32 columns of the overlap come first: the last ones of accumulator 0, the first ones of 1
            const bool backwards = half == 1 && (n_done & 1u) == 0;
            if (t.expert >= 0) {
                if (!mbar_wait_warp(smem_u32(&acc_full_bar[n_done & 1u]), (n_done >> 1) & 1u, abort_ptr, p.status)) break;
                tc_fence_after();
            }
            const int col = t.w0 + static_cast<int>(rank) * 128 + quad * 32 + (lane & 3) * 8;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                const int r0 = (backwards ? 3 - i : i) * 32;  // rows r0 .. r0 + 31 of this half
                float v[32];                                  // 16 weight rows x 32 rows of a, and the next 16
                if (t.expert >= 0) {
                    if (half * 128 + r0 < t.n) tc_load_32x32_fragments(acc + half * 128 + r0, v);
                    if (i == 0) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_rank(smem_u32(&acc_empty_bar), 0));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0.f;
                }
                if (r0 >= t.rows) continue;
                // turned on the way into the patch: 32 rows of a x 64 bytes, read four lanes to a row of a
                const uint32_t patch = patches + (2 * (warp - 2) + (n_chunks++ & 1u)) * F8_PATCH_BYTES;
                if (lane == 0) bulk_wait_read_but_one();  // what left from this patch has been read
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int q = 0; q < 4; q += 2) {
                        // matrices: weight rows 16 h + 0-7 and 8-15, for rows of a 8 q .. 8 q + 7 and the next eight
                        const float* m = v + 16 * h + 4 * q;
                        const uint4 w = pack8(m, f16);
                        const int row = 8 * q + ((lane >> 4) << 3) + (lane & 7), piece = 2 * h + ((lane >> 3) & 1);
                        st_matrix_turned(patch + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4), w.x, w.y, w.z, w.w);
                    }
                }
                if (r0 + 32 <= t.rows) {
                    fence_smem_to_async();
                    __syncwarp();
                    const int first = t.w0 + static_cast<int>(rank) * 128 + quad * 32;
                    if (lane == 0) {
                        if (first < p.n_cols) tma_store_3d(&p.map_out, patch, first, static_cast<int>(t.out_row) + r0, 0);
                        bulk_commit();
                    }
                } else {  // a box would reach into the next expert's rows
                    __syncwarp();
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        const int row = it * 8 + (lane >> 2);
                        const uint4 w = ld_shared_16(patch + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4));
                        if (r0 + row < t.rows && col < p.n_cols) st_global_16(out + (t.out_row + r0 + row) * p.n_cols + col, w);
                    }
                    if (lane == 0) bulk_commit();  // an empty group, so that groups count the patches
                }
            }
            if (t.expert >= 0) ++n_done;
        }
        if (lane == 0) bulk_wait_all();
    } else {
        // ------------------------------ scales (both CTAs) ------------------------------
        // All four warps bring the same words, each into its 32 lanes: word j of lane l is row j * 32 + l.  The 128 weight
        // rows of a CTA are one block and share one word.
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
            if (!f8_decode(p, tile, a_ntiles, 0, t) || t.expert < 0) continue;
            const int block = t.w0 / FP8_BLOCK + static_cast<int>(rank);
            const int piece = t.a_row / 32;  // in 32 rows: a scale tile holds four
            for (int kb = 0; kb < p.k_blocks; kb += 4) {
                const int q = kb >> 2;
                const uint32_t one = 0x01010101u * FP8_SCALE_ONE;
                uint32_t ww = one, wa[8];
                if (TURNED) {
                    // one byte of each of the four words, which lie in four scale tiles
                    const int rb = kb + (lane & 3);
                    uint32_t byte = FP8_SCALE_ONE;
                    if (rb < p.k_blocks && block < p.w_blocks)
                        byte = __ldg(p.w_scales + (static_cast<int64_t>(block >> 2) * p.w_tiles + t.expert * p.w_tiles_expert + rb) * FP8_TILE_BYTES +
                                     (block & 3));
                    ww = byte << (8 * (lane & 3));
                    ww |= __shfl_xor_sync(0xffffffffu, ww, 1);
                    ww |= __shfl_xor_sync(0xffffffffu, ww, 2);
                } else if (block < p.w_blocks)
                    ww = __ldg(reinterpret_cast<const uint32_t*>(
                        p.w_scales + (static_cast<int64_t>(q) * p.w_tiles + t.expert * p.w_tiles_expert + block) * FP8_TILE_BYTES));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    wa[j] = one;
                    if (j * 32 < t.n && (piece + j) / 4 < p.a_tiles)
                        wa[j] = __ldg(reinterpret_cast<const uint32_t*>(
                            p.a_scales + (static_cast<int64_t>(q) * p.a_tiles + (piece + j) / 4) * FP8_TILE_BYTES + lane * 16 + ((piece + j) & 3) * 4));
                }
                if (ends[buf] > 0) {
                    const uint32_t last = ends[buf] - 1;
                    if (!mbar_wait_warp(smem_u32(&empty_bar[last % F8_STAGES]), (last / F8_STAGES) & 1u, abort_ptr, p.status)) {
                        alive = false;
                        break;
                    }
                }
                n_stages += min(kStagesPerGroup, (p.k_blocks - kb + F8_STAGE_KB - 1) / F8_STAGE_KB);
                ends[buf] = n_stages;
                tc_fence_after();
                __syncwarp();
                const uint32_t at = tmem_base + lanes + F8_SCALE_COL + buf * F8_SCALE_COLS;
                tc_store_4(at, make_uint4(ww, ww, ww, ww));
                tc_store_4(at + 4, make_uint4(wa[0], wa[1], wa[2], wa[3]));
                tc_store_4(at + 8, make_uint4(wa[4], wa[5], wa[6], wa[7]));
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
// Rows of a per tile.  High tiles read the weights least often; but the launch takes as long as its fullest pair of SMs,
// so where the number of rows is known (no experts) the height that makes waves * (height + 128) smallest is taken: a
// tile costs its rows, and its loads of the weights as much as 128 rows more.  Measured, 4096 x 4096 weights: 256 rows 15.7 us,
// with 256 rows per tile 17.3; 2048 rows 29.2, with 192 per tile 37; 4096 rows 53.6, with 192 / 128 per tile 61 / 77 (a rule that
// took the weights for 24 rows chose 128); 1536 x 2048 weights: 384 rows 10.5, with 256 per tile 11.7.  It misses little: of 104
// cases (8 shapes, 64 to 8192 rows) one by more than 5 %, 3000 rows of 8192 x 8192, 167 against 151 with 256 per tile.
static int rows_per_tile(int64_t rows, int N) {
    const int64_t pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1, w = (N + 255) / 256;
    const int64_t fewest = (rows + F8_TILE_ROWS - 1) / F8_TILE_ROWS;
    int best = 0;
    int64_t best_cost = 0;
    for (int64_t n = fewest; n <= rows / 64 + 1; ++n) {
        const int64_t height = ((rows + n - 1) / n + 31) / 32 * 32;  // paired MMAs take whole 32 columns
        const int64_t tiles = (rows + height - 1) / height;
        const int64_t cost = (w * tiles + pairs - 1) / pairs * (height + 128);
        if (best == 0 || cost < best_cost) {
            best = static_cast<int>(height);
            best_cost = cost;
        }
        if (w * n > 16 * pairs) break;  // many waves: the highest tile
    }
    return best;
}

// Whether tiles of 128 weight rows and up to 128 rows of x, spread over clusters along k, are the faster way: with few
// rows, where the pair tiles leave at least half of the pairs without work, and up to 128 rows of a matrix, or per expert, if
// there is much to share along k.  Measured from captured graphs, quantising x included, this way / pair tiles, us: 4096 x 4096 (16
// pair tiles) with 17 / 64 / 128 rows 10.8 / 12.5 / 15.0 against 17.2 to 17.8, 4096 x 14336 18.5 / 21.0 / 25.7 against 39.4 to 40.3,
// 8192 x 4096 (32) 24 / 96 rows 14.0 / 17.0 against 17.9 / 18.5; but 2048 x 768 48 / 64 rows 8.8 / 9.5 against 9.3 / 9.0, and
// 14336 x 4096 (56) 24 / 64 / 128 rows 19.5 / 21.0 / 24.7 against 19.4 / 19.7 / 20.7.  Two experts of 4096 x 4096 (32) with 48 / 96
// rows each 22.0 / 25.5 against 22.4 / 24.6, of 4096 x 14336 with 64 rows 48.8 against 58.4, of 1024 x 14336 33 against 53, four of
// 1024 x 4096 with 96 rows 21.3 against 23.7; but eight of 14336 x 4096 101 against 97, 128 of 1536 x 2048 91 to 106 against 90 to 97.
static bool some_rows_suit(int64_t layout_rows, int64_t out_rows, int32_t E, int32_t N, int32_t K, bool experts, bool tile_rows) {
    if (!fp8_some_rows_fits(K) || E * ((N + 255LL) / 256) * 2 > sm_count() / 2) return false;
    if (!experts) return layout_rows <= 48 || (layout_rows <= 128 && K >= 1536);
    return tile_rows && out_rows <= (K >= 2LL * N ? 128LL : 48LL) * E;  // without tile_rows the rows of a layout are not known here
}

template <bool TURNED>
static int launch_fp8(GemmFp8Params& p, cudaStream_t s) {
    static bool configured[64] = {false};  // per device: the attribute applies to the current device only
    const int dev = current_device_slot();
    FMAB_REQUIRE(dev >= 0, FMA_B200_ERR_LAUNCH, "no current CUDA device with an ordinal below 64");
    if (!configured[dev]) {
        FMAB_CUDA(cudaFuncSetAttribute(gemm_fp8_kernel<TURNED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F8_SMEM));
        configured[dev] = true;
    }
    const int64_t total = (p.layout_rows + p.tile_rows_most - 1) / p.tile_rows_most * p.w_ntiles;
    FMAB_REQUIRE(total < (1LL << 31), FMA_B200_ERR_BAD_ARG, "too many tiles");
    const int64_t max_pairs = sm_count() >= 2 ? sm_count() / 2 : 1;
    const int pairs = static_cast<int>(total < max_pairs ? total : max_pairs);
    return launch_kernel("8-bit grouped GEMM", gemm_fp8_kernel<TURNED>, dim3(2 * pairs), F8_THREADS, F8_SMEM, 0, s, p);
}

template <bool TURNED>
static int fp8_product(const void* a, const void* a_scales, int64_t layout_rows, const void* w, const void* w_scales, int32_t E, int32_t N,
                       int32_t K, void* out, int32_t dtype, int64_t out_rows, const int32_t* tile_expert, const int32_t* tile_row,
                       const int32_t* tile_rows, const int32_t* rows_used, const int32_t* row_offsets, const int32_t* row_counts,
                       cudaStream_t s) {
    FMAB_REQUIRE(dtype == FMA_B200_BF16 || dtype == FMA_B200_F16, FMA_B200_ERR_UNSUPPORTED,
                 "dtype %d: the 8-bit product returns bfloat16 or half", dtype);
    FMAB_REQUIRE(layout_rows >= 0 && layout_rows < (1LL << 31) - 256 && out_rows >= 0, FMA_B200_ERR_BAD_ARG,
                 "layout_rows=%lld, out_rows=%lld", (long long)layout_rows, (long long)out_rows);
    FMAB_REQUIRE(E >= 1 && E <= 1024, FMA_B200_ERR_BAD_ARG, "E=%d not in [1,1024]", E);
    FMAB_REQUIRE(N >= 8 && K >= 8 && N % 8 == 0 && K % 8 == 0 && N < (1 << 30) && K < (1 << 30), FMA_B200_ERR_BAD_ARG,
                 "N=%d and K=%d must be positive multiples of 8", N, K);
    FMAB_REQUIRE(static_cast<int64_t>(E) * (TURNED ? K : N) < (1LL << 31) - 1024, FMA_B200_ERR_BAD_ARG, "E*%s overflows", TURNED ? "K" : "N");
    FMAB_REQUIRE(E == 1 || tile_expert != nullptr, FMA_B200_ERR_BAD_ARG, "several experts need tile_expert");
    FMAB_REQUIRE((row_offsets == nullptr) == (row_counts == nullptr) && !(row_counts && (tile_row || tile_rows || !tile_expert)),
                 FMA_B200_ERR_BAD_ARG, "row_offsets and row_counts come together, beside tile_expert, without tile_row and tile_rows");
    if (layout_rows == 0 || out_rows == 0) return FMA_B200_OK;
    FMAB_REQUIRE(a && a_scales && w && w_scales && out, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(a) && aligned16(a_scales) && aligned16(w) && aligned16(w_scales) && aligned16(out),
                 FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    if (!TURNED && some_rows_suit(layout_rows, out_rows, E, N, K, tile_expert != nullptr, tile_rows != nullptr))
        return fp8_some_rows(a, a_scales, layout_rows, w, w_scales, E, N, K, out, dtype, out_rows, tile_expert, tile_row, tile_rows,
                             rows_used, tile_expert != nullptr ? (E < out_rows ? E : out_rows) : 1, s);
    GemmFp8Params p;
    memset(&p, 0, sizeof(p));
    p.status = device_status_ptr();
    FMAB_REQUIRE(p.status != nullptr, FMA_B200_ERR_LAUNCH, "no device status word");
    p.out = out;
    p.tile_expert = tile_expert;
    p.tile_row = tile_row;
    p.tile_rows = tile_rows;
    p.rows_used = rows_used;
    p.row_offsets = row_offsets;
    p.row_counts = row_counts;
    p.out_rows = out_rows;
    p.layout_rows = layout_rows;
    p.n_cols = N;
    p.k_blocks = (K + BK8 - 1) / BK8;
    p.tile_rows_most = tile_expert || tile_row || tile_rows ? F8_TILE_ROWS : rows_per_tile(layout_rows, N);
    p.w_ntiles = (N + 255) / 256;
    p.a_scales = static_cast<const uint8_t*>(a_scales);
    p.w_scales = static_cast<const uint8_t*>(w_scales);
    p.a_tiles = static_cast<int32_t>(fp8_row_tiles(layout_rows));
    p.w_blocks = (N + FP8_BLOCK - 1) / FP8_BLOCK;
    p.w_tiles_expert = static_cast<int32_t>(fp8_row_tiles(TURNED ? K : N));
    p.w_tiles = E * p.w_tiles_expert;
    p.f16 = dtype == FMA_B200_F16 ? 1 : 0;
    for (int b = 0; b < F8_BOXES; ++b)
        if (int rc = encode_bytes(&p.map_a[b], a, K, layout_rows, fp8_pitch(K), 16 << b)) return rc;
    if (TURNED) {
        if (int rc = encode_bytes_3d(&p.map_w, w, N, K, E, fp8_pitch(N), 128)) return rc;
    } else {
        if (int rc = encode_bytes(&p.map_w, w, K, static_cast<uint64_t>(E) * N, fp8_pitch(K), 128)) return rc;
    }
    if (int rc = encode_3d(&p.map_out, out, N, out_rows, 1, N, static_cast<uint64_t>(out_rows) * N, 32, 32, p.f16 != 0)) return rc;
    return launch_fp8<TURNED>(p, s);
}

}  // namespace fmab

extern "C" {

int fma_b200_fp8_gemm(const void* a, const void* a_scales, int64_t layout_rows, const void* w, const void* w_scales,
                      int32_t E, int32_t N, int32_t K, void* out, int32_t dtype, int64_t out_rows,
                      const int32_t* tile_expert, const int32_t* tile_row, const int32_t* tile_rows,
                      const int32_t* rows_used, const int32_t* row_offsets, const int32_t* row_counts, void* stream) {
    return fmab::fp8_product<false>(a, a_scales, layout_rows, w, w_scales, E, N, K, out, dtype, out_rows, tile_expert, tile_row, tile_rows,
                                    rows_used, row_offsets, row_counts, static_cast<cudaStream_t>(stream));
}

int fma_b200_fp8_gemm_dgrad(const void* dy, const void* dy_scales, int64_t layout_rows, const void* w, const void* w_scales,
                            int32_t E, int32_t N, int32_t K, void* dx, int32_t dtype, int64_t out_rows,
                            const int32_t* tile_expert, const int32_t* tile_row, const int32_t* tile_rows,
                            const int32_t* rows_used, const int32_t* row_offsets, const int32_t* row_counts, void* stream) {
    return fmab::fp8_product<true>(dy, dy_scales, layout_rows, w, w_scales, E, K, N, dx, dtype, out_rows, tile_expert, tile_row, tile_rows,
                                   rows_used, row_offsets, row_counts, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
