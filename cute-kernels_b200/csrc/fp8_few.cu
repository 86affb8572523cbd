// The 8-bit product for a few rows (serving single tokens): out[r, :] = x[r, :] . w[e(r)]^T in ONE launch, the rows of x
// quantised on the way in.  The weights are read once, N * K bytes, and that is what bounds it; up to 16 rows ride along.
//
// The weights are the 128-row operand of tcgen05.mma and the tokens its 16 columns, so a tile is 128 weight rows and
// TMA streams it without any thread touching it.  A cluster of up to eight CTAs shares a tile, each with its part of the
// reduction (whole groups of 512 columns): 4096 weight rows are only 32 tiles, and every SM has to load for the memory
// to run at its rate.  The parts are added through distributed shared memory in the order of the ranks.
// (With mma.sync and weights from global memory into registers one row of 14336 x 4096 took 17 to 23 us, this way 14 from a
// captured graph, 16.5 call by call: the 8-bit mma.sync costs several times the instructions of the loads.)
#include "fp8.cuh"
#include "gemm_pair.cuh"

namespace fmab {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewRows = 16;                          // rows of x per pass over the weights
constexpr int kFewStages = 4;                         // k-blocks of 128 x 128 bytes in flight
constexpr int kFewStageBytes = 128 * FP8_BLOCK;
constexpr int kFewXBytes = kFewRows * FP8_BLOCK;      // rows of x per k-block
constexpr int kFewScaleCol = 16;                      // tensor memory: accumulator 0-15, then 8 columns per quad
constexpr int kFewScaleCols = 8;                      // (weights 4, rows of x 1)

struct FewRows {
    CUtensorMap map_w;
    const void* x;
    const uint8_t* w_scales;
    void* out;
    const void* counts;  // rows per expert; null: one expert
    int32_t* status;
    int64_t x_pitch;
    int32_t index_bytes, E, rows, N, K, k_blocks, quads, tiles, b_tiles, split, quads_most;
    uint32_t tmem_cols;
};

__device__ __forceinline__ void tc_mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_commit_elected(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 ld_shared_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

// Expert, first row and number of rows of a chunk of at most 16 rows; experts in order, then the rows of no expert
// (expert -2).  false: there are fewer chunks.  Counts that overshoot are cut off at p.rows.  Every warp for itself.
__device__ __forceinline__ bool few_locate(const FewRows& p, int chunk, int& expert, int& row0, int& rows) {
    const int lane = threadIdx.x & 31;
    int done_rows = 0, done_chunks = 0;
    if (p.counts == nullptr) {
        expert = 0;
        row0 = chunk * kFewRows;
        rows = min(kFewRows, p.rows - row0);
        return rows > 0;
    }
    for (int e0 = 0; e0 < p.E; e0 += 32) {
        int end = e0 + lane < p.E ? fp8_count(p.counts, p.index_bytes, e0 + lane, p.rows) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {  // running sum, cut off at p.rows
            const int v = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = min(end + v, p.rows);
        }
        end = min(done_rows + end, p.rows);
        int begin = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) begin = done_rows;
        const int mine = (end - begin + kFewRows - 1) / kFewRows;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const int first = done_chunks + upto - mine;  // this expert's first chunk
        const uint32_t hit = __ballot_sync(0xffffffffu, chunk >= first && chunk < first + mine);
        if (hit != 0) {
            const int src = __ffs(hit) - 1;
            expert = e0 + src;
            row0 = __shfl_sync(0xffffffffu, begin + (chunk - first) * kFewRows, src);
            rows = min(kFewRows, __shfl_sync(0xffffffffu, end, src) - row0);
            return true;
        }
        done_rows = __shfl_sync(0xffffffffu, end, 31);
        done_chunks += __shfl_sync(0xffffffffu, upto, 31);
    }
    expert = -2;
    row0 = done_rows + (chunk - done_chunks) * kFewRows;
    rows = min(kFewRows, p.rows - row0);
    return rows > 0;
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads, 3) few_rows_kernel(const __grid_constant__ FewRows p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kFewStages], empty_bar[kFewStages], scale_bar, acc_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int item = blockIdx.x / p.split;
    const int chunk = item / p.tiles, n0 = (item - chunk * p.tiles) * 128;
    int expert, row0, rows;
    if (!few_locate(p, chunk, expert, row0, rows)) return;  // the whole cluster
    T* const out = static_cast<T*>(p.out) + static_cast<int64_t>(row0) * p.N + n0;
    if (expert < 0) {
        if (rank == 0)
            for (int i = tid; i < rows * 128; i += kFewThreads)
                if (n0 + (i & 127) < p.N) out[static_cast<int64_t>(i >> 7) * p.N + (i & 127)] = float_to_elem<T>(0.f);
        return;
    }
    const int q0 = p.quads * rank / p.split, q1 = p.quads * (rank + 1) / p.split;  // this CTA's groups of 512 columns
    const int k0 = 4 * q0, n_kb = min(4 * q1, p.k_blocks) - k0;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t xs = ring + kFewStages * kFewStageBytes;
    uint8_t* const base = smem_raw + (ring - smem_u32(smem_raw));
    uint8_t* const x8 = base + kFewStages * kFewStageBytes;
    uint32_t* const sx = reinterpret_cast<uint32_t*>(x8 + 4 * p.quads_most * kFewXBytes);  // [quad][16]
    volatile int* abort_ptr = &abort_flag;

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < kFewStages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        mbar_init(smem_u32(&scale_bar), 4);
        mbar_init(smem_u32(&acc_bar), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        for (int kb = 0; kb < min(kFewStages, n_kb); ++kb) {  // the weights start to flow before anything else is done
            mbar_arrive_expect_tx(smem_u32(&full_bar[kb]), kFewStageBytes);
            tma_load_2d(ring + kb * kFewStageBytes, &p.map_w, smem_u32(&full_bar[kb]), (k0 + kb) * FP8_BLOCK, expert * p.N + n0);
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // the rows of x in 8 bits, in the 128-byte swizzle of an MMA operand
    {
        constexpr int AHEAD = 4;  // rows whose loads are in flight together
        const int n = rows * (q1 - q0), s = lane & 7, g = lane >> 3;
        for (int i0 = warp; i0 < n; i0 += kFewWarps * AHEAD) {
            uint4 raw[AHEAD][2];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = i0 + u * kFewWarps, q = i / rows, r = i - q * rows;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int c = (k0 + 4 * q + g) * FP8_BLOCK + LaneBlock<T>::column(s, j);
                    raw[u][j] = i < n && c < p.K ? ld_global_16(static_cast<const T*>(p.x) + (row0 + r) * p.x_pitch + c) : make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = i0 + u * kFewWarps, q = i / rows, r = i - q * rows, kb = 4 * q + g;
                if (i >= n) break;
                uint32_t w[4];
                const uint32_t word = scale_word_of(quantize_lane_raw<T>(raw[u], w));
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int c = LaneBlock<T>::column(s, j);
                    *reinterpret_cast<uint2*>(x8 + kb * kFewXBytes + r * FP8_BLOCK + (((c >> 4) ^ (r & 7)) << 4) + (c & 15)) =
                        make_uint2(w[2 * j], w[2 * j + 1]);
                }
                if (lane == 0) sx[q * kFewRows + r] = word;
            }
        }
    }
    fence_smem_to_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            for (int kb = kFewStages; kb < n_kb; ++kb) {
                const int s = kb % kFewStages;
                if (!mbar_wait(smem_u32(&empty_bar[s]), (kb / kFewStages - 1) & 1u, abort_ptr, p.status)) break;
                mbar_arrive_expect_tx(smem_u32(&full_bar[s]), kFewStageBytes);
                tma_load_2d(ring + s * kFewStageBytes, &p.map_w, smem_u32(&full_bar[s]), (k0 + kb) * FP8_BLOCK, expert * p.N + n0);
            }
        }
    } else if (warp == 1) {
        bool alive = mbar_wait_warp(smem_u32(&scale_bar), 0, abort_ptr, p.status);
        for (int kb = 0; kb < n_kb && alive; ++kb) {
            const int s = kb % kFewStages;
            alive = mbar_wait_warp(smem_u32(&full_bar[s]), (kb / kFewStages) & 1u, abort_ptr, p.status);
            if (!alive) break;
            tc_fence_after();
            const uint32_t byte = kb & 3, scales = tmem + kFewScaleCol + (kb >> 2) * kFewScaleCols;
            const uint32_t idesc = (byte << 4) | (static_cast<uint32_t>(kFewRows >> 3) << 17) | (1u << 23) | (8u << 24) | (byte << 29);
            const uint64_t a = make_smem_desc<false>(ring + s * kFewStageBytes);
            const uint64_t b = make_smem_desc<false>(xs + kb * kFewXBytes);
#pragma unroll
            for (int ks = 0; ks < FP8_BLOCK / 32; ++ks)
                tc_mma_f8(tmem, a + ks * 2, b + ks * 2, idesc, scales, scales + 4, (kb | ks) != 0);
            tc_commit_elected(smem_u32(&empty_bar[s]));
        }
        if (alive) tc_commit_elected(smem_u32(&acc_bar));
    }
    float* const part = reinterpret_cast<float*>(base);  // [16 rows of x][128 weight rows], over the drained ring
    if (warp >= 4) {
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        for (int q = 0; q < q1 - q0; ++q) {
            const uint32_t ww = __ldg(reinterpret_cast<const uint32_t*>(
                p.w_scales + (static_cast<int64_t>(q0 + q) * p.b_tiles + static_cast<int64_t>(expert) * p.tiles + n0 / 128) * FP8_TILE_BYTES));
            const uint32_t wx = sx[q * kFewRows + (lane & 15)];
            const uint32_t at = tmem + lanes + kFewScaleCol + q * kFewScaleCols;
            asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(ww) : "memory");
            asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(at + 4), "r"(wx) : "memory");
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&scale_bar));
        if (mbar_wait_warp(smem_u32(&acc_bar), 0, abort_ptr, p.status)) {
            tc_fence_after();
            uint32_t v[16];
            asm volatile(
                "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                  "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                : "r"(tmem + lanes)
                : "memory");
            tc_load_wait();
            const int n = (warp & 3) * 32 + lane;
            if (p.split == 1) {
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
                    if (r < rows && n0 + n < p.N) out[static_cast<int64_t>(r) * p.N + n] = float_to_elem<T>(__uint_as_float(v[r]));
            } else {
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
                    if (r < rows) part[r * 128 + n] = __uint_as_float(v[r]);
            }
        }
    }
    __syncwarp();
    if (abort_flag && tid == 0) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land
    }
    __syncwarp();
    if (p.split > 1) {
        cluster_sync_all();  // every part is in its CTA's shared memory
        const int width = 128 / p.split;  // this CTA adds and writes its share of the weight rows
        for (int i = tid; i < rows * width; i += kFewThreads) {
            const int r = i / width, n = rank * width + i % width;
            float v[8], sum = 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = c < p.split ? ld_shared_cluster_f32(map_to_rank(ring + (r * 128 + n) * 4, c)) : 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) sum += v[c];
            if (n0 + n < p.N) out[static_cast<int64_t>(r) * p.N + n] = float_to_elem<T>(sum);
        }
        tc_fence_before();
        cluster_sync_all();  // nobody leaves while its part is being read
    } else {
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
}

// ---- tiles of up to 128 rows, quantised before ------------------------------------------------------------
// The same shape of product for tens of rows, where the pair tiles of gemm_fp8.cu are too few for the GPU (its rule has
// the figures): 128 weight rows against a 128-row tile of x, of which the 16, 32, 64 or 128 rows that cover its rows are the
// columns of the MMA and are streamed beside the weights.  A cluster shares each tile along the reduction, which is what
// pair tiles cannot do.  Weights are still what moves.  Quantising on the way in would be repeated by every tile of
// weights (1 us per row of 4096 columns, measured), so it is a launch of its own here.
constexpr int kSomeThreads = 192;
constexpr int kSomeStagesMost = 5;
constexpr int kSomeBoxes = 4;  // loads of 16, 32, 64, 128 rows of x
constexpr int kSomeQuadsFit = 16;  // scales of 512-column groups beside a 128-column accumulator in 256 columns

struct SomeRows {
    CUtensorMap map_w;
    CUtensorMap map_x[kSomeBoxes];
    const uint8_t *w_scales, *x_scales;
    void* out;
    const int32_t *tile_expert, *tile_row, *tile_rows, *rows_used;  // as for the pair tiles
    int32_t* status;
    int64_t out_rows, layout_rows;
    int32_t N, k_blocks, quads, tiles, w_tiles, x_tiles, split, quads_most, stages, cols_most;
    uint32_t tmem_cols;
};

template <typename T>
__global__ void __launch_bounds__(kSomeThreads) some_rows_kernel(const __grid_constant__ SomeRows p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kSomeStagesMost], empty_bar[kSomeStagesMost], scale_bar, acc_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int item = blockIdx.x / p.split;
    const int x_tile = item / p.tiles, tile = item - x_tile * p.tiles, n0 = tile * 128;
    if (p.rows_used != nullptr && static_cast<int64_t>(x_tile) * 128 >= __ldg(p.rows_used)) return;  // the whole cluster
    const int expert = p.tile_expert != nullptr ? __ldg(p.tile_expert + x_tile) : 0;
    const int64_t out_row = p.tile_row != nullptr ? __ldg(p.tile_row + x_tile) : static_cast<int64_t>(x_tile) * 128;
    const int64_t left = p.tile_rows != nullptr ? __ldg(p.tile_rows + x_tile) : p.out_rows - out_row;
    const int rows = static_cast<int>(left > 128 ? 128 : left);
    if (expert == -1 || rows <= 0) return;
    T* const out = static_cast<T*>(p.out) + out_row * p.N + n0;
    if (expert < 0) {  // rows of no expert
        if (rank == 0)
            for (int i = tid; i < rows * 128; i += kSomeThreads)
                if (n0 + (i & 127) < p.N) out[static_cast<int64_t>(i >> 7) * p.N + (i & 127)] = float_to_elem<T>(0.f);
        return;
    }
    const int box = rows <= 16 ? 0 : (rows <= 32 ? 1 : (rows <= 64 ? 2 : 3)), cols = 16 << box;
    const int q0 = p.quads * rank / p.split, q1 = p.quads * (rank + 1) / p.split;  // this CTA's groups of 512 columns
    const int k0 = 4 * q0, n_kb = min(4 * q1, p.k_blocks) - k0;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t stage_bytes = kFewStageBytes + p.cols_most * FP8_BLOCK;
    uint8_t* const base = smem_raw + (ring - smem_u32(smem_raw));
    volatile int* abort_ptr = &abort_flag;

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        mbar_init(smem_u32(&scale_bar), 4);
        mbar_init(smem_u32(&acc_bar), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            for (int kb = 0; kb < n_kb; ++kb) {
                const int s = kb % p.stages;
                if (kb >= p.stages && !mbar_wait(smem_u32(&empty_bar[s]), (kb / p.stages - 1) & 1u, abort_ptr, p.status)) break;
                const uint32_t at = ring + s * stage_bytes, bar = smem_u32(&full_bar[s]);
                mbar_arrive_expect_tx(bar, kFewStageBytes + cols * FP8_BLOCK);
                tma_load_2d(at, &p.map_w, bar, (k0 + kb) * FP8_BLOCK, expert * p.N + n0);
                tma_load_2d(at + kFewStageBytes, &p.map_x[box], bar, (k0 + kb) * FP8_BLOCK, x_tile * 128);
            }
        }
    } else if (warp == 1) {
        bool alive = mbar_wait_warp(smem_u32(&scale_bar), 0, abort_ptr, p.status);
        for (int kb = 0; kb < n_kb && alive; ++kb) {
            const int s = kb % p.stages;
            alive = mbar_wait_warp(smem_u32(&full_bar[s]), (kb / p.stages) & 1u, abort_ptr, p.status);
            if (!alive) break;
            tc_fence_after();
            const uint32_t byte = kb & 3, scales = tmem + p.cols_most + (kb >> 2) * kFewScaleCols;
            const uint32_t idesc = (byte << 4) | (static_cast<uint32_t>(cols >> 3) << 17) | (1u << 23) | (8u << 24) | (byte << 29);
            const uint64_t a = make_smem_desc<false>(ring + s * stage_bytes);
            const uint64_t b = make_smem_desc<false>(ring + s * stage_bytes + kFewStageBytes);
#pragma unroll
            for (int ks = 0; ks < FP8_BLOCK / 32; ++ks)
                tc_mma_f8(tmem, a + ks * 2, b + ks * 2, idesc, scales, scales + 4, (kb | ks) != 0);
            tc_commit_elected(smem_u32(&empty_bar[s]));
        }
        if (alive) tc_commit_elected(smem_u32(&acc_bar));
    } else {
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        for (int q = 0; q < q1 - q0; ++q) {
            const uint32_t ww = __ldg(reinterpret_cast<const uint32_t*>(
                p.w_scales + (static_cast<int64_t>(q0 + q) * p.w_tiles + static_cast<int64_t>(expert) * p.tiles + tile) * FP8_TILE_BYTES));
            const uint4 wx = __ldg(reinterpret_cast<const uint4*>(p.x_scales + (static_cast<int64_t>(q0 + q) * p.x_tiles + x_tile) * FP8_TILE_BYTES) + lane);
            const uint32_t at = tmem + lanes + p.cols_most + q * kFewScaleCols;
            asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(ww) : "memory");
            asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};"
                         ::"r"(at + 4), "r"(wx.x), "r"(wx.y), "r"(wx.z), "r"(wx.w)
                         : "memory");
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&scale_bar));
        if (mbar_wait_warp(smem_u32(&acc_bar), 0, abort_ptr, p.status)) {
            tc_fence_after();
            float* const part = reinterpret_cast<float*>(base);  // [rows of x][128 weight rows], over the drained ring
            const int n = (warp & 3) * 32 + lane;
#pragma unroll 1
            for (int r0 = 0; r0 < rows; r0 += 16) {
                uint32_t v[16];
                asm volatile(
                    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                    : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                      "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                    : "r"(tmem + lanes + r0)
                    : "memory");
                tc_load_wait();
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (p.split > 1)
                        part[(r0 + r) * 128 + n] = __uint_as_float(v[r]);
                    else if (r0 + r < rows && n0 + n < p.N)
                        out[static_cast<int64_t>(r0 + r) * p.N + n] = float_to_elem<T>(__uint_as_float(v[r]));
                }
            }
        }
    }
    __syncwarp();
    if (abort_flag && tid == 0) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land
    }
    __syncwarp();
    if (p.split > 1) {
        cluster_sync_all();  // every part is in its CTA's shared memory
        const int r_begin = rows * rank / p.split, r_end = rows * (rank + 1) / p.split;  // this CTA adds and writes these
        for (int i = tid; i < (r_end - r_begin) * 32; i += kSomeThreads) {
            const int r = r_begin + (i >> 5), n = (i & 31) * 4;
            float4 v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c)
                v[c] = c < p.split ? ld_shared_cluster_f32x4(map_to_rank(ring + (r * 128 + n) * 4, c)) : make_float4(0.f, 0.f, 0.f, 0.f);
            float4 sum = v[0];
#pragma unroll
            for (int c = 1; c < 8; ++c) {
                sum.x += v[c].x;
                sum.y += v[c].y;
                sum.z += v[c].z;
                sum.w += v[c].w;
            }
            if (n0 + n < p.N) {  // N is a multiple of 8
                const T w[4] = {float_to_elem<T>(sum.x), float_to_elem<T>(sum.y), float_to_elem<T>(sum.z), float_to_elem<T>(sum.w)};
                *reinterpret_cast<uint2*>(out + static_cast<int64_t>(r) * p.N + n) = *reinterpret_cast<const uint2*>(w);
            }
        }
        tc_fence_before();
        cluster_sync_all();  // nobody leaves while its part is being read
    } else {
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
}

// CTAs per tile, in whole groups of 512 columns: until nearly every SM has one, on while a CTA would read four groups (256 KB)
// or more and there is room for all of them (three per SM), and on while its part is too long: longer than what fits into tensor
// memory, or in the product that quantises x itself than what leaves room for a second CTA on the SM.  Measured from captured
// graphs, weights not in L2: one row of 14336 x 4096 (112 tiles) 15.6 / 13.9 / 17.5 us with 1 / 2 / 4 CTAs per tile, 8192 x 4096 (64)
// 12.3 / 10.5 / 14.2 with 2 / 4 / 8, 4096 x 4096 (32) 10.2 / 8.8 / 8.2, 4096 x 14336 (32) 16.7 / 14.3 with 4 / 8; eight rows of eight
// experts, 5 of them hit, of 1536 x 2048 10.0 / 9.0 / 9.2 with 1 / 2 / 4, 4096 x 4096 27.7 / 23.8 / 25.8, 8192 x 8192 82.7 / 80.9 / 69.0;
// 64 rows, tiles of up to 128, quantising included, 8192 x 4096 17.6 / 15.6 / 22.9 with 2 / 4 / 8, 4096 x 4096 15.8 / 12.5 / 13.8.
constexpr int FEW_QUADS_MOST = 18;  // rows of x in 8 bits that fit into shared memory beside the ring
constexpr int FEW_QUADS_TWO = 5;    // and that leave room for a second CTA on the SM
static int few_split(int64_t items, int quads, int quads_fit) {
    const int64_t sms = sm_count();
    int split = 1;
    while (split < 8 && 2 * split <= quads &&
           (100 * items * split < 85 * sms || (quads >= 4 * split && 2 * items * split <= 3 * sms) || quads > quads_fit * split))
        split *= 2;
    return split;
}
static int64_t few_smem(int quads_most) {
    return kFewStages * static_cast<int64_t>(kFewStageBytes) + static_cast<int64_t>(quads_most) * (4 * kFewXBytes + kFewRows * 4) + 1024;
}
static int64_t few_chunks(int64_t rows, int32_t E, bool counts) {  // at most
    if (!counts) return (rows + kFewRows - 1) / kFewRows;
    const int64_t groups = E + 1 < rows ? E + 1 : rows, n = rows / kFewRows + groups;
    return n < rows ? n : rows;
}

static int64_t few_chunks_even(int64_t rows, int32_t E) {  // if the rows are spread evenly
    const int64_t n = (rows + kFewRows - 1) / kFewRows, hit = rows < E ? rows : E;
    return n > hit ? n : hit;
}

// Opts a kernel into large dynamic shared memory, once per kernel and device.
template <typename Kernel>
static int allow_smem(Kernel kernel) {
    static const void* done[64][4] = {};  // kernels of the same type: bfloat16 and half of one kernel
    const int dev = current_device_slot();
    FMAB_REQUIRE(dev >= 0, FMA_B200_ERR_LAUNCH, "no current CUDA device with an ordinal below 64");
    const void* const key = reinterpret_cast<const void*>(kernel);
    for (int i = 0; i < 4; ++i) {
        if (done[dev][i] == key) return FMA_B200_OK;
        if (done[dev][i] == nullptr) {
            FMAB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
            done[dev][i] = key;
            return FMA_B200_OK;
        }
    }
    return FMA_B200_OK;
}

template <typename T>
static int launch_few(const FewRows& p, int64_t items, cudaStream_t s) {
    if (int rc = allow_smem(few_rows_kernel<T>)) return rc;
    return launch_kernel("fp8_few_rows", few_rows_kernel<T>, dim3(static_cast<unsigned>(items * p.split)), kFewThreads,
                          static_cast<size_t>(few_smem(p.quads_most)), static_cast<unsigned>(p.split), s, p);
}

template <typename T>
static int launch_some(const SomeRows& p, int64_t items, cudaStream_t s) {
    if (int rc = allow_smem(some_rows_kernel<T>)) return rc;
    const size_t smem = static_cast<size_t>(p.stages) * (kFewStageBytes + p.cols_most * FP8_BLOCK) + 1024;
    return launch_kernel("fp8_some_rows", some_rows_kernel<T>, dim3(static_cast<unsigned>(items * p.split)), kSomeThreads, smem,
                          static_cast<unsigned>(p.split), s, p);
}

// Called by fma_b200_fp8_gemm, which has checked its arguments; `active` = row tiles that are expected to have rows.
int fp8_some_rows(const void* x, const void* x_scales, int64_t layout_rows, const void* w, const void* w_scales, int32_t E, int32_t N,
                  int32_t K, void* out, int32_t dtype, int64_t out_rows, const int32_t* tile_expert, const int32_t* tile_row,
                  const int32_t* tile_rows, const int32_t* rows_used, int64_t active, cudaStream_t s) {
    SomeRows p;
    memset(&p, 0, sizeof(p));
    p.status = device_status_ptr();
    FMAB_REQUIRE(p.status != nullptr, FMA_B200_ERR_LAUNCH, "no device status word");
    p.w_scales = static_cast<const uint8_t*>(w_scales);
    p.x_scales = static_cast<const uint8_t*>(x_scales);
    p.out = out;
    p.tile_expert = tile_expert;
    p.tile_row = tile_row;
    p.tile_rows = tile_rows;
    p.rows_used = rows_used;
    p.out_rows = out_rows;
    p.layout_rows = layout_rows;
    p.N = N;
    p.k_blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    p.quads = static_cast<int32_t>(fp8_quads(K));
    p.tiles = static_cast<int32_t>(fp8_row_tiles(N));
    p.w_tiles = E * p.tiles;
    p.x_tiles = static_cast<int32_t>(fp8_row_tiles(layout_rows));
    p.split = few_split(active * p.tiles, p.quads, kSomeQuadsFit);
    p.quads_most = (p.quads + p.split - 1) / p.split;
    p.cols_most = 128;
    if (tile_expert == nullptr) p.cols_most = layout_rows <= 16 ? 16 : (layout_rows <= 32 ? 32 : (layout_rows <= 64 ? 64 : 128));
    p.tmem_cols = 32;
    while (p.tmem_cols < static_cast<uint32_t>(p.cols_most + kFewScaleCols * p.quads_most)) p.tmem_cols *= 2;
    p.stages = 104 * 1024 / (kFewStageBytes + p.cols_most * FP8_BLOCK);  // two CTAs per SM; the ring later holds the parts
    const int64_t items = static_cast<int64_t>(p.x_tiles) * p.tiles;
    FMAB_REQUIRE(items * p.split < (1LL << 31), FMA_B200_ERR_BAD_ARG, "too many tiles");
    if (int rc = encode_bytes(&p.map_w, w, K, static_cast<uint64_t>(E) * N, fp8_pitch(K), 128)) return rc;
    for (int i = 0; i < kSomeBoxes; ++i)
        if (int rc = encode_bytes(&p.map_x[i], x, K, static_cast<uint64_t>(layout_rows), fp8_pitch(K), 16u << i)) return rc;
    return dtype == FMA_B200_BF16 ? launch_some<__nv_bfloat16>(p, items, s) : launch_some<__half>(p, items, s);
}
bool fp8_some_rows_fits(int32_t K) { return fp8_quads(K) <= 8LL * kSomeQuadsFit; }

}  // namespace fmab

extern "C" {

int fma_b200_fp8_few_rows(const void* x, int64_t x_pitch, int32_t dtype, int64_t rows, const void* w, const void* w_scales,
                          int32_t E, int32_t N, int32_t K, const void* counts, int32_t index_bytes, void* out, void* stream) {
    using namespace fmab;
    FMAB_REQUIRE(dtype == FMA_B200_BF16 || dtype == FMA_B200_F16, FMA_B200_ERR_UNSUPPORTED,
                 "dtype %d: the 8-bit product takes and returns bfloat16 or half", dtype);
    FMAB_REQUIRE(rows >= 0 && rows < (1LL << 30), FMA_B200_ERR_BAD_ARG, "rows=%lld", (long long)rows);
    FMAB_REQUIRE(E >= 1 && E <= 1024, FMA_B200_ERR_BAD_ARG, "E=%d not in [1,1024]", E);
    FMAB_REQUIRE(N >= 8 && K >= 8 && N % 8 == 0 && K % 8 == 0 && N < (1 << 30) && K < (1 << 30), FMA_B200_ERR_BAD_ARG,
                 "N=%d and K=%d must be positive multiples of 8", N, K);
    FMAB_REQUIRE(static_cast<int64_t>(E) * N < (1LL << 31) - 1024, FMA_B200_ERR_BAD_ARG, "E*N overflows");
    FMAB_REQUIRE(x_pitch >= K && x_pitch % 8 == 0, FMA_B200_ERR_BAD_ARG, "x: row pitch %lld", (long long)x_pitch);
    FMAB_REQUIRE(E == 1 || counts != nullptr, FMA_B200_ERR_BAD_ARG, "several experts need their counts");
    FMAB_REQUIRE(counts == nullptr || known_index_bytes(index_bytes), FMA_B200_ERR_UNSUPPORTED, "index_bytes=%d", index_bytes);
    if (rows == 0) return FMA_B200_OK;
    FMAB_REQUIRE(x && w && w_scales && out, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(x) && aligned16(w) && aligned16(w_scales) && aligned16(out), FMA_B200_ERR_BAD_ARG,
                 "pointers not 16-byte aligned");
    FewRows p;
    memset(&p, 0, sizeof(p));
    p.status = device_status_ptr();
    FMAB_REQUIRE(p.status != nullptr, FMA_B200_ERR_LAUNCH, "no device status word");
    p.x = x;
    p.x_pitch = x_pitch;
    p.w_scales = static_cast<const uint8_t*>(w_scales);
    p.out = out;
    p.counts = counts;
    p.index_bytes = index_bytes;
    p.E = E;
    p.rows = static_cast<int32_t>(rows);
    p.N = N;
    p.K = K;
    p.k_blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    p.quads = static_cast<int32_t>(fp8_quads(K));
    p.tiles = static_cast<int32_t>(fp8_row_tiles(N));
    p.b_tiles = E * p.tiles;
    const int64_t items = few_chunks(rows, E, counts != nullptr) * p.tiles;
    p.split = few_split(few_chunks_even(rows, E) * p.tiles, p.quads, FEW_QUADS_TWO);
    p.quads_most = (p.quads + p.split - 1) / p.split;
    p.tmem_cols = 32;
    while (p.tmem_cols < static_cast<uint32_t>(kFewScaleCol + kFewScaleCols * p.quads_most)) p.tmem_cols *= 2;
    FMAB_REQUIRE(p.quads_most <= FEW_QUADS_MOST, FMA_B200_ERR_UNSUPPORTED, "K=%d is too large for the product of a few rows", K);
    FMAB_REQUIRE(items * p.split < (1LL << 31), FMA_B200_ERR_BAD_ARG, "too many tiles");
    if (int rc = encode_bytes(&p.map_w, w, K, static_cast<uint64_t>(E) * N, fp8_pitch(K), 128)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == FMA_B200_BF16 ? launch_few<__nv_bfloat16>(p, items, s) : launch_few<__half>(p, items, s);
}

}  // extern "C"
