// Kernels around the 8-bit format of fp8.cuh: quantising rows (plain, grouped by expert, or scattered to the expert
// layout of the MoE layer), quantising weights, dequantising, and SwiGLU that keeps its inputs in 8 bits for the backward
// pass.  All are bound by HBM traffic: one pass over the data, 128-bit reads, every value read once and written once; the
// block maximum lives in registers between the two.
#include "fp8.cuh"
#include "gemm_tc.cuh"

namespace fmab {

constexpr int kQThreads = 256;
constexpr int kQWarps = kQThreads / 32;

// Work of the row kernels: blocks of 128 columns, row after row; 8 lanes have a block each, a warp four in a row, and the
// loads of several such steps are in flight before the first is touched, one where there are few blocks.  With rows as the
// unit (four groups of 512 columns in flight) widths that are no multiple of 2048 left lanes or loads idle: 65536 rows of
// 768 / 1536 / 2048 columns took 47 / 59 / 71.7 us and take 32 / 55 / 70.7 (4096: 131 us, 6.1 TB/s), back to 16 bits 41 / 56 /
// 69 and 32 / 54 / 69.
struct RowItems {
    uint32_t units, blocks;            // blocks in all, and in a row
    uint32_t step_rows, step_blocks;   // four blocks further
    int32_t ahead;                     // steps of a warp at a time: a template argument of the kernels
};
struct RowPlace {
    uint32_t row, block;
    __device__ __forceinline__ RowPlace(const RowItems& w, uint32_t unit) : row(unit / w.blocks), block(unit - row * w.blocks) {}
    __device__ __forceinline__ void next(const RowItems& w) {
        row += w.step_rows;
        block += w.step_blocks;
        if (block >= w.blocks) {
            block -= w.blocks;
            ++row;
        }
    }
};
template <typename T>
constexpr int kAhead = Elem<T>::kPerVec == 8 ? 4 : 2;

// Where a source row goes.  rows: to itself.  groups: rows of expert e are consecutive in the source
// ([offsets[e], offsets[e+1])) and start at pad_offsets[e] in the layout.  slots: source row t goes to the k rows
// row_of_slot[t*k ..] of the MoE layer's layout.
constexpr int TO_ROWS = 0, TO_GROUPS = 1, TO_SLOTS = 2;
struct QuantRows {
    const void* x;
    void* copy;               // groups: the rows themselves in the padded layout too, or null
    uint8_t* values;
    uint8_t* scales;
    const int32_t* offsets;
    const int32_t* pad_offsets;
    const int32_t* row_of_slot;
    const int32_t* slot_of_row;
    const int32_t* rows_used; // rows: source rows from here on are left alone; null: all rows
    int64_t x_pitch;
    int64_t rows;             // source rows
    RowItems work;
    uint32_t row_blocks;      // blocks that quantise; the others zero the padding rows
    int64_t layout_rows;
    int64_t row_tiles;        // scale tiles per quad
    int32_t cols, pitch, n_groups, k;
};

// Largest e with offsets[e] <= row (empty experts are skipped: of equal offsets the last one counts).
__device__ __forceinline__ int group_of_row(const int32_t* offsets, int n, int32_t row) {
    int lo = 0, hi = n;  // offsets[lo] <= row < offsets[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(offsets + mid) <= row) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ void zero_row(const QuantRows& p, int64_t row) {
    const int lane = threadIdx.x & 31;
    for (int c = lane * 16; c < p.pitch; c += 512) st_global_16(p.values + row * p.pitch + c, make_uint4(0, 0, 0, 0));
    for (int q = lane; q * 4 < static_cast<int>(p.work.blocks); q += 32)
        *reinterpret_cast<uint32_t*>(p.scales + fp8_scale_word(row, q, p.row_tiles)) = 0x01010101u * FP8_SCALE_ONE;
    if (p.copy != nullptr) {
        constexpr int V = Elem<T>::kPerVec;
        for (int c = lane * V; c < p.cols; c += 32 * V) st_global_16(static_cast<T*>(p.copy) + row * p.cols + c, make_uint4(0, 0, 0, 0));
    }
}

// Padding rows: zero values, zero copies.  slots: all below the layout's used end, since whole tiles are written from
// them; groups: up to a multiple of 64, the rows that the weight gradient reads.
template <typename T, int TO>
__device__ void zero_padding_rows(const QuantRows& p, uint32_t warp_id, uint32_t n_warps) {
    if (TO == TO_SLOTS) {
        const int64_t used = min(static_cast<int64_t>(p.pad_offsets[p.n_groups]), p.layout_rows);
        for (int64_t row = warp_id; row < used; row += n_warps)
            if (p.slot_of_row[row] < 0) zero_row<T>(p, row);
    } else {
        for (uint32_t i = warp_id; i < static_cast<uint32_t>(p.n_groups) * 8; i += n_warps) {  // eight warps per group
            const int e = static_cast<int>(i >> 3);
            const int64_t count = p.offsets[e + 1] - p.offsets[e], first = p.pad_offsets[e];
            const int64_t end = min(first + (count + 63) / 64 * 64, p.layout_rows);
            for (int64_t row = first + count + (i & 7); row < end; row += 8) zero_row<T>(p, row);
        }
    }
}

template <typename T, int TO, int AHEAD>
__global__ void __launch_bounds__(kQThreads) quantize_rows_kernel(const QuantRows p) {
    constexpr int N = LaneBlock<T>::N;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = lane & 7, g = lane >> 3;
    if (TO != TO_ROWS && blockIdx.x >= p.row_blocks) {
        zero_padding_rows<T, TO>(p, (blockIdx.x - p.row_blocks) * kQWarps + warp, (gridDim.x - p.row_blocks) * kQWarps);
        return;
    }
    const int64_t rows = TO == TO_ROWS && p.rows_used != nullptr ? min(p.rows, static_cast<int64_t>(*p.rows_used)) : p.rows;
    const int64_t known = TO == TO_GROUPS ? min(rows, static_cast<int64_t>(__ldg(p.offsets + p.n_groups))) : rows;  // the others: no expert
    const uint32_t n_warps = p.row_blocks * kQWarps;
    for (uint64_t first = (blockIdx.x * kQWarps + warp) * 4ull * AHEAD; first < p.work.units; first += n_warps * 4ull * AHEAD) {
        RowPlace at(p.work, static_cast<uint32_t>(first) + g);  // units stay below 2^32 by more than a step
        uint32_t row[AHEAD], block[AHEAD];
        uint4 raw[AHEAD][N];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            row[u] = at.row;
            block[u] = at.block;
            const T* const src = static_cast<const T*>(p.x) + at.row * p.x_pitch;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int c = static_cast<int>(at.block) * FP8_BLOCK + LaneBlock<T>::column(s, j);
                raw[u][j] = row[u] < known && c < p.cols ? ld_stream_16(src + c) : make_uint4(0, 0, 0, 0);
            }
            at.next(p.work);
        }
        int64_t layout_row = -1;  // groups: lane s finds where row[s] goes, while the loads are on their way
        if (TO == TO_GROUPS) {
            uint32_t mine = row[0];
#pragma unroll
            for (int u = 1; u < AHEAD; ++u) mine = s == u ? row[u] : mine;
            if (mine < known) {
                const int e = group_of_row(p.offsets, p.n_groups, static_cast<int32_t>(mine));
                layout_row = __ldg(p.pad_offsets + e) + (static_cast<int64_t>(mine) - __ldg(p.offsets + e));
                if (layout_row >= p.layout_rows) layout_row = -1;
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int col0 = static_cast<int>(block[u]) * FP8_BLOCK;
            uint32_t w[4];
            const uint32_t byte = quantize_lane_raw<T>(raw[u], w);
            int64_t to = row[u];
            if (TO == TO_GROUPS) to = __shfl_sync(0xffffffffu, layout_row, (lane & 24) | u);
            if (row[u] >= known || to < 0) continue;
            const int copies = TO == TO_SLOTS ? p.k : 1;
            for (int j = 0; j < copies; ++j) {
                if (TO == TO_SLOTS) {
                    to = __ldg(p.row_of_slot + static_cast<int64_t>(row[u]) * p.k + j);
                    if (to < 0 || to >= p.layout_rows) continue;
                }
                store_lane_bytes<T>(p.values + to * p.pitch, col0, p.pitch, s, w);
                if (s == 0) p.scales[fp8_scale_word(to, block[u] >> 2, p.row_tiles) + (block[u] & 3)] = static_cast<uint8_t>(byte);
            }
            if (TO == TO_GROUPS && p.copy != nullptr) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int c = col0 + LaneBlock<T>::column(s, j);
                    if (c < p.cols) st_global_16(static_cast<T*>(p.copy) + to * p.cols + c, raw[u][j]);
                }
            }
        }
    }
}

// ---- weights ---------------------------------------------------------------------------------------
// One CTA per block of 128 x 128.  A thread holds 8 rows x 8 columns; its rows leave as 8-byte pieces.
struct QuantWeight {
    const void* w;
    uint8_t *values, *scales;
    int32_t E, N, K, pitch;
    int32_t n_blocks, k_blocks;  // per expert
};

template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(const QuantWeight p) {
    __shared__ uint32_t warp_max[8];
    constexpr int V = Elem<T>::kPerVec;
    const int tid = threadIdx.x;
    const int kb = blockIdx.x % p.k_blocks;
    const int nb = blockIdx.x / p.k_blocks;
    const int e = blockIdx.y;
    const int r0 = nb * FP8_BLOCK + (tid >> 4) * 8, c0 = kb * FP8_BLOCK + (tid & 15) * 8;
    const T* src = static_cast<const T*>(p.w) + (static_cast<int64_t>(e) * p.N + r0) * p.K + c0;
    uint4 raw[8][8 / V];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8 / V; ++j)
            raw[i][j] = (r0 + i < p.N && c0 < p.K) ? ld_stream_16(src + static_cast<int64_t>(i) * p.K + j * V) : make_uint4(0, 0, 0, 0);
    auto block_max = [&](uint32_t m) {
        m = __reduce_max_sync(0xffffffffu, m);
        if ((tid & 31) == 0) warp_max[tid >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, warp_max[i]);
        return m;
    };
    uint32_t m = 0;
    bool finite = false;
    if constexpr (Magnitude16<T>::kPacked) {
        uint32_t pair = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) pair = max_magnitudes16(pair, raw[i][0]);
        m = block_max(max(pair & 0xffffu, pair >> 16));
        finite = m < Magnitude16<T>::kInf;
        m = Magnitude16<T>::float_bits(m);
        if (!finite) __syncthreads();  // warp_max is written again
    }
    if (!finite) {
        m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8 / V; ++j) {
                float x[V];
                Elem<T>::unpack(raw[i][j], x);
#pragma unroll
                for (int v = 0; v < V; ++v) m = max(m, fp8_magnitude(x[v]));
            }
        m = block_max(m);
    }
    const uint32_t byte = fp8_scale_byte(m);
    const float inverse = fp8_inverse(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8 / V; ++j) Elem<T>::unpack(raw[i][j], x + j * V);
        const uint32_t lo = finite ? fp8_pack4_finite(x, inverse) : fp8_pack4(x, inverse);
        const uint32_t hi = finite ? fp8_pack4_finite(x + 4, inverse) : fp8_pack4(x + 4, inverse);
        if (r0 + i < p.N && c0 < p.pitch)
            *reinterpret_cast<uint2*>(p.values + (static_cast<int64_t>(e) * p.N + r0 + i) * p.pitch + c0) = make_uint2(lo, hi);
    }
    if (tid < FP8_BLOCK)
        p.scales[fp8_scale_word((static_cast<int64_t>(e) * p.n_blocks + nb) * FP8_BLOCK + tid, kb >> 2,
                                static_cast<int64_t>(p.E) * p.n_blocks) + (kb & 3)] = static_cast<uint8_t>(byte);
}

// ---- back to 16 or 32 bits -------------------------------------------------------------------------
// Rounds once; what a rounding up to e4m3 lifted above the type's range comes back as its largest finite value.
template <typename T>
__device__ __forceinline__ float finite_in(float x);
template <>
__device__ __forceinline__ float finite_in<float>(float x) { return fabsf(x) > 3.402823466e38f ? copysignf(3.402823466e38f, x) : x; }
template <>
__device__ __forceinline__ float finite_in<__nv_bfloat16>(float x) { return fabsf(x) > 3.389531390e38f ? copysignf(3.389531390e38f, x) : x; }
template <>
__device__ __forceinline__ float finite_in<__half>(float x) { return fabsf(x) > 65504.f ? copysignf(65504.f, x) : x; }

struct Dequant {
    const uint8_t *values, *scales;
    void* out;
    const int32_t* rows_used;  // rows from here on are left alone; null: all rows
    int64_t rows, row_tiles;   // rows over the whole batch
    RowItems work;
    int32_t batch, rows_per, tiles_per, cols, pitch;  // of one matrix of the batch
};

template <typename T, int AHEAD>
__global__ void __launch_bounds__(kQThreads) dequantize_rows_kernel(const Dequant p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = lane & 7, g = lane >> 3;
    const int64_t rows = p.rows_used != nullptr ? min(p.rows, static_cast<int64_t>(*p.rows_used)) : p.rows;
    for (uint64_t first = (blockIdx.x * kQWarps + warp) * 4ull * AHEAD; first < p.work.units; first += gridDim.x * kQWarps * 4ull * AHEAD) {
        RowPlace at(p.work, static_cast<uint32_t>(first) + g);
        uint32_t row[AHEAD], block[AHEAD], w[AHEAD][4];
        uint8_t byte[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            row[u] = at.row;
            block[u] = at.block;
            byte[u] = FP8_SCALE_ONE;
            if (row[u] < rows) {
                int64_t scale_row = at.row;
                if (p.batch > 1) {
                    const uint32_t b = at.row / static_cast<uint32_t>(p.rows_per);
                    scale_row = static_cast<int64_t>(b) * p.tiles_per * FP8_TILE_ROWS + (at.row - static_cast<int64_t>(b) * p.rows_per);
                }
                load_lane_bytes<T>(p.values + static_cast<int64_t>(at.row) * p.pitch, static_cast<int>(at.block) * FP8_BLOCK, p.pitch, s, w[u]);
                byte[u] = p.scales[fp8_scale_word(scale_row, at.block >> 2, p.row_tiles) + (at.block & 3)];
            }
            at.next(p.work);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (row[u] >= rows) continue;
            const float factor = fp8_factor(byte[u]);
            float x[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) fp8_unpack4(w[u][j], factor, x + 4 * j);
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = finite_in<T>(x[j]);
            store_lane_block<T>(static_cast<T*>(p.out) + static_cast<int64_t>(row[u]) * p.cols, static_cast<int>(block[u]) * FP8_BLOCK, p.cols, s, x);
        }
    }
}

// ---- SwiGLU with 8-bit checkpoints -----------------------------------------------------------------
// forward:  out = up * gate * sigmoid(gate) from the inputs as they came; up and gate are kept in 8 bits, and, for the
// next 8-bit product, out as well.  backward: from the kept values,
//   d_up = d * silu(gate),  d_gate = d * up * (s + silu(gate) * (1 - s)),  s = sigmoid(gate).
// Next to the 16-bit SwiGLU the forward pass writes 2 bytes more per element and the backward reads 2 fewer; what
// stays alive between the two is half as large.  16-bit results take the approximate exponential and reciprocal
// (two units in the last place of fp32), fp32 results the full ones.
// 16 values of up (u) and gate (x): x = u * x * sigmoid(x).  For results of 16 bits with the packed arithmetic and the
// approximate exponential and reciprocal of the product's epilogue.
template <typename T>
__device__ __forceinline__ void swiglu_16(const float* u, float* x) {
    swiglu_fwd8(u, x, x);
    swiglu_fwd8(u + 8, x + 8, x + 8);
}
template <>
__device__ __forceinline__ void swiglu_16<float>(const float* u, float* x) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = u[j] * x[j] * sigmoid_clamped(x[j]);
}
// and with the upstream gradient d: u and x become their gradients
template <typename T>
__device__ __forceinline__ void swiglu_grad_16(const float* d, float* u, float* x) {
    swiglu_bwd8(d, u, x, u, x);
    swiglu_bwd8(d + 8, u + 8, x + 8, u + 8, x + 8);
}
template <>
__device__ __forceinline__ void swiglu_grad_16<float>(const float* d, float* u, float* x) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float sg = sigmoid_clamped(x[j]);
        const float silu = x[j] * sg;
        x[j] = d[j] * u[j] * (sg + silu * (1.f - sg));
        u[j] = d[j] * silu;
    }
}

// Here every 8 lanes take the next block of 128 columns, whichever row it is in: with widths that are no multiple of 512
// no lane is idle (768 columns: 517 us for 294912 rows with a group of 512 columns per warp).
struct SwigluFp8 {
    const void *gate, *up, *dy;
    void *out, *gate_grad, *up_grad;
    int64_t gate_pitch, up_pitch, dy_pitch, out_pitch, gate_grad_pitch, up_grad_pitch;
    uint8_t *gate8, *gate_scales, *up8, *up_scales, *out8, *out_scales;
    uint8_t *grad8, *grad_scales;  // backward: [up_grad | gate_grad] in 8 bits, rows of 2 cols
    const int32_t* rows_used;
    int64_t rows, row_tiles;
    int32_t cols, pitch, blocks;   // blocks of 128 columns per row
};
// The blocks of 8 lanes in turn: the next one is a fixed number of rows and blocks further.  Behind the last row `in` is
// false and the place is one that exists.
struct LanePlace {
    int64_t row;
    int32_t block, col0;
    bool in;
    __device__ __forceinline__ LanePlace(uint32_t unit, uint32_t step, int64_t rows, int32_t blocks) : rows_(rows), blocks_(blocks) {
        const uint32_t n = blocks, at = unit / n;
        at_ = at;
        block = static_cast<int32_t>(unit - at * n);
        step_rows_ = step / n;
        step_blocks_ = static_cast<int32_t>(step - step_rows_ * n);
        set();
    }
    __device__ __forceinline__ void next() {
        at_ += step_rows_;
        block += step_blocks_;
        if (block >= blocks_) {
            block -= blocks_;
            ++at_;
        }
        set();
    }

private:
    int64_t at_, rows_;
    uint32_t step_rows_;
    int32_t blocks_, step_blocks_;
    __device__ __forceinline__ void set() {
        in = at_ < rows_;
        row = in ? at_ : 0;
        col0 = block * FP8_BLOCK;
    }
};
template <typename T>
__device__ __forceinline__ void load_lane_raw(const void* base, int64_t row, int64_t pitch, const LanePlace& t, int cols, int s, uint4* raw) {
#pragma unroll
    for (int j = 0; j < LaneBlock<T>::N; ++j) {
        const int c = t.col0 + LaneBlock<T>::column(s, j);
        raw[j] = t.in && c < cols ? ld_stream_16(static_cast<const T*>(base) + row * pitch + c) : make_uint4(0, 0, 0, 0);
    }
}
// Quantises a lane's 16 values of the block `block` of an 8-bit matrix with row pitch `pitch` and its scales.
template <typename T>
__device__ __forceinline__ void store_lane_quantized(const uint4* raw, uint8_t* values, uint8_t* scales, int64_t row, int block, int pitch,
                                                     int64_t row_tiles, bool in, int s) {
    uint32_t w[4];
    const uint32_t byte = quantize_lane_raw<T>(raw, w);
    if (!in) return;
    store_lane_bytes<T>(values + row * pitch, block * FP8_BLOCK, pitch, s, w);
    if (s == 0) scales[fp8_scale_word(row, block >> 2, row_tiles) + (block & 3)] = static_cast<uint8_t>(byte);
}
template <typename T>
__device__ __forceinline__ void pack_lane(const float* x, uint4* raw) {
#pragma unroll
    for (int j = 0; j < LaneBlock<T>::N; ++j) raw[j] = Elem<T>::pack(x + j * LaneBlock<T>::V);
}
template <typename T>
__device__ __forceinline__ void store_lane_raw(const uint4* raw, void* base, int64_t pitch, const LanePlace& t, int cols, int s) {
#pragma unroll
    for (int j = 0; j < LaneBlock<T>::N; ++j) {
        const int c = t.col0 + LaneBlock<T>::column(s, j);
        if (t.in && c < cols) st_global_16(static_cast<T*>(base) + t.row * pitch + c, raw[j]);
    }
}

// What bounds both, where the layer has all results written, is instructions (81 % of the issue slots before the packed
// arithmetic, 131072 rows of 768 columns forward 153 us, 133 with it, 5.3 TB/s; backward 192 and 164, 6.1 TB/s).
template <typename T>
__global__ void __launch_bounds__(kQThreads) swiglu_fp8_forward_kernel(const SwigluFp8 p) {
    constexpr int N = LaneBlock<T>::N, V = LaneBlock<T>::V;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = lane & 7, g = lane >> 3;
    const int64_t rows = p.rows_used != nullptr ? min(p.rows, static_cast<int64_t>(*p.rows_used)) : p.rows;
    const uint32_t first = (blockIdx.x * kQWarps + warp) * 4, step = gridDim.x * kQWarps * 4;
    for (LanePlace t(first + g, step, rows, p.blocks); __any_sync(0xffffffffu, t.in); t.next()) {
        uint4 rg[N], ru[N];
        load_lane_raw<T>(p.gate, t.row, p.gate_pitch, t, p.cols, s, rg);
        load_lane_raw<T>(p.up, t.row, p.up_pitch, t, p.cols, s, ru);
        if (p.gate8 != nullptr) store_lane_quantized<T>(rg, p.gate8, p.gate_scales, t.row, t.block, p.pitch, p.row_tiles, t.in, s);
        if (p.up8 != nullptr) store_lane_quantized<T>(ru, p.up8, p.up_scales, t.row, t.block, p.pitch, p.row_tiles, t.in, s);
        float x[16], u[16];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            Elem<T>::unpack(rg[j], x + j * V);
            Elem<T>::unpack(ru[j], u + j * V);
        }
        swiglu_16<T>(u, x);
        pack_lane<T>(x, rg);
        if (p.out != nullptr) store_lane_raw<T>(rg, p.out, p.out_pitch, t, p.cols, s);
        // from the rounded values: what a separate quantisation of `out` gives
        if (p.out8 != nullptr) store_lane_quantized<T>(rg, p.out8, p.out_scales, t.row, t.block, p.pitch, p.row_tiles, t.in, s);
    }
}

// Four blocks per SM: 131072 rows of 768 columns with grad8 164 us; with the three or five that other register counts give
// 178 and 182.
template <typename T>
__global__ void __launch_bounds__(kQThreads, sizeof(T) == 4 ? 3 : 4) swiglu_fp8_backward_kernel(const SwigluFp8 p) {
    constexpr int N = LaneBlock<T>::N, V = LaneBlock<T>::V;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = lane & 7, g = lane >> 3;
    const int64_t rows = p.rows_used != nullptr ? min(p.rows, static_cast<int64_t>(*p.rows_used)) : p.rows;
    const uint32_t first = (blockIdx.x * kQWarps + warp) * 4, step = gridDim.x * kQWarps * 4;
    for (LanePlace t(first + g, step, rows, p.blocks); __any_sync(0xffffffffu, t.in); t.next()) {
        const int64_t scale_at = fp8_scale_word(t.row, t.block >> 2, p.row_tiles) + (t.block & 3);
        uint32_t wg[4], wu[4];
        uint4 rd[N];
        load_lane_bytes<T>(p.gate8 + t.row * p.pitch, t.col0, p.pitch, s, wg);
        load_lane_bytes<T>(p.up8 + t.row * p.pitch, t.col0, p.pitch, s, wu);
        load_lane_raw<T>(p.dy, t.row, p.dy_pitch, t, p.cols, s, rd);
        const float fg = fp8_factor(p.gate_scales[scale_at]), fu = fp8_factor(p.up_scales[scale_at]);
        float d[16], x[16], u[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            fp8_unpack4(wg[j], fg, x + 4 * j);
            fp8_unpack4(wu[j], fu, u + 4 * j);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) Elem<T>::unpack(rd[j], d + j * V);
        swiglu_grad_16<T>(d, u, x);
        uint4 raw[N];
        pack_lane<T>(u, raw);
        store_lane_raw<T>(raw, p.up_grad, p.up_grad_pitch, t, p.cols, s);
        if (p.grad8 != nullptr) store_lane_quantized<T>(raw, p.grad8, p.grad_scales, t.row, t.block, 2 * p.cols, p.row_tiles, t.in, s);
        pack_lane<T>(x, raw);
        store_lane_raw<T>(raw, p.gate_grad, p.gate_grad_pitch, t, p.cols, s);
        if (p.grad8 != nullptr) store_lane_quantized<T>(raw, p.grad8, p.grad_scales, t.row, t.block + p.blocks, 2 * p.cols, p.row_tiles, t.in, s);
    }
}

// ---- maps of rows that are grouped by expert without alignment -------------------------------------
// One block.  offsets[e] = first source row of expert e, limited to the rows there are (a count that overshoots is cut
// off, never followed); pad_offsets[e] = first row of e in the 256-aligned layout; per 128-row tile of the layout the
// expert, the first source row and the number of source rows.  Source rows behind the last expert's are a group of
// their own with expert -2: the product writes zeros for them.  Tiles behind the last used one have expert -1.
constexpr int kMapThreads = 1024;
struct GroupMaps {
    const void* counts;
    int32_t *offsets, *pad_offsets, *group_rows, *tile_expert, *tile_row, *tile_rows;
    int64_t rows;
    int32_t index_bytes, E, n_tiles;
};

// Inclusive running sum over the block, cut off at `most` (below 2^31) at every step: cut-off sums add up in any order.
__device__ __forceinline__ uint32_t running_sum(uint32_t v, uint32_t most, uint32_t* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t add = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v = min(v + add, most);
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    uint32_t before = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t add = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before = min(before + add, most);
    }
    before = __shfl_sync(0xffffffffu, before, warp > 0 ? warp - 1 : 0);
    return warp > 0 ? min(v + before, most) : v;
}

// 128 experts, 16384 rows: 2.7 us; with sums over shared memory in log2(1024) rounds 4.2.
__global__ void __launch_bounds__(kMapThreads) group_maps_kernel(const GroupMaps p) {
    static_assert(kMapThreads == 1024, "32 warps, one lane each");
    __shared__ int32_t off[1024 + 2], pad[1024 + 3];
    __shared__ uint32_t warp_sums[2][32];
    const int t = threadIdx.x;
    const int n = p.E;  // groups 0..n-1 are experts, group n the rows of no expert
    const uint32_t c = t < n ? static_cast<uint32_t>(fp8_count(p.counts, p.index_bytes, t, p.rows)) : 0;
    const uint32_t end = running_sum(c, static_cast<uint32_t>(p.rows), warp_sums[0]);
    if (t < n) off[t + 1] = static_cast<int32_t>(end);
    if (t == 0) off[0] = 0;
    __syncthreads();
    const uint32_t tiles = t < n ? (off[t + 1] - off[t] + 255) / 256 : 0;
    const uint32_t tiles_end = running_sum(tiles, 0x7fffffffu, warp_sums[1]);
    if (t < n) pad[t + 1] = static_cast<int32_t>(tiles_end * 256);
    if (t == 0) pad[0] = 0;
    __syncthreads();
    const int32_t rest = static_cast<int32_t>(p.rows) - off[n];
    if (t == 0) pad[n + 1] = pad[n] + (rest + 255) / 256 * 256;
    __syncthreads();
    if (t < n) p.group_rows[t] = off[t + 1] - off[t];
    for (int i = t; i <= n; i += kMapThreads) {  // n + 1 entries: one more than threads with 1024 experts
        p.offsets[i] = off[i];
        p.pad_offsets[i] = pad[i];
    }
    if (t == 0) p.pad_offsets[n + 1] = pad[n + 1];
    for (int i = t; i < p.n_tiles; i += kMapThreads) {
        const int32_t row = i * 128;
        int32_t e = -1, first = 0, count = 0;
        if (row < pad[n + 1]) {
            int lo = 0, hi = n + 1;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (pad[mid] <= row) lo = mid; else hi = mid;
            }
            const int32_t inside = row - pad[lo];
            const int32_t size = lo < n ? off[lo + 1] - off[lo] : rest;
            first = off[lo] + inside;
            count = max(0, min(128, size - inside));
            e = lo < n ? lo : -2;
        }
        p.tile_expert[i] = e;
        p.tile_row[i] = first;
        p.tile_rows[i] = count;
    }
}

// ---- host side -------------------------------------------------------------------------------------
// At most 32 blocks of 256 threads per SM, about six rounds of them: 16384 x 4096 to 8 bits and back 71.7 us (64: 73.5, 8:
// 73.5), SwiGLU of 32781 x 1536 forward and backward 134 us (137, 144).
static uint32_t row_grid(int64_t items) {
    const int64_t want = (items + kQWarps - 1) / kQWarps;
    const int64_t cap = static_cast<int64_t>(sm_count()) * 32;
    return static_cast<uint32_t>(want < 1 ? 1 : (want > cap ? cap : want));
}
static int make_items(RowItems& w, int64_t rows, int64_t cols, int32_t most) {
    w.blocks = static_cast<uint32_t>((cols + FP8_BLOCK - 1) / FP8_BLOCK);
    w.step_rows = 4 / w.blocks;
    w.step_blocks = 4 % w.blocks;
    const int64_t units = rows * w.blocks;
    FMAB_REQUIRE(units < (1LL << 32) - (1LL << 10), FMA_B200_ERR_BAD_ARG, "rows=%lld of %lld columns are too many", (long long)rows,
                 (long long)cols);
    w.units = static_cast<uint32_t>(units);
    w.ahead = most;
    if (units < 16LL * sm_count() * 4 * most) w.ahead = 1;  // 16 warps on every SM come first
    return FMA_B200_OK;
}

static int check_rows_cols(int32_t dtype, int64_t rows, int64_t cols) {
    FMAB_REQUIRE(known_dtype(dtype), FMA_B200_ERR_UNSUPPORTED, "dtype %d", dtype);
    FMAB_REQUIRE(rows >= 0 && rows < (1LL << 31), FMA_B200_ERR_BAD_ARG, "rows=%lld not in [0, 2^31)", (long long)rows);
    FMAB_REQUIRE(cols >= 8 && cols % 8 == 0 && cols < (1LL << 30), FMA_B200_ERR_BAD_ARG,
                 "cols=%lld must be a positive multiple of 8 below 2^30", (long long)cols);
    return FMA_B200_OK;
}
static int check_pitch(const char* what, int32_t dtype, int64_t pitch, int64_t cols) {
    FMAB_REQUIRE(pitch >= cols && pitch % elems_per_16_bytes(dtype) == 0, FMA_B200_ERR_BAD_ARG,
                 "%s: row pitch %lld is below the width or not a multiple of 16 bytes", what, (long long)pitch);
    return FMA_B200_OK;
}

template <int TO>
static int launch_quantize(QuantRows& p, int32_t dtype, int64_t extra_rows, cudaStream_t s) {
    p.row_blocks = row_grid((p.work.units + 4LL * p.work.ahead - 1) / (4 * p.work.ahead));
    const uint32_t grid = p.row_blocks + (TO != TO_ROWS ? row_grid(extra_rows) : 0);
    int rc = FMA_B200_OK;
    dispatch_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        rc = launch_kernel("fp8_quantize", p.work.ahead == 1 ? quantize_rows_kernel<T, TO, 1> : quantize_rows_kernel<T, TO, kAhead<T>>,
                           dim3(grid), kQThreads, 0, 0, s, p);
    });
    return rc;
}

static int fill_quantize(QuantRows& p, const void* x, int64_t x_pitch, int32_t dtype, int64_t rows, int64_t cols,
                         int64_t layout_rows, void* values, void* scales) {
    if (int rc = check_rows_cols(dtype, rows, cols)) return rc;
    if (int rc = check_rows_cols(dtype, layout_rows, cols)) return rc;
    if (int rc = check_pitch("x", dtype, x_pitch, cols)) return rc;
    memset(&p, 0, sizeof(p));
    p.x = x;
    p.x_pitch = x_pitch;
    p.rows = rows;
    p.layout_rows = layout_rows;
    p.row_tiles = fp8_row_tiles(layout_rows);
    p.cols = static_cast<int32_t>(cols);
    p.pitch = static_cast<int32_t>(fp8_pitch(cols));
    if (int rc = make_items(p.work, rows, cols, dtype == FMA_B200_F32 ? kAhead<float> : kAhead<__nv_bfloat16>)) return rc;
    p.values = static_cast<uint8_t*>(values);
    p.scales = static_cast<uint8_t*>(scales);
    if (rows == 0) return FMA_B200_OK;
    FMAB_REQUIRE(x && values && scales, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(x) && aligned16(values) && aligned16(scales), FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    return FMA_B200_OK;
}

}  // namespace fmab

extern "C" {

int64_t fma_b200_fp8_scale_bytes(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 0) return 0;
    return fmab::fp8_quads(cols) * fmab::fp8_row_tiles(rows) * fmab::FP8_TILE_BYTES;
}

int fma_b200_fp8_quantize_rows(const void* x, int64_t x_pitch, int32_t dtype, int64_t rows, int64_t cols,
                               const int32_t* rows_used, void* values, void* scales, void* stream) {
    using namespace fmab;
    QuantRows p;
    if (int rc = fill_quantize(p, x, x_pitch, dtype, rows, cols, rows, values, scales)) return rc;
    if (rows == 0) return FMA_B200_OK;
    p.rows_used = rows_used;
    return launch_quantize<TO_ROWS>(p, dtype, 0, static_cast<cudaStream_t>(stream));
}

int fma_b200_fp8_quantize_groups(const void* x, int64_t x_pitch, int32_t dtype, int64_t rows, int64_t cols,
                                 const int32_t* offsets, const int32_t* pad_offsets, int32_t E, int64_t layout_rows,
                                 void* values, void* scales, void* copy, void* stream) {
    using namespace fmab;
    QuantRows p;
    if (int rc = fill_quantize(p, x, x_pitch, dtype, rows, cols, layout_rows, values, scales)) return rc;
    FMAB_REQUIRE(E >= 1 && E <= 1024, FMA_B200_ERR_BAD_ARG, "E=%d not in [1,1024]", E);
    if (rows == 0) return FMA_B200_OK;
    FMAB_REQUIRE(offsets && pad_offsets, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(copy), FMA_B200_ERR_BAD_ARG, "copy is not 16-byte aligned");
    p.copy = copy;
    p.offsets = offsets;
    p.pad_offsets = pad_offsets;
    p.n_groups = E;
    return launch_quantize<TO_GROUPS>(p, dtype, E * 8LL, static_cast<cudaStream_t>(stream));
}

int fma_b200_fp8_quantize_scatter(const void* x, int32_t dtype, int64_t T, int64_t cols, int32_t k,
                                  const int32_t* row_of_slot, const int32_t* slot_of_row, const int32_t* pad_offsets,
                                  int32_t E, int64_t layout_rows, void* values, void* scales, void* stream) {
    using namespace fmab;
    QuantRows p;
    if (int rc = fill_quantize(p, x, cols, dtype, T, cols, layout_rows, values, scales)) return rc;
    FMAB_REQUIRE(E >= 1 && k >= 1, FMA_B200_ERR_BAD_ARG, "E=%d, k=%d", E, k);
    if (T == 0) return FMA_B200_OK;
    FMAB_REQUIRE(row_of_slot && slot_of_row && pad_offsets, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    p.row_of_slot = row_of_slot;
    p.slot_of_row = slot_of_row;
    p.pad_offsets = pad_offsets;
    p.n_groups = E;
    p.k = k;
    return launch_quantize<TO_SLOTS>(p, dtype, E * 64LL, static_cast<cudaStream_t>(stream));
}

int fma_b200_fp8_quantize_weight(const void* w, int32_t dtype, int32_t E, int32_t N, int32_t K, void* values,
                                 void* scales, void* stream) {
    using namespace fmab;
    if (int rc = check_rows_cols(dtype, N, K)) return rc;
    FMAB_REQUIRE(E >= 1 && E <= 1024, FMA_B200_ERR_BAD_ARG, "E=%d not in [1,1024]", E);
    FMAB_REQUIRE(N >= 8 && N % 8 == 0, FMA_B200_ERR_BAD_ARG, "N=%d must be a positive multiple of 8", N);
    FMAB_REQUIRE(static_cast<int64_t>(E) * N < (1LL << 31) - 1024 && static_cast<int64_t>(E) * K < (1LL << 31) - 1024,
                 FMA_B200_ERR_BAD_ARG, "E*N or E*K overflows");
    FMAB_REQUIRE(w && values && scales, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(w) && aligned16(values) && aligned16(scales), FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    QuantWeight p;
    p.w = w;
    p.values = static_cast<uint8_t*>(values);
    p.scales = static_cast<uint8_t*>(scales);
    p.E = E;
    p.N = N;
    p.K = K;
    p.pitch = static_cast<int32_t>(fp8_pitch(K));
    p.n_blocks = (N + FP8_BLOCK - 1) / FP8_BLOCK;
    p.k_blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    FMAB_REQUIRE(static_cast<int64_t>(p.n_blocks) * p.k_blocks < (1LL << 31), FMA_B200_ERR_BAD_ARG, "N*K overflows");
    const dim3 grid(static_cast<unsigned>(p.n_blocks * p.k_blocks), static_cast<unsigned>(E));
    int rc = FMA_B200_OK;
    dispatch_dtype(dtype, [&](auto tag) {
        rc = launch_kernel("fp8_quantize_weight", quantize_weight_kernel<decltype(tag)>, grid, 256, 0, 0,
                            static_cast<cudaStream_t>(stream), p);
    });
    return rc;
}

int fma_b200_fp8_dequantize(const void* values, const void* scales, int32_t batch, int64_t rows, int64_t cols,
                            const int32_t* rows_used, void* out, int32_t dtype, void* stream) {
    using namespace fmab;
    if (int rc = check_rows_cols(dtype, rows, cols)) return rc;
    FMAB_REQUIRE(batch >= 1 && batch * rows < (1LL << 31), FMA_B200_ERR_BAD_ARG, "batch=%d", batch);
    if (rows == 0) return FMA_B200_OK;
    FMAB_REQUIRE(values && scales && out, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    FMAB_REQUIRE(aligned16(values) && aligned16(scales) && aligned16(out), FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    Dequant p;
    p.values = static_cast<const uint8_t*>(values);
    p.scales = static_cast<const uint8_t*>(scales);
    p.out = out;
    p.rows_used = rows_used;
    p.rows = batch * rows;
    p.rows_per = static_cast<int32_t>(rows);
    p.tiles_per = static_cast<int32_t>(fp8_row_tiles(rows));
    p.row_tiles = static_cast<int64_t>(batch) * p.tiles_per;
    p.batch = batch;
    p.cols = static_cast<int32_t>(cols);
    p.pitch = static_cast<int32_t>(fp8_pitch(cols));
    if (int rc = make_items(p.work, p.rows, cols, 2)) return rc;
    int rc = FMA_B200_OK;
    dispatch_dtype(dtype, [&](auto tag) {
        rc = launch_kernel("fp8_dequantize", p.work.ahead == 1 ? dequantize_rows_kernel<decltype(tag), 1> : dequantize_rows_kernel<decltype(tag), 2>,
                           dim3(row_grid((p.work.units + 4LL * p.work.ahead - 1) / (4 * p.work.ahead))), kQThreads, 0, 0,
                            static_cast<cudaStream_t>(stream), p);
    });
    return rc;
}

int fma_b200_fp8_group_maps(const void* counts, int32_t index_bytes, int32_t E, int64_t rows, int64_t layout_rows,
                            int32_t* offsets, int32_t* pad_offsets, int32_t* group_rows, int32_t* tile_expert,
                            int32_t* tile_row, int32_t* tile_rows, void* stream) {
    using namespace fmab;
    FMAB_REQUIRE(known_index_bytes(index_bytes), FMA_B200_ERR_UNSUPPORTED, "index_bytes=%d", index_bytes);
    FMAB_REQUIRE(E >= 1 && E <= kMapThreads, FMA_B200_ERR_BAD_ARG, "E=%d not in [1,1024]", E);
    FMAB_REQUIRE(rows >= 0 && layout_rows % 256 == 0 && layout_rows < (1LL << 31) &&
                     layout_rows >= (rows + 255) / 256 * 256 + 256LL * (E < rows ? E : rows),
                 FMA_B200_ERR_BAD_ARG, "layout_rows=%lld is too small for %lld rows of %d experts", (long long)layout_rows,
                 (long long)rows, E);
    FMAB_REQUIRE(counts && offsets && pad_offsets && group_rows && tile_expert && tile_row && tile_rows, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    GroupMaps p;
    p.counts = counts;
    p.index_bytes = index_bytes;
    p.E = E;
    p.rows = rows;
    p.n_tiles = static_cast<int32_t>(layout_rows / 128);
    p.offsets = offsets;
    p.pad_offsets = pad_offsets;
    p.group_rows = group_rows;
    p.tile_expert = tile_expert;
    p.tile_row = tile_row;
    p.tile_rows = tile_rows;
    return launch_kernel("fp8_group_maps", group_maps_kernel, dim3(1), kMapThreads, 0, 0, static_cast<cudaStream_t>(stream), p);
}

int fma_b200_swiglu_fp8_forward(const void* gate, int64_t gate_pitch, const void* up, int64_t up_pitch, void* out,
                                int64_t out_pitch, int32_t dtype, int64_t rows, int64_t cols, const int32_t* rows_used,
                                void* gate8, void* gate_scales, void* up8, void* up_scales, void* out8, void* out_scales,
                                void* stream) {
    using namespace fmab;
    if (int rc = check_rows_cols(dtype, rows, cols)) return rc;
    if (int rc = check_pitch("gate", dtype, gate_pitch, cols)) return rc;
    if (int rc = check_pitch("up", dtype, up_pitch, cols)) return rc;
    if (out != nullptr)
        if (int rc = check_pitch("out", dtype, out_pitch, cols)) return rc;
    FMAB_REQUIRE((gate8 == nullptr) == (gate_scales == nullptr) && (up8 == nullptr) == (up_scales == nullptr) &&
                     (out8 == nullptr) == (out_scales == nullptr),
                 FMA_B200_ERR_BAD_ARG, "8-bit values and their scales come together");
    if (rows == 0) return FMA_B200_OK;
    FMAB_REQUIRE(gate && up, FMA_B200_ERR_BAD_ARG, "NULL pointer");
    const void* all[9] = {gate, up, out, gate8, gate_scales, up8, up_scales, out8, out_scales};
    for (const void* ptr : all) FMAB_REQUIRE(aligned16(ptr), FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    SwigluFp8 p;
    memset(&p, 0, sizeof(p));
    p.gate = gate;
    p.up = up;
    p.out = out;
    p.gate_pitch = gate_pitch;
    p.up_pitch = up_pitch;
    p.out_pitch = out_pitch;
    p.gate8 = static_cast<uint8_t*>(gate8);
    p.gate_scales = static_cast<uint8_t*>(gate_scales);
    p.up8 = static_cast<uint8_t*>(up8);
    p.up_scales = static_cast<uint8_t*>(up_scales);
    p.out8 = static_cast<uint8_t*>(out8);
    p.out_scales = static_cast<uint8_t*>(out_scales);
    p.rows_used = rows_used;
    p.rows = rows;
    p.row_tiles = fp8_row_tiles(rows);
    p.cols = static_cast<int32_t>(cols);
    p.pitch = static_cast<int32_t>(fp8_pitch(cols));
    p.blocks = static_cast<int32_t>((cols + FP8_BLOCK - 1) / FP8_BLOCK);
    int rc = FMA_B200_OK;
    dispatch_dtype(dtype, [&](auto tag) {
        rc = launch_kernel("swiglu_fp8_forward", swiglu_fp8_forward_kernel<decltype(tag)>, dim3(row_grid((rows * p.blocks + 3) / 4)), kQThreads, 0, 0,
                            static_cast<cudaStream_t>(stream), p);
    });
    return rc;
}

int fma_b200_swiglu_fp8_backward(const void* gate8, const void* gate_scales, const void* up8, const void* up_scales,
                                 const void* dy, int64_t dy_pitch, void* gate_grad, int64_t gate_grad_pitch,
                                 void* up_grad, int64_t up_grad_pitch, int32_t dtype, int64_t rows, int64_t cols,
                                 const int32_t* rows_used, void* grad8, void* grad_scales, void* stream) {
    using namespace fmab;
    if (int rc = check_rows_cols(dtype, rows, cols)) return rc;
    if (int rc = check_pitch("dy", dtype, dy_pitch, cols)) return rc;
    if (int rc = check_pitch("gate_grad", dtype, gate_grad_pitch, cols)) return rc;
    if (int rc = check_pitch("up_grad", dtype, up_grad_pitch, cols)) return rc;
    FMAB_REQUIRE((grad8 == nullptr) == (grad_scales == nullptr) && (grad8 == nullptr || cols % FP8_BLOCK == 0), FMA_B200_ERR_BAD_ARG,
                 "grad8 comes with its scales, and for widths that are multiples of 128 (cols=%lld)", (long long)cols);
    FMAB_REQUIRE(aligned16(grad8) && aligned16(grad_scales), FMA_B200_ERR_BAD_ARG, "pointers not 16-byte aligned");
    if (rows == 0) return FMA_B200_OK;
    const void* all[7] = {gate8, gate_scales, up8, up_scales, dy, gate_grad, up_grad};
    for (const void* ptr : all)
        FMAB_REQUIRE(ptr != nullptr && aligned16(ptr), FMA_B200_ERR_BAD_ARG, "pointer NULL or not 16-byte aligned");
    SwigluFp8 p;
    memset(&p, 0, sizeof(p));
    p.dy = dy;
    p.dy_pitch = dy_pitch;
    p.gate_grad = gate_grad;
    p.gate_grad_pitch = gate_grad_pitch;
    p.up_grad = up_grad;
    p.up_grad_pitch = up_grad_pitch;
    p.gate8 = static_cast<uint8_t*>(const_cast<void*>(gate8));
    p.gate_scales = static_cast<uint8_t*>(const_cast<void*>(gate_scales));
    p.up8 = static_cast<uint8_t*>(const_cast<void*>(up8));
    p.up_scales = static_cast<uint8_t*>(const_cast<void*>(up_scales));
    p.rows_used = rows_used;
    p.rows = rows;
    p.row_tiles = fp8_row_tiles(rows);
    p.cols = static_cast<int32_t>(cols);
    p.pitch = static_cast<int32_t>(fp8_pitch(cols));
    p.grad8 = static_cast<uint8_t*>(grad8);
    p.grad_scales = static_cast<uint8_t*>(grad_scales);
    p.blocks = static_cast<int32_t>((cols + FP8_BLOCK - 1) / FP8_BLOCK);
    int rc = FMA_B200_OK;
    dispatch_dtype(dtype, [&](auto tag) {
        rc = launch_kernel("swiglu_fp8_backward", swiglu_fp8_backward_kernel<decltype(tag)>, dim3(row_grid((rows * p.blocks + 3) / 4)), kQThreads, 0, 0,
                            static_cast<cudaStream_t>(stream), p);
    });
    return rc;
}

}  // extern "C"
