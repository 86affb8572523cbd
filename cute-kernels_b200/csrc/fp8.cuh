// The 8-bit format of this library, shared by the kernels that write it (fp8_quant.cu) and the products that read it
// (gemm_fp8.cu, fp8_few.cu).
//
// A tensor [rows, cols] is held as e4m3 values [rows, pitch] (pitch = cols rounded up to 16, the extra columns zero)
// and one power-of-two scale per block of 128 columns of a row, or of 128 x 128 (weights).  With amax the largest
// finite magnitude of the block, the scale is 2^e with e the smallest integer such that amax <= 448 * 2^e (0 for a
// block of zeros, never outside [-127, 127]); the value is e4m3(x * 2^-e).  Infinities and NaN become e4m3's NaN and
// leave their neighbours' scale alone.
//
// Why powers of two: x * 2^-e is exact, so the only rounding is the one to e4m3; a dequantised value is exact in
// bfloat16 as well (4 significant bits); and the tensor cores apply such scales themselves (the ue8m0 scale operands
// of tcgen05.mma block scaling), so the accumulator never has to leave tensor memory between blocks.
//
// Scales are one byte, e + 127, in the order in which the tensor cores take them: for every group of four k-blocks
// (512 columns) and every 128 rows a tile of 512 bytes, the four bytes of a row next to each other at
// (row % 32) * 16 + (row / 32 % 4) * 4.  A tile is one 32-lane x 16-byte copy into tensor memory.
#pragma once

#include <cuda_fp8.h>
#include <string.h>

#include "common.cuh"

namespace fmab {

constexpr int FP8_BLOCK = 128;             // columns per scale
constexpr int FP8_QUAD = 4 * FP8_BLOCK;    // columns per scale tile
constexpr int FP8_TILE_ROWS = 128;         // rows per scale tile
constexpr int FP8_TILE_BYTES = 512;
constexpr int FP8_SCALE_ONE = 127;

inline int64_t fp8_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }
inline int64_t fp8_quads(int64_t cols) { return (cols + FP8_QUAD - 1) / FP8_QUAD; }
inline int64_t fp8_row_tiles(int64_t rows) { return (rows + FP8_TILE_ROWS - 1) / FP8_TILE_ROWS; }

// Byte offset of the four scales of (row, k-blocks 4q..4q+3); row_tiles = scale tiles per quad.
__host__ __device__ __forceinline__ int64_t fp8_scale_word(int64_t row, int64_t q, int64_t row_tiles) {
    return (q * row_tiles + (row >> 7)) * FP8_TILE_BYTES + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// Scale byte of a block from the bits of its amax (finite, not negative).  The exponent field grows by one where the
// fraction is above 1.75 = 448 / 2^8: adding 0x1fffff carries exactly then.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bits) {
    const int b = static_cast<int>((amax_bits + 0x1fffffu) >> 23) - 8;
    return amax_bits == 0 ? FP8_SCALE_ONE : static_cast<uint32_t>(b > 0 ? b : 0);
}
__device__ __forceinline__ float fp8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }  // 2^-e
__device__ __forceinline__ float fp8_factor(uint32_t byte) {                                                 // 2^e
    return __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
}
// |x| as ordered bits; infinities and NaN count as zero.
__device__ __forceinline__ uint32_t fp8_magnitude(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
// Four values, scaled, as e4m3 bytes (first in the lowest byte).  y * 0 + y is y, except that an infinity becomes NaN
// (the conversion would saturate it to 448).
__device__ __forceinline__ uint32_t fp8_pack4(const float* x, float inverse) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = x[i] * inverse;
        y[i] = fmaf(y[i], 0.f, y[i]);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ void fp8_unpack4(uint32_t w, float factor, float* x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * i)), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        x[2 * i] = f.x * factor;
        x[2 * i + 1] = f.y * factor;
    }
}

// These kernels are launched without programmatic stream serialization, although that takes 1 to 2 us off each launch of
// a chain (one row of 14336 x 4096 14.7 instead of 16.6 us): a chain of seven of them, forward and backward of a large
// linear map, stood still for good under a profiler with it, and not without.
template <typename... Params, typename... Args>
static int launch_kernel(const char* what, void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, unsigned cluster,
                          cudaStream_t s, Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute cluster_size;
    cluster_size.id = cudaLaunchAttributeClusterDimension;
    cluster_size.val.clusterDim.x = cluster;
    cluster_size.val.clusterDim.y = 1;
    cluster_size.val.clusterDim.z = 1;
    config.attrs = &cluster_size;
    config.numAttrs = cluster > 0 ? 1 : 0;  // 0: as the kernel itself says
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(FMA_B200_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
    }
    return FMA_B200_OK;
}

// Rows of expert e, at most `rows`; none for a negative count.  index_bytes: 8 and 4 for signed integers, -4 for unsigned ones.
__device__ __forceinline__ int32_t fp8_count(const void* counts, int32_t index_bytes, int e, int64_t rows) {
    const long long c = index_bytes == 8   ? static_cast<const long long*>(counts)[e]
                        : index_bytes == 4 ? static_cast<long long>(static_cast<const int32_t*>(counts)[e])
                                           : static_cast<long long>(static_cast<const uint32_t*>(counts)[e]);
    return static_cast<int32_t>(c < 0 ? 0 : (c > rows ? rows : c));
}
inline bool known_index_bytes(int32_t n) { return n == 4 || n == 8 || n == -4; }

// Row access: a warp takes 512 columns of a row (one scale word); 8 lanes share a block of 128 columns, so the block
// maximum is three shuffles and every load instruction of the 8 lanes covers 128 contiguous bytes.
template <typename T>
struct LaneBlock {                                    // a lane's 16 of the block's 128 columns
    static constexpr int V = Elem<T>::kPerVec;        // columns per 128-bit access
    static constexpr int N = 16 / V;                  // accesses
    // column (inside the block) of access j for the lane's place s = lane % 8
    __device__ static __forceinline__ int column(int s, int j) { return j * 8 * V + s * V; }
};

__device__ __forceinline__ uint32_t max_over_8_lanes(uint32_t v) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The lane's 16 values to columns [col0, cols).
template <typename T>
__device__ __forceinline__ void store_lane_block(T* row, int col0, int cols, int s, const float* x) {
    using B = LaneBlock<T>;
#pragma unroll
    for (int j = 0; j < B::N; ++j) {
        const int c = col0 + B::column(s, j);
        if (c < cols) st_global_16(row + c, Elem<T>::pack(x + j * B::V));
    }
}
// The lane's 16 bytes to / from the value row (pitch columns, of which those from `cols` on are zero).
template <typename T>
__device__ __forceinline__ void store_lane_bytes(uint8_t* row, int col0, int pitch, int s, const uint32_t* w) {
    using B = LaneBlock<T>;
#pragma unroll
    for (int j = 0; j < B::N; ++j) {
        const int c = col0 + B::column(s, j);
        if (c >= pitch) continue;
        if (B::V == 8)
            *reinterpret_cast<uint2*>(row + c) = make_uint2(w[2 * j], w[2 * j + 1]);
        else
            *reinterpret_cast<uint32_t*>(row + c) = w[j];
    }
}
template <typename T>
__device__ __forceinline__ void load_lane_bytes(const uint8_t* row, int col0, int pitch, int s, uint32_t* w) {
    using B = LaneBlock<T>;
#pragma unroll
    for (int j = 0; j < B::N; ++j) {
        const int c = col0 + B::column(s, j);
        if (B::V == 8) {
            const uint2 v = c < pitch ? *reinterpret_cast<const uint2*>(row + c) : make_uint2(0, 0);
            w[2 * j] = v.x;
            w[2 * j + 1] = v.y;
        } else {
            w[j] = c < pitch ? *reinterpret_cast<const uint32_t*>(row + c) : 0u;
        }
    }
}
// The 16-bit types' magnitudes are compared two at a time as integers, and only a block with an infinity or NaN takes
// the general way (150 instructions per 16 values, against about 75).
template <typename T>
struct Magnitude16 {
    static constexpr bool kPacked = false;
};
template <>
struct Magnitude16<__nv_bfloat16> {
    static constexpr bool kPacked = true;
    static constexpr uint32_t kInf = 0x7f80;
    __device__ static __forceinline__ uint32_t float_bits(uint32_t m) { return m << 16; }
};
template <>
struct Magnitude16<__half> {
    static constexpr bool kPacked = true;
    static constexpr uint32_t kInf = 0x7c00;
    __device__ static __forceinline__ uint32_t float_bits(uint32_t m) {
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
    }
};
__device__ __forceinline__ uint32_t max_magnitudes16(uint32_t m, const uint4& v) {
    m = __vmaxu2(m, v.x & 0x7fff7fffu);
    m = __vmaxu2(m, v.y & 0x7fff7fffu);
    m = __vmaxu2(m, v.z & 0x7fff7fffu);
    return __vmaxu2(m, v.w & 0x7fff7fffu);
}
// Four finite values, scaled, as e4m3 bytes.
__device__ __forceinline__ uint32_t fp8_pack4_finite(const float* x, float inverse) {
    const float2 by = make_float2(inverse, inverse);
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(__fmul2_rn(make_float2(x[0], x[1]), by), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(__fmul2_rn(make_float2(x[2], x[3]), by), __NV_SATFINITE, __NV_E4M3);
    return __byte_perm(lo, hi, 0x5410);
}
// The warp's scale word (all lanes) from each lane's scale byte.
__device__ __forceinline__ uint32_t scale_word_of(uint32_t byte) {
    uint32_t word = byte << (8 * ((threadIdx.x & 31) >> 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    return word | __shfl_xor_sync(0xffffffffu, word, 16);
}
// The 16 packed values of a lane; returns the scale byte of its 8 lanes' block.
__device__ __forceinline__ uint32_t quantize_lane_block(const float* x, uint32_t* w) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, fp8_magnitude(x[i]));
    const uint32_t byte = fp8_scale_byte(max_over_8_lanes(m));
    const float inverse = fp8_inverse(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = fp8_pack4(x + 4 * i, inverse);
    return byte;
}
// The same from the lane's values as they were loaded.
template <typename T>
__device__ __forceinline__ uint32_t quantize_lane_raw(const uint4* raw, uint32_t* w) {
    float x[16];
#pragma unroll
    for (int j = 0; j < LaneBlock<T>::N; ++j) Elem<T>::unpack(raw[j], x + j * LaneBlock<T>::V);
    if constexpr (Magnitude16<T>::kPacked) {
        const uint32_t pair = max_magnitudes16(max_magnitudes16(0, raw[0]), raw[1]);
        const uint32_t m = max_over_8_lanes(max(pair & 0xffffu, pair >> 16));
        if (!__any_sync(0xffffffffu, m >= Magnitude16<T>::kInf)) {
            const uint32_t byte = fp8_scale_byte(Magnitude16<T>::float_bits(m));
            const float inverse = fp8_inverse(byte);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = fp8_pack4_finite(x + 4 * i, inverse);
            return byte;
        }
    }
    return quantize_lane_block(x, w);
}

}  // namespace fmab
