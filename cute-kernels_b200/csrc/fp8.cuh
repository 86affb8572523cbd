// The 8-bit format of this library, shared by the kernels that write it (fp8_quant.cu) and the products that read it
// (gemm_fp8.cu).
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

}  // namespace fmab
