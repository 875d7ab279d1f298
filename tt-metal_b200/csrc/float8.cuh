// float8 numbers (e4m3: four exponent bits, three of mantissa, largest value 448, no infinities) with one fp32 scale for a block of
// 128 values of a row (activations) or of 128 x 128 (weights): value = code * scale, scale = max(amax, 2^-100) / 448, code = x / scale
// rounded to the nearest e4m3 number, ties to even. Both divisions are correctly rounded, so that the same values give the same codes
// everywhere; quotients of short numbers lie exactly between two codes often enough for a rounded reciprocal to show.
// A NaN becomes the NaN code and leaves its block's scale alone; a block with an infinity gets the scale inf.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace ttb {

constexpr int kF8Block = 128;
constexpr int kF8BlockBytes = kF8Block * kF8Block;

__host__ __device__ constexpr int64_t f8_blocks(int64_t n) { return (n + kF8Block - 1) / kF8Block; }
__host__ __device__ constexpr int64_t f8_rows_padded(int64_t rows) { return (rows + 7) / 8 * 8; }   // whole swizzle atoms
__host__ __device__ constexpr int64_t f8_scale_pitch(int64_t k) { return (f8_blocks(k) + 3) / 4 * 4; }

__device__ __forceinline__ float f8_scale(float amax) { return __fdiv_rn(fmaxf(amax, 0x1p-100f), 448.0f); }

// Eight values as codes, the first in the lowest byte.
__device__ __forceinline__ uint2 f8_pack8(const float (&v)[8], float scale) {
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        h[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[2 * j], scale), __fdiv_rn(v[2 * j + 1], scale)), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// The same with the scale's reciprocal, for values that are rounded sums themselves: a quotient that this moves by a unit in the last place was as uncertain
// before, and the divisions of a tile are some 20 KB of code.
__device__ __forceinline__ uint32_t f8_pack4_by(const float *v, float inverse) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0] * inverse, v[1] * inverse), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2] * inverse, v[3] * inverse), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Quantised activations in scratch: for every block of 128 columns all rows, 128 bytes each, with the 16-byte chunks of a row
// exchanged as the MMA's 128-byte-swizzled K-major operand wants them (chunk ^= row % 8), so that any run of rows that starts at a
// multiple of eight is one contiguous copy. Byte of (row, block, column-in-block):
__device__ __forceinline__ int64_t f8_act_offset(int64_t rows_padded, int64_t block, int64_t row, int col) {
    return (block * rows_padded + row) * kF8Block + ((((col >> 4) ^ (int)(row & 7)) << 4) | (col & 15));
}

}  // namespace ttb
