// float8 numbers (e4m3: four exponent bits, three of mantissa, largest value 448, no infinities) with one fp32 scale for a block of
// 128 values of a row (activations) or of 128 x 128 (weights): value = code * scale, scale = max(amax, 2^-100) / 448, code = x / scale
// rounded to the nearest e4m3 number, ties to even. Both divisions are correctly rounded, so that the same values give the same codes
// everywhere; quotients of short numbers lie exactly between two codes often enough for a rounded reciprocal to show.
// A NaN becomes the NaN code and leaves its block's scale alone; a block with an infinity gets the scale inf.
#pragma once
#include <cuda_fp8.h>
#include <math_constants.h>

#include "common.cuh"

namespace ttb {

constexpr int kF8Block = 128;
constexpr int kF8BlockBytes = kF8Block * kF8Block;

__host__ __device__ constexpr int64_t f8_blocks(int64_t n) { return (n + kF8Block - 1) / kF8Block; }
__host__ __device__ constexpr int64_t f8_rows_padded(int64_t rows) { return (rows + 7) / 8 * 8; }   // whole swizzle atoms
__host__ __device__ constexpr int64_t f8_scale_pitch(int64_t k) { return (f8_blocks(k) + 3) / 4 * 4; }

// Two fp32 numbers a register pair.
__device__ __forceinline__ uint64_t f8_two(float lo, float hi) { return ((uint64_t)__float_as_uint(hi) << 32) | __float_as_uint(lo); }
__device__ __forceinline__ uint64_t f8_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f8_mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// x / d, correctly rounded, from nx = -x and ny = -1 / d, the latter correctly rounded: Markstein's correction by the remainder (IBM J. Res. Dev. 34, 1990), twice.
// The first makes the product x (1 / d), off by up to 1.5 units in the last place, a neighbour of the quotient, the second the nearest. The remainders are exact
// while x and d are far from the smallest numbers; that of -x keeps the sign of a zero. (With __fdiv_rn 8192 x 8192 bfloat16 took 93 us by blocks, 81 by rows.)
__device__ __forceinline__ uint64_t f8_quotient2(uint64_t nx, uint64_t d, uint64_t ny) {
    const uint64_t q = f8_mul2(nx, ny), near = f8_fma2(f8_fma2(q, d, nx), ny, q);
    return f8_fma2(f8_fma2(near, d, nx), ny, near);
}
__device__ __forceinline__ float f8_scale(float amax) { return __fdiv_rn(fmaxf(amax, 0x1p-100f), 448.0f); }

// Codes of the values of one block: what their quotients by its scale have in common, and four of them, the first in the lowest byte.
struct F8Codes {
    uint64_t d, ny;
    bool small;   // (for the remainders; the quotients stay)
    __device__ __forceinline__ explicit F8Codes(float scale) : small(scale < 0x1p-60f) {
        if (small) scale *= 0x1p64f;
        const float inverse = __frcp_rn(scale), divisor = scale < CUDART_INF_F ? scale : 0.0f;   // scale inf: 0 for the finite values, else NaN
        d = f8_two(divisor, divisor);
        ny = f8_two(-inverse, -inverse);
    }
    __device__ __forceinline__ uint32_t two(float x0, float x1) const {
        uint64_t nx = f8_two(-x0, -x1);
        if (small) nx = f8_mul2(nx, f8_two(0x1p64f, 0x1p64f));
        const uint64_t q = f8_quotient2(nx, d, ny);
        return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float((uint32_t)q), __uint_as_float((uint32_t)(q >> 32))), __NV_SATFINITE, __NV_E4M3);
    }
    __device__ __forceinline__ uint32_t four(const float *x) const { return two(x[0], x[1]) | (two(x[2], x[3]) << 16); }
};
__device__ __forceinline__ uint2 f8_pack8(const float (&x)[8], float scale) {
    const F8Codes codes(scale);
    return make_uint2(codes.four(x), codes.four(x + 4));
}

// Quantised activations in scratch: for every block of 128 columns all rows, 128 bytes each, with the 16-byte chunks of a row
// exchanged as the MMA's 128-byte-swizzled K-major operand wants them (chunk ^= row % 8), so that any run of rows that starts at a
// multiple of eight is one contiguous copy. Byte of (row, block, column-in-block):
__device__ __forceinline__ int64_t f8_act_offset(int64_t rows_padded, int64_t block, int64_t row, int col) {
    return (block * rows_padded + row) * kF8Block + ((((col >> 4) ^ (int)(row & 7)) << 4) | (col & 15));
}

}  // namespace ttb
