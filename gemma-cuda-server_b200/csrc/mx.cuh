// mx.cuh -- MXFP4 (OCP microscaling) numerics shared by the quantisers and the block norm.
//
// A block is 32 consecutive elements along K.  With A = max |x| of the block:
//   e     = max(floor(log2 A) - 2, -127)     (2 = the exponent of the largest e2m1 value, 6 = 1.5 * 2^2)
//   byte  = e + 127                          (e8m0; a block of zeros has byte 0)
//   code  = nearest e2m1 to x / 2^e, ties to even, saturated at 6; the sign of x is kept, also on zero codes
// A block that holds a NaN or a magnitude of 2^128 or more (every infinity) has byte 0xFF (the e8m0 NaN) and codes 0.
// floor(log2 A) is A's exponent field, so for fp32 the byte is max(field, 2) - 2 and x / 2^e is one exact product.
//
// Where x itself is a rounded fp32 result (norm, gate), the codes stored are those of its float64 value: the fp32
// estimate carries a bound d on its error, the block is encoded from x - d and x + d, and where both agree no
// rounding boundary lies between them.  Blocks that disagree are redone in float64 (mx_code64).
#pragma once

#include "common.cuh"

namespace nvfp4b {

// Scale byte of a block from max |x| as fp32 bits (sign cleared).
__device__ __forceinline__ uint32_t mx_byte(uint32_t amax_bits) {
    const uint32_t f = amax_bits >> 23;
    return f == 255u ? 255u : (f < 2u ? 0u : f - 2u);
}

// 1 / 2^e of a scale byte up to 252 (the largest that a finite fp32 block has): a normal power of two.
__device__ __forceinline__ float mx_inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// 2^e of any scale byte: 2^-127 (subnormal) for 0, NaN for 0xFF.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 0x7FFFFFFFu : byte << 23));
}

// Offset of the scale byte of (row m, block b) in the 128x4-tile layout with `tile_cols` tiles along K.
__device__ __forceinline__ size_t mx_scale_offset(int m, int b, int tile_cols) {
    return ((size_t)(m >> 7) * tile_cols + (b >> 2)) * 512 + (m & 31) * 16 + ((m & 127) >> 5) * 4 + (b & 3);
}

// Scale byte of a float64 block maximum.
__device__ __forceinline__ uint32_t mx_byte64(double amax) {
    if (!(amax < 3.402823669209384634634e38)) return 255u;       // 2^128 and more, infinities, NaN
    const int f = (int)(__double_as_longlong(amax) >> 52);       // biased by 1023
    const int byte = f - 1023 - 2 + 127;
    return byte < 0 ? 0u : (uint32_t)byte;
}

// Code of one float64 element under a scale byte below 255.
__device__ __forceinline__ uint32_t mx_code64(double x, uint32_t byte) {
    const double y = fabs(x) * pow2d(127 - (int)byte);
    const uint32_t c = (uint32_t)(y > 0.25) + (uint32_t)(y >= 0.75) + (uint32_t)(y > 1.25) + (uint32_t)(y >= 1.75) +
                       (uint32_t)(y > 2.5) + (uint32_t)(y >= 3.5) + (uint32_t)(y > 5.0);
    return c | (__double_as_longlong(x) < 0 ? 8u : 0u);
}

}  // namespace nvfp4b
