// What the 8-bit kernels share: the number format, the block scale and the tile layout of packed weights.
//
// e4m3 (OCP: 4 exponent bits, bias 7, 3 mantissa bits, largest 448, no infinities, NaN = 0x7f), one fp32 scale per block of 128
// consecutive inputs of a row: value = e4m3 number * scale.  For a block with largest magnitude a,
//     f = max(a, 2^-96),   scale = f / 448 (1 when a = 0),   q = e4m3(y * (448 / f)), round to nearest even.
// 448 is the largest e4m3 number, so the block's largest element uses the whole range and nothing saturates (448 / f is rounded
// to fp32, the product lies at most 2 ulp above 448 and rounds to it).  2^-96 keeps 448 / f finite.  An infinity or a NaN
// in a block makes scale inf or NaN and at least that element NaN: every value of the block, hence every output of the row, is
// NaN, and no other row is touched.
#pragma once

#include "ha_common.h"

#define HA_FP8_MAX 448.0f
#define HA_FP8_FLOOR 0x1p-96f

#define HA_FP8_MAX_K (2147483647 - HA_FP8_BLOCK)  // a row's positions, rounded up to whole blocks, are 32-bit

// a launch holds fewer than 2^32 threads
static inline bool ha_fits_launch(int64_t groups, int threads) { return groups <= 0xFFFFFFFFLL / threads; }

static inline int ha_fp8_blocks(int K) { return K / HA_FP8_BLOCK + (K % HA_FP8_BLOCK != 0); }

#ifdef __HIPCC__

// four floats -> four e4m3 bytes, the first in the lowest byte
__device__ __forceinline__ uint32_t ha_fp8x4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// |y| as bits: ordered as unsigned numbers, finite < infinity < NaN, so a maximum of bits carries a NaN where fmaxf drops it
__device__ __forceinline__ uint32_t ha_abs_bits(float y) { return __float_as_uint(y) & 0x7FFFFFFFu; }

struct HaFp8Scale {
    float scale, inv;
};
// The numbers of the block are y = p * common; top_bits is the largest |p|.  inv turns a p (not a y) into its e4m3 number: a factor
// that all share falls out of p / |p|max, and its rounding with it.
__device__ __forceinline__ HaFp8Scale ha_fp8_scale(uint32_t top_bits, float common = 1.0f) {
    const float a = __uint_as_float(top_bits), f = a * common;
    HaFp8Scale r;
    if (f < HA_FP8_FLOOR) {  // a NaN compares false
        r.inv = HA_FP8_MAX / HA_FP8_FLOOR * common;
        r.scale = top_bits == 0u ? 1.0f : HA_FP8_FLOOR / HA_FP8_MAX;
    } else {
        r.inv = HA_FP8_MAX / a;
        r.scale = f / HA_FP8_MAX;
    }
    return r;
}

// g / (1 + exp(-g)) to a relative 2^-21 while exp(-g) is finite (g above -88.72): exp(-g) as 2^t with the rounding error of t put back
// (2 ulp; 2^t alone loses |t| ulp), the reciprocal to 1 ulp.  A quarter of the instructions of expf and an IEEE division, which bound
// the SwiGLU of a prompt (4096 x 14336: 79 us, the memory's time is 60).  Further out exp(-g) overflows to infinity and the quotient is 0,
// or it vanishes and the quotient is g; the correction is left out there (t itself may have overflowed, and its error is no number
// then).  Numerator and denominator are both taken at an eighth (powers of two: exact but for gates below 2^-123): the reciprocal of a
// denominator above 2^126 would be subnormal, which the instruction does not give.
__device__ __forceinline__ float ha_silu(float g) {
    const float h = g * 0.125f, t = h * -11.5415603f;
    const float lost = fmaf(h, -11.5415603f, -t) + h * -1.54077039e-7f;  // 8 log2(e) is 11.5415603 + 1.5408e-7
    float e = __builtin_amdgcn_exp2f(t);
    if (fabsf(t) < 128.0f) e = fmaf(e, lost * 0.693147181f, e);
    return h * __builtin_amdgcn_rcpf((1.0f + e) * 0.125f);
}

#endif  // __HIPCC__
