// The 8-bit cache's number format: e4m3 codes (four significant bits, exponents
// -6..8, steps of 2^-9 below, largest 448, 0x7f and 0xff NaN, no infinities) and
// a scale 2^e, e in -100..119, for each block of 16 tokens and KV head.
//
// With a power of two a code's value has at most four significant bits and an
// exponent of bf16's, so bf16 holds it exactly: reading back and the operands of
// the attention's products add no rounding.  A free scale would put a block's
// largest value at 448 exactly and gain up to a binary place at the small end
// only, since the codes' precision is relative.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"
#include "paged.hpp"

namespace tiattn {

// Two codes of a word (its upper half's or its lower half's) to packed bf16.
template <bool HI>
__device__ __forceinline__ uint32_t fp8x2_to_bf16(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
__device__ __forceinline__ uint4 fp8x8_to_bf16(uint2 w, float scale) {
    return make_uint4(fp8x2_to_bf16<false>(w.x, scale), fp8x2_to_bf16<true>(w.x, scale),
                      fp8x2_to_bf16<false>(w.y, scale), fp8x2_to_bf16<true>(w.y, scale));
}

// Nearest code to x / scale, halves to even; finite values past the largest code
// (they are past 448 * 2^119) take it, infinities are NaN as NaN is.
__device__ __forceinline__ float fp8_saturated(float x) {
    return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -448.0f, 448.0f) : x;
}
__device__ __forceinline__ uint32_t fp8x4_of(float a, float b, float c, float d, float inv_scale) {
    uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_saturated(a * inv_scale), fp8_saturated(b * inv_scale), 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(fp8_saturated(c * inv_scale), fp8_saturated(d * inv_scale), w, true);
}

__device__ __forceinline__ float fp8_scale(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// Exponent of the smallest scale with which most * 2^down is at most 448 = 1.75 * 2^8.
__device__ __forceinline__ int fp8_exponent_for(float most, int down) {
    const uint32_t b = __float_as_uint(most);
    return min(max((int)(b >> 23) - 127 - 8 + down + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), kFp8Low), kFp8High);
}
// Whether a block's scale is one that the writer makes; of memory that it has not
// written, any.
__device__ __forceinline__ bool fp8_scale_valid(float s) {
    const uint32_t b = __float_as_uint(s);
    return (b & 0x807fffffu) == 0 && b >= (uint32_t)(kFp8Low + 127) << 23 && b <= (uint32_t)(kFp8High + 127) << 23;
}

}  // namespace tiattn
