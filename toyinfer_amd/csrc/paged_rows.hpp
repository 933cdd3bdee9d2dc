// RMSNorm and rotate-half RoPE of a row held by D / 16 lanes, for the paged
// prologues: lane c has the eight pairs (8c + k, 8c + k + D/2).
#pragma once

#include <math.h>

#include "common.hpp"

namespace tiattn {

__device__ __forceinline__ void bf16x8_to_f32(uint4 x, float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[2 * k] = bf16_lo(word_of(x, k));
        f[2 * k + 1] = bf16_hi(word_of(x, k));
    }
}

// In fp32 throughout: the caller rounds the result, once.  (The unfused sequence
// rounds the norm's result as well.)  cs: (cos, sin) of the lane's pairs.
template <int D>
__device__ __forceinline__ void norm_rope_f32(uint4 xr, uint4 xi, uint4 wr, uint4 wi, const float4 (&cs)[4], float eps,
                                              float (&re)[8], float (&im)[8]) {
    float ss = 0.0f;
    bf16x8_to_f32(xr, re);
    bf16x8_to_f32(xi, im);
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fmaf(re[k], re[k], fmaf(im[k], im[k], ss));
    // The lanes of a row take the branches around this together.
    ss += dpp_f32<kDppXor1>(ss);
    ss += dpp_f32<kDppXor2>(ss);
    if constexpr (D == 128) ss += dpp_f32<kDppRowHalfMirror>(ss);
    const float inv = 1.0f / sqrtf(ss * (1.0f / D) + eps);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t gr = word_of(wr, k), gi = word_of(wi, k);
        const float r0 = re[2 * k] * inv * bf16_lo(gr), r1 = re[2 * k + 1] * inv * bf16_hi(gr);
        const float i0 = im[2 * k] * inv * bf16_lo(gi), i1 = im[2 * k + 1] * inv * bf16_hi(gi);
        re[2 * k] = cs[k].x * r0 - cs[k].y * i0;
        re[2 * k + 1] = cs[k].z * r1 - cs[k].w * i1;
        im[2 * k] = cs[k].x * i0 + cs[k].y * r0;
        im[2 * k + 1] = cs[k].z * i1 + cs[k].w * r1;
    }
}

__device__ __forceinline__ uint4 pack_bf16x8(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

}  // namespace tiattn
