// Rows to 8-bit integers with a scale each, shared by the quantizer (linear_i8.hip) and
// the RMS norm (rms_norm.hip):
//   scale = max|v| / 127, q = rint(v * (127 / max|v|))
// The product and the rounding are two roundings, as the formula says, never one
// fused: adding 1.5 * 2^23 rounds the product to an integer, ties to even, and
// leaves it in the sum's low byte.
#pragma once

#include "pxs_common.h"

namespace pxs {

constexpr uint32_t kQuantFinite = 0x7F800000u;   // infinity's bits
constexpr float kQuantLeast = 0x1p-100f;         // rows below count as zero: 127 / max stays finite
constexpr float kRoundMagic = 12582912.0f;       // 1.5 * 2^23

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The scale of a row with this largest magnitude, and what its values are multiplied with.
__device__ __forceinline__ void row_scale(uint32_t top_bits, float & scale, float & per) {
    const float top = __uint_as_float(top_bits);
    scale = 0.0f;
    per = 0.0f;
    if (top_bits >= kQuantFinite) {
        scale = __uint_as_float(0x7FC00000u);  // NaN: the row's products are NaN
    } else if (top >= kQuantLeast) {
        scale = top / 127.0f;
        per = 127.0f / top;
    }
}

// The bytes of eight values of a row whose factor is `per`.
__device__ __forceinline__ uint2 q8_bytes(const float (&v)[8], float per) {
#pragma clang fp contract(off)
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(v[i] * per + kRoundMagic);
    return make_uint2((b[0] & 255u) | (b[1] & 255u) << 8 | (b[2] & 255u) << 16 | b[3] << 24,
                      (b[4] & 255u) | (b[5] & 255u) << 8 | (b[6] & 255u) << 16 | b[7] << 24);
}

} // namespace pxs
