// The 8-bit form with one fp32 scale per block of 128: value = scale * e4m3 code.  A block is 128 neighbours of one row
// (activations) or 128 x 128 (weights).  The quantizers here choose the smallest power of two that brings the block's largest
// magnitude to 448 or less, so scaling is exact and only the rounding to e4m3 (half a step, 2^-4) loses anything; consumers
// take any fp32 scale.
#pragma once

#include "mxfp8.cuh"

namespace mok {

constexpr int kScaleBlock = 128;

// Largest magnitude of a block as the bits of an fp32 value: integer order is that of magnitudes, infinities come above the
// finite values and NaNs above those, where fmaxf would drop them.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Scale of a block and its reciprocal, both exact.  448 = 1.75 * 2^8: 2^k with k = exponent - 8, one more where the mantissa is
// above 1.75; at least 2^-126 (blocks of zeros too).  A block that holds an infinity or a NaN gets scale and reciprocal NaN, so
// that every value read from it is NaN.
__device__ __forceinline__ float block_scale(uint32_t amax_bits, float& reciprocal) {
    const int biased = static_cast<int>(amax_bits >> 23);
    if (biased == 255) {
        reciprocal = __uint_as_float(0x7FC00000u);
        return reciprocal;
    }
    const int k = max(biased - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0), 1);   // biased exponent of the scale
    reciprocal = __uint_as_float(static_cast<uint32_t>(254 - k) << 23);
    return __uint_as_float(static_cast<uint32_t>(k) << 23);
}

}  // namespace mok
