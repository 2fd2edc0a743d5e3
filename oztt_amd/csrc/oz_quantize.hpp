// Rows as 8-bit integers: the definition, and the launch that oz_linear_i8 shares with oz_quantize_rows.
#pragma once
#include "oz_types.hpp"

struct oz_dev;

namespace ozq {

// A row's scale and its reciprocal from the bits of its largest |x| (as an unsigned number: an infinity and, above it, NaN are larger
// than all others). The least a makes the scale a normal number and keeps the reciprocal finite.
struct Scale {
    float scale, inverse;
};
__device__ __forceinline__ Scale scale_of(unsigned top) {
    if (top >= 0x7F800000u) return {__uint_as_float(0x7FC00000u), 0.0f};
    const float a = fmaxf(__uint_as_float(top), 127.0f * 0x1p-126f);
    return {a * (1.0f / 127.0f), 127.0f * (1.0f / a)};
}
__device__ __forceinline__ unsigned bits_of(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
// Four values as bytes; zeros in a row without a scale (inverse 0), whose x may be anything.
__device__ __forceinline__ unsigned pack4(const float* x, float inverse) {
    unsigned w = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) w |= ((unsigned)(int)__builtin_rintf(x[k] * inverse) & 255u) << (8 * k);
    return inverse > 0.0f ? w : 0u;
}

// Q and scale from X; columns K to `fill` of Q become zeros.
int launch_quantize(oz_dev* dev, int type, long long M, int K, const void* X, long long ldx, int8_t* Q, long long ldq, int fill, float* scale);

}  // namespace ozq
