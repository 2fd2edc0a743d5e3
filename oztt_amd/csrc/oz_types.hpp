// The value types of the operators around a product (oz_type): loads and stores as FP32, vectors of the
// matrix instructions, activations.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "oz_hip.h"

namespace ozt {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

inline __host__ __device__ int size_of(int type) { return type == OZ_F32 ? 4 : 2; }
inline bool is_16bit(int type) { return type == OZ_BF16 || type == OZ_F16; }

// A 16-bit type by its oz_type number.
template <int TYPE>
struct Half;
template <>
struct Half<OZ_BF16> {
    typedef __bf16 t;
    typedef bf16x8 x8;
    typedef f32x4 sums;
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Half<OZ_F16> {
    typedef _Float16 t;
    typedef f16x8 x8;
    typedef f32x4 sums;
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// 8-bit integers: 16 of them where the others have 8 values, the sums exact.
struct Int8 {
    typedef i32x4 x8;
    typedef i32x4 sums;
    __device__ static i32x4 mfma(x8 a, x8 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// Value i of an array of the given type, as FP32, and back (rounded to nearest even).
__device__ __forceinline__ float load(const void* p, int type, long long i) {
    if (type == OZ_F32) return static_cast<const float*>(p)[i];
    if (type == OZ_BF16) return (float)static_cast<const __bf16*>(p)[i];
    return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store(void* p, int type, long long i, float x) {
    if (type == OZ_F32) static_cast<float*>(p)[i] = x;
    else if (type == OZ_BF16) static_cast<__bf16*>(p)[i] = (__bf16)x;
    else static_cast<_Float16*>(p)[i] = (_Float16)x;
}

// Sixteen bytes at any address that a value's type allows: the hardware's vector accesses of global memory take them.
template <class T>
__device__ __forceinline__ T get16(const void* p) {
    T x;
    __builtin_memcpy(&x, __builtin_assume_aligned(p, 2), 16);
    return x;
}
template <class T>
__device__ __forceinline__ void put16(void* p, T x) {
    __builtin_memcpy(__builtin_assume_aligned(p, 2), &x, 16);
}

// Eight values of a register's 16 bytes, of a 16-bit type.
__device__ __forceinline__ void widen8(u32x4 w, int type, float* x) {
    union {
        u32x4 w;
        bf16x8 b;
        f16x8 h;
    } u;
    u.w = w;
    if (type == OZ_BF16) {
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = (float)u.b[k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = (float)u.h[k];
    }
}

// Eight values from i on (type uniform over the wave: one branch).
__device__ __forceinline__ void load8(const void* p, int type, long long i, float* x) {
    if (type == OZ_F32) {
        const float* q = static_cast<const float*>(p) + i;
        const f32x4 a = get16<f32x4>(q), b = get16<f32x4>(q + 4);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = a[k], x[4 + k] = b[k];
    } else {
        widen8(get16<u32x4>(static_cast<const uint16_t*>(p) + i), type, x);
    }
}
__device__ __forceinline__ void store8(void* p, int type, long long i, const float* x) {
    if (type == OZ_F32) {
        float* q = static_cast<float*>(p) + i;
        put16(q, f32x4{x[0], x[1], x[2], x[3]});
        put16(q + 4, f32x4{x[4], x[5], x[6], x[7]});
    } else if (type == OZ_BF16) {
        bf16x8 a;
#pragma unroll
        for (int k = 0; k < 8; k++) a[k] = (__bf16)x[k];
        put16(static_cast<__bf16*>(p) + i, a);
    } else {
        f16x8 a;
#pragma unroll
        for (int k = 0; k < 8; k++) a[k] = (_Float16)x[k];
        put16(static_cast<_Float16*>(p) + i, a);
    }
}
// The first `count` of eight values.
__device__ __forceinline__ void load_some(const void* p, int type, long long i, int count, float* x) {
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = k < count ? load(p, type, i + k) : 0.0f;
}
__device__ __forceinline__ void store_some(void* p, int type, long long i, int count, const float* x) {
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (k < count) store(p, type, i + k, x[k]);
}

// Activations. GELU in its tanh form is z s with s = (1 + tanh u)/2 = 1 / (1 + exp(-2u)), u = sqrt(2/pi) (z + 0.044715 z^3), so
// GELU' = s + z (s - s^2) 2u'. SILU is z s with s = 1 / (1 + exp(-z)). The exponential (base 2, its factor folded into the
// constants) and the reciprocal are the hardware's, within a few units in the last place. z^2 is held below 10^4:
// beyond |z| = 100 s is 0 or 1 whatever the square, and s - s^2, which multiplies it, is 0. A z whose exponential overflows gives
// s = 0. Written with fused products: these 12 to 17 operations a value are what an epilogue and the gradients' pass
// over Z spend their vector time on (the pass over 8192 x 8192 values: 100 us with twice as many, 80, the copy rate).
constexpr float kGelu0 = 0.7978845608028654f, kGelu1 = 0.044715f, kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float logistic2(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x)); }  // 1 / (1 + 2^x)
__device__ __forceinline__ float gelu_s(float z, float zz) {
    return logistic2(z * __builtin_fmaf(zz, -2.0f * kLog2e * kGelu0 * kGelu1, -2.0f * kLog2e * kGelu0));
}
__device__ __forceinline__ float act(float z, int a) {
    switch (a) {
        case OZ_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;
        case OZ_ACT_GELU: return z * gelu_s(z, fminf(z * z, 1e4f));
        case OZ_ACT_SILU: return z * logistic2(-kLog2e * z);
        default: return z;
    }
}
// Eight values, one branch for all: a branch for each keeps the exponentials from overlapping.
__device__ __forceinline__ void act8(float* z, int a) {
    auto all = [&](auto A) {
#pragma unroll
        for (int k = 0; k < 8; k++) z[k] = act(z[k], decltype(A)::value);
    };
    if (a == OZ_ACT_GELU) all(std::integral_constant<int, OZ_ACT_GELU>{});
    else if (a == OZ_ACT_SILU) all(std::integral_constant<int, OZ_ACT_SILU>{});
    else if (a == OZ_ACT_RELU) all(std::integral_constant<int, OZ_ACT_RELU>{});
}
// dY act'(z). ReLU selects, so that what it masks goes no further whatever it is; a z that is not a number, which the activation
// hands on, is handed on here too. GELU's and SILU's slopes at infinity (an FP16 Z beyond its range) are their limits: the z that
// multiplies s - s^2 is held within 100, beyond which that difference is 0.
__device__ __forceinline__ float held(float z) { return __builtin_amdgcn_fmed3f(z, -100.0f, 100.0f); }
__device__ __forceinline__ float act_grad(float dy, float z, int a) {
    switch (a) {
        case OZ_ACT_RELU: return z > 0.0f ? dy : z != z ? z : 0.0f;
        case OZ_ACT_GELU: {
            const float y = held(z), zz = y * y, s = gelu_s(z, zz);
            return dy * __builtin_fmaf(y * __builtin_fmaf(-s, s, s), __builtin_fmaf(zz, 6.0f * kGelu0 * kGelu1, 2.0f * kGelu0), s);
        }
        case OZ_ACT_SILU: {
            const float s = logistic2(-kLog2e * z);
            return dy * __builtin_fmaf(held(z), __builtin_fmaf(-s, s, s), s);
        }
        default: return dy;
    }
}

}  // namespace ozt
