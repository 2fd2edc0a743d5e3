// The value types of the operators around a product (oz_type): loads and stores as FP32, vectors of the
// matrix instructions, activations.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "oz_hip.h"

namespace ozt {

typedef float f32x4 __attribute__((ext_vector_type(4)));
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
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Half<OZ_F16> {
    typedef _Float16 t;
    typedef f16x8 x8;
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
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

// Activations. GELU in its tanh form is z / (1 + exp(-2u)), u = sqrt(2/pi) (z + 0.044715 z^3), since
// (1 + tanh u)/2 = 1/(1 + exp(-2u)); an overflow of z^3 or of the exponential gives the limits z and -0.
// The exponential and the reciprocal are the hardware's (a few units in the last place of FP32).
constexpr float kGelu0 = 0.7978845608028654f, kGelu1 = 0.044715f;
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }
__device__ __forceinline__ float act(float z, int a) {
    switch (a) {
        case OZ_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;
        case OZ_ACT_GELU: return z * sigmoid(2.0f * kGelu0 * z * (1.0f + kGelu1 * z * z));
        case OZ_ACT_SILU: return z * sigmoid(z);
        default: return z;
    }
}
// act'(z). Beyond |z| = 32 the curved ones' second term is below FP32's smallest value and 1 or 0 is left; left
// in, it would be 0 times infinity where z^2 overflows.
__device__ __forceinline__ float act_grad(float z, int a) {
    switch (a) {
        case OZ_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case OZ_ACT_GELU: {
            const float s = sigmoid(2.0f * kGelu0 * z * (1.0f + kGelu1 * z * z));
            const float t = z * (s * (1.0f - s)) * (2.0f * kGelu0 * (1.0f + 3.0f * kGelu1 * z * z));
            return fabsf(z) > 32.0f ? s : s + t;
        }
        case OZ_ACT_SILU: {
            const float s = sigmoid(z);
            return fabsf(z) > 128.0f ? s : s + z * (s * (1.0f - s));
        }
        default: return 1.0f;
    }
}

}  // namespace ozt
