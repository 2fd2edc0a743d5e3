// AdamW over many tensors in one launch, states in 32 bits or in 8 (include/oz_hip.h, oz_adamw_step).
//
// Every value is independent but for the scale that the 64 values of a block share in 8-bit states, so the
// step is one pass over memory: 28 bytes a value with 32-bit states (BF16 param and gradient, FP32 master),
// 16 with 8-bit ones; 1e8 values take 522 us (5.4 TB/s) and 320 us (5.0 TB/s; the VALU counts too: 360 to 410 us in long rows of passes, whose clock
// falls to 1.8 GHz). A workgroup takes one chunk of one tensor, found in the plan's list; a lane takes 8 values
// in a row (one or two 16-byte accesses of every array, 8 bytes of 8-bit states), so 8 neighbouring lanes hold a
// block and its maximum is three exchanges away. The file is compiled without contraction: the order of
// operations is the header's, each rounded once.
#include <cmath>
#include <type_traits>
#include <vector>

#include "oz_internal.hpp"
#include "oz_types.hpp"

namespace {

using namespace ozt;

constexpr int V = 8, THREADS = 256;  // values of a lane, lanes
static_assert(OZ_ADAMW_BLOCK == 8 * V, "a block is 8 lanes' values");

// Values of a chunk: one round of a workgroup's threads, 8 of lists of which those would be too many workgroups. Rounds in turn
// by one workgroup are slower, as the next one's loads wait for this one's stores: 1e8 values with 32-bit states take 523 us in
// chunks of one round, 537 of two, 549 of four, 590 of sixteen. Loads and stores past the caches gain nothing (521 us; loads 577).
int chunk_of(long long values) { return values >> 33 ? 8 * V * THREADS : V * THREADS; }

// The plan's memory: one Entry a tensor, then for each chunk its tensor (uint32), its place in it follows
// from the tensor's first chunk.
struct Entry {
    oz_adamw_tensor t;
    long long first_chunk;
    uint32_t first_block;  // blocks of the tensors before, modulo 2^32
    int chunk;             // values of a chunk
};

struct Step {
    float b1, a1, b2, a2, root, eps, rate, lr;  // a = 1 - b; root = 1 / sqrt(1 - b2^t); rate = lr / (1 - b1^t)
    uint32_t seed;
    const float* grad_scale;
};

// Value `code` of an e4m3 byte, exact: the hardware's conversion of four bytes at once.
__device__ __forceinline__ void from_e4m3(uint32_t w, float* x) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}

__device__ __forceinline__ float power(int e) { return __uint_as_float(e < -126 ? 0x00400000u : (uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }  // x >= 0

// The header's hash: two rounds of shift, xor and odd product, a bijection of 32 bits, its shifts and factors those that C. Wellons'
// search for such hashes of low bias published in 2018.
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7FEB352Du;
    x ^= x >> 15;
    x *= 0x846CA68Bu;
    return x ^ (x >> 16);
}

// The scale exponent of the block whose values 8 lanes hold: the least e >= -127 with max |x| <= 448 * 2^e.
__device__ __forceinline__ int block_exponent(const float* x) {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < V; k++) {
        const float a = fabsf(x[k]);
        top = fmaxf(top, a < INFINITY ? a : 0.0f);
    }
#pragma unroll
    for (int s = 1; s < 8; s *= 2) top = fmaxf(top, __shfl_xor(top, s, 8));
    return max(exponent(top) - 8 + ((__float_as_uint(top) & 0x7FFFFF) > 0x600000), -127);  // 448 = 1.75 * 2^8
}

// e4m3 byte of x / 2^e, rounded up where the distance from the lower neighbour (in steps of the
// neighbours' distance) and u together reach 1. With ey the exponent of the value's binade, at least -6 (below it
// the steps stay 2^-9), the value is t 2^(ey - 3), t < 16, and the byte 8 (ey + 6) + floor(t + u), carries
// into the exponent included.
__device__ __forceinline__ uint32_t to_e4m3(float x, int e, float u, bool root) {
    const float a = fabsf(x), y = a * power(-e);
    const int ey = max(exponent(y), -6);
    int code = 8 * (ey + 6) + (int)floorf(y * power(3 - ey) + u);
    if (root && a > 0.0f) code = max(code, 1);
    if (!(a < INFINITY)) code = 127;
    return (uint32_t)code | (x < 0.0f ? 128u : 0u);
}

__device__ __forceinline__ void from_8bit(const uint8_t* p, uint8_t scale, float* x) {
    u32x2 w;
    __builtin_memcpy(&w, p, 8);
    from_e4m3(w[0], x);
    from_e4m3(w[1], x + 4);
    const float s = power((int)scale - 127);
#pragma unroll
    for (int k = 0; k < V; k++) x[k] *= s;
}

// The first `count` of 8 values from i on.
__device__ __forceinline__ void put(void* p, int type, long long i, int count, bool whole, const float* x) {
    if (whole) store8(p, type, i, x);
    else store_some(p, type, i, count, x);
}

// One chunk of a tensor whose types are known here: with a branch on them at every access the loads of a round would each be
// waited for where the branches meet.
template <int BITS, int PARAM, int GRAD, bool MASTER>
__device__ __forceinline__ void step_chunk(const Entry& E, const Step& o) {
    const oz_adamw_tensor& t = E.t;
    const long long n = t.n, begin = (blockIdx.x - E.first_chunk) * E.chunk;
    const float gs = o.grad_scale ? *o.grad_scale : 1.0f;
    const float keep = 1.0f - o.lr * t.weight_decay;
    const long long end = begin + E.chunk < n ? begin + E.chunk : n;
    // whole blocks of lanes go through, so that the exchanges of a block's lanes always find them
    for (long long i = begin + V * (long long)threadIdx.x; i - V * (threadIdx.x & 7) < end; i += V * THREADS) {
        const int count = (int)(end - i < V ? (end - i > 0 ? end - i : 0) : V);
        const bool whole = count == V;
        float g[V], p[V], m[V], v[V], r[V];
        const void* from = MASTER ? t.master : t.param;
        constexpr int FROM = MASTER ? OZ_F32 : PARAM;
        if (whole) {
            load8(t.grad, GRAD, i, g);
            load8(from, FROM, i, p);
            if constexpr (BITS == 32) {
                load8(t.m, OZ_F32, i, m);
                load8(t.v, OZ_F32, i, v);
            } else {
                from_8bit(static_cast<uint8_t*>(t.m) + i, t.m_scale[i / OZ_ADAMW_BLOCK], m);
                from_8bit(static_cast<uint8_t*>(t.v) + i, t.v_scale[i / OZ_ADAMW_BLOCK], r);
            }
        } else {
            load_some(t.grad, GRAD, i, count, g);
            load_some(from, FROM, i, count, p);
            if constexpr (BITS == 32) {
                load_some(t.m, OZ_F32, i, count, m);
                load_some(t.v, OZ_F32, i, count, v);
            } else {
                const uint8_t *pm = static_cast<uint8_t*>(t.m) + i, *pv = static_cast<uint8_t*>(t.v) + i;
                const int ms = count ? t.m_scale[i / OZ_ADAMW_BLOCK] : 0, vs = count ? t.v_scale[i / OZ_ADAMW_BLOCK] : 0;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    float x[4];
                    from_e4m3(k < count ? pm[k] | (uint32_t)pv[k] << 8 : 0u, x);
                    m[k] = x[0] * power(ms - 127);
                    r[k] = x[1] * power(vs - 127);
                }
            }
        }
        if constexpr (BITS == 8) {
#pragma unroll
            for (int k = 0; k < V; k++) v[k] = r[k] * r[k];
        }
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float x = g[k] * gs;
            m[k] = o.b1 * m[k] + o.a1 * x;
            v[k] = o.b2 * v[k] + (o.a2 * x) * x;
            r[k] = sqrtf(v[k]);
            p[k] = p[k] * keep - (m[k] / (r[k] * o.root + o.eps)) * o.rate;
        }
        put(t.param, PARAM, i, count, whole, p);
        if constexpr (MASTER) put(t.master, OZ_F32, i, count, whole, p);
        if constexpr (BITS == 32) {
            put(t.m, OZ_F32, i, count, whole, m);
            put(t.v, OZ_F32, i, count, whole, v);
        } else {
            const int em = block_exponent(m), ev = block_exponent(r);
            uint32_t cm[2] = {0, 0}, cv[2] = {0, 0};
            const uint32_t place = E.first_block * OZ_ADAMW_BLOCK + (uint32_t)i;
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t h = mix((place + k) ^ o.seed);
                cm[k / 4] |= to_e4m3(m[k], em, ((float)(h & 0xFFFF) + 0.5f) * 0x1p-16f, false) << (8 * (k % 4));
                cv[k / 4] |= to_e4m3(r[k], ev, ((float)(h >> 16) + 0.5f) * 0x1p-16f, true) << (8 * (k % 4));
            }
            uint8_t *pm = static_cast<uint8_t*>(t.m) + i, *pv = static_cast<uint8_t*>(t.v) + i;
            if (whole) {
                __builtin_memcpy(pm, cm, 8);
                __builtin_memcpy(pv, cv, 8);
            } else {
#pragma unroll
                for (int k = 0; k < V; k++)
                    if (k < count) {
                        pm[k] = (uint8_t)(cm[k / 4] >> (8 * (k % 4)));
                        pv[k] = (uint8_t)(cv[k / 4] >> (8 * (k % 4)));
                    }
            }
            if (count && !(threadIdx.x & 7)) {
                t.m_scale[i / OZ_ADAMW_BLOCK] = (uint8_t)(em + 127);
                t.v_scale[i / OZ_ADAMW_BLOCK] = (uint8_t)(ev + 127);
            }
        }
    }
}

template <int BITS>
__global__ void __launch_bounds__(THREADS) adamw_kernel(const Entry* __restrict__ entries, const uint32_t* __restrict__ owner, Step o) {
    const Entry& E = entries[owner[blockIdx.x]];
    const auto by_grad = [&](auto P, auto M) {
        constexpr int p = decltype(P)::value;
        constexpr bool m = decltype(M)::value;
        if (E.t.grad_type == OZ_F32) step_chunk<BITS, p, OZ_F32, m>(E, o);
        else if (E.t.grad_type == OZ_BF16) step_chunk<BITS, p, OZ_BF16, m>(E, o);
        else step_chunk<BITS, p, OZ_F16, m>(E, o);
    };
    const auto by_param = [&](auto M) {
        if (E.t.param_type == OZ_BF16) by_grad(std::integral_constant<int, OZ_BF16>{}, M);
        else by_grad(std::integral_constant<int, OZ_F16>{}, M);
    };
    if (E.t.param_type == OZ_F32) by_grad(std::integral_constant<int, OZ_F32>{}, std::false_type{});
    else if (E.t.master) by_param(std::true_type{});
    else by_param(std::false_type{});
}

long long chunks_of(long long n, int chunk) { return (n + chunk - 1) / chunk; }

// Chunks of a list and their size, or a negative status and what is wrong.
int check(const oz_adamw_tensor* t, int count, long long* chunks, int* chunk, const char** what) {
    *chunks = 0;
    *chunk = 0;
    *what = "no tensors";
    if (count < 0 || (count > 0 && !t)) return OZ_ERR_ARG;
    long long values = 0;
    for (int k = 0; k < count; k++) {
        *what = "a tensor's size";
        if (t[k].n < 0 || t[k].n > 1ll << 36) return OZ_ERR_ARG;
        values += t[k].n;
        *what = "too many values";
        if (values > 1ll << 36) return OZ_ERR_ARG;
    }
    *chunk = chunk_of(values);
    for (int k = 0; k < count; k++) *chunks += chunks_of(t[k].n, *chunk);
    *what = "too many values";
    return *chunks > 1ll << 23 ? OZ_ERR_ARG : OZ_OK;
}

long long bytes_of(int count, long long chunks) { return (long long)count * sizeof(Entry) + chunks * 4 + 16; }

}  // namespace

extern "C" {

long long oz_adamw_plan_bytes(const oz_adamw_tensor* tensors, int count) {
    long long chunks;
    int chunk;
    const char* what;
    if (int st = check(tensors, count, &chunks, &chunk, &what)) return st;
    return bytes_of(count, chunks);
}

int oz_adamw_make_plan(oz_dev* dev, const oz_adamw_tensor* tensors, int count, int state_bits, void* memory,
                       size_t bytes, oz_adamw_plan* plan) {
    if (!plan) return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_make_plan: no plan to fill");
    *plan = oz_adamw_plan{};
    if (state_bits != 32 && state_bits != 8) return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_make_plan: states of %d bits", state_bits);
    long long chunks;
    int chunk;
    const char* what;
    if (int st = check(tensors, count, &chunks, &chunk, &what)) return oz::fail(dev, st, "oz_adamw_make_plan: %s", what);
    for (int k = 0; k < count; k++) {
        const oz_adamw_tensor& t = tensors[k];
        const auto known = [](int type) { return type == OZ_F32 || is_16bit(type); };
        if (!known(t.param_type) || !known(t.grad_type) || (t.master && t.param_type == OZ_F32))
            return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_make_plan: types of tensor %d", k);
        if (t.n && (!t.param || !t.grad || !t.m || !t.v || (state_bits == 8) != (t.m_scale && t.v_scale) ||
                    (state_bits == 32 && (t.m_scale || t.v_scale))))
            return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_make_plan: arrays of tensor %d", k);
        const int es = state_bits == 32 ? 4 : 1;
        if (((uintptr_t)t.param & (size_of(t.param_type) - 1)) || ((uintptr_t)t.grad & (size_of(t.grad_type) - 1)) ||
            ((uintptr_t)t.master & 3) || ((uintptr_t)t.m & (es - 1)) || ((uintptr_t)t.v & (es - 1)))
            return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_make_plan: tensor %d at an address that its type does not allow", k);
        if (!(t.weight_decay >= 0.0f && t.weight_decay < INFINITY))
            return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_make_plan: weight decay of tensor %d", k);
    }
    const long long need = bytes_of(count, chunks);
    if (!memory || (long long)bytes < need || ((uintptr_t)memory & 15))
        return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_make_plan: %zu bytes, %lld needed (16-byte aligned)", bytes, need);
    try {
        std::vector<unsigned char> image((size_t)need);
        Entry* e = reinterpret_cast<Entry*>(image.data());
        uint32_t* owner = reinterpret_cast<uint32_t*>(image.data() + (size_t)count * sizeof(Entry));
        long long first = 0;
        uint32_t block = 0;
        for (int k = 0; k < count; k++) {
            const oz_adamw_tensor& t = tensors[k];
            e[k] = Entry{t, first, block, chunk};
            for (long long c = chunks_of(t.n, chunk); c > 0; c--) owner[first++] = (uint32_t)k;
            block += (uint32_t)((t.n + OZ_ADAMW_BLOCK - 1) / OZ_ADAMW_BLOCK);
        }
        // The memory may come from an allocator that hands out again what kernels of its own stream still write: the kernel
        // takes its addresses from here, so the copy waits for the device.
        if (int st = oz::use(dev)) return st;
        if (int st = oz::hip_check(dev, hipDeviceSynchronize(), "hipDeviceSynchronize")) return st;
        if (int st = oz_memcpy_h2d(dev, memory, image.data(), image.size())) return st;
    } catch (const std::bad_alloc&) {
        return oz::fail(dev, OZ_ERR_NOMEM, "oz_adamw_make_plan: host memory");
    }
    *plan = oz_adamw_plan{memory, chunks, count, state_bits};
    return OZ_OK;
}

int oz_adamw_step(oz_dev* dev, const oz_adamw_plan* plan, const oz_adamw_options* o) {
    if (!plan || !o || !plan->memory) return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_step: no plan or options");
    const auto in = [](double x, double below) { return x >= 0.0 && x < below; };
    if (!in(o->lr, INFINITY) || !in(o->eps, INFINITY) || !in(o->beta1, 1.0) || !in(o->beta2, 1.0) || o->step < 1)
        return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_step: lr %g, beta1 %g, beta2 %g, eps %g, step %lld", o->lr, o->beta1, o->beta2, o->eps, o->step);
    if ((uintptr_t)o->grad_scale & 3) return oz::fail(dev, OZ_ERR_ARG, "oz_adamw_step: grad_scale at an odd address");
    if (int st = oz::use(dev)) return st;
    if (!plan->chunks) return OZ_OK;
    Step s;
    s.b1 = (float)o->beta1, s.a1 = (float)(1.0 - o->beta1);
    s.b2 = (float)o->beta2, s.a2 = (float)(1.0 - o->beta2);
    s.root = (float)(1.0 / std::sqrt(1.0 - std::pow(o->beta2, (double)o->step)));
    s.rate = (float)(o->lr / (1.0 - std::pow(o->beta1, (double)o->step)));
    s.eps = (float)o->eps, s.lr = (float)o->lr, s.seed = o->seed, s.grad_scale = o->grad_scale;
    const Entry* e = static_cast<const Entry*>(plan->memory);
    const uint32_t* owner = reinterpret_cast<const uint32_t*>(e + plan->count);
    const dim3 grid((unsigned)plan->chunks), block(THREADS);
    if (plan->state_bits == 32) hipLaunchKernelGGL(adamw_kernel<32>, grid, block, 0, dev->stream, e, owner, s);
    else hipLaunchKernelGGL(adamw_kernel<8>, grid, block, 0, dev->stream, e, owner, s);
    return oz::launch_check(dev, "adamw_kernel");
}

}  // extern "C"
