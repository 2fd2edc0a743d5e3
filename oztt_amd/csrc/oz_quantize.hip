// Rows as 8-bit integers with a scale each (include/oz_hip.h, oz_quantize_rows).
#include "oz_quantize.hpp"

#include "oz_internal.hpp"

namespace {

using namespace ozt;
using namespace ozq;

constexpr int THREADS = 256, V = 8;

// LANES threads a row (part of a wave, a wave or a workgroup), PIECES pieces of 8 values each, which stay in registers between the largest value and the
// integers; PIECES = 0: rows that do not fit, read twice. Bound by memory: 8192^2 BF16 values in 40 us (201 MB, 5.0 TB/s; read twice, the second
// time out of the caches, 47.7).
template <int TYPE, int LANES, int PIECES>
__global__ void __launch_bounds__(THREADS) quantize_kernel(long long M, int K, const void* __restrict__ X, long long ldx, int8_t* __restrict__ Q, long long ldq,
                                                           int fill, float* __restrict__ scale) {
    __shared__ unsigned part[THREADS / 64];
    const int lane = threadIdx.x % LANES;
    const long long row = (blockIdx.x + (long long)gridDim.x * blockIdx.y) * (THREADS / LANES) + threadIdx.x / LANES;
    const bool in = row < M;
    auto get = [&](int col, float* x) {
        if (col + V <= K) load8(X, TYPE, row * ldx + col, x);
        else load_some(X, TYPE, row * ldx + col, max(K - col, 0), x);
    };
    float kept[PIECES ? PIECES : 1][V];
    unsigned top = 0;
    auto look = [&](const float* x) {
#pragma unroll
        for (int k = 0; k < V; k++) top = max(top, bits_of(x[k]));
    };
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int j = 0; j < PIECES; j++) {
            const int col = V * (LANES * j + lane);
#pragma unroll
            for (int k = 0; k < V; k++) kept[j][k] = 0.0f;
            if (in && col < K) get(col, kept[j]);
        }
#pragma unroll
        for (int j = 0; j < PIECES; j++) look(kept[j]);
    } else if (in) {
        for (int col = V * lane; col < K; col += V * LANES) {
            float x[V];
            get(col, x);
            look(x);
        }
    }
#pragma unroll
    for (int d = (LANES < 64 ? LANES : 64) / 2; d > 0; d /= 2) top = max(top, (unsigned)__shfl_xor(top, d));
    if constexpr (LANES > 64) {
        if (!(threadIdx.x & 63)) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < THREADS / 64; k++) top = max(top, part[k]);
    }
    if (!in) return;
    const Scale s = scale_of(top);
    if (lane == 0) scale[row] = s.scale;
    auto put = [&](int col, const float* x) {
        const unsigned w[2] = {pack4(x, s.inverse), pack4(x + 4, s.inverse)};
        int8_t* to = Q + row * ldq + col;
        if (col + V <= fill) {
            __builtin_memcpy(to, w, V);
        } else {
#pragma unroll
            for (int k = 0; k < V; k++)
                if (col + k < fill) to[k] = (int8_t)(w[k / 4] >> (8 * (k % 4)));
        }
    };
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int j = 0; j < PIECES; j++) put(V * (LANES * j + lane), kept[j]);
        // the zeros behind K, where the pieces end before
        const float none[V] = {};
        for (int col = V * (LANES * PIECES + lane); col < fill; col += V * LANES) put(col, none);
    } else {
        for (int col = V * lane; col < fill; col += V * LANES) {
            float x[V];
            get(col, x);
            put(col, x);
        }
    }
}

template <int TYPE, int LANES, int PIECES>
void launch(oz_dev* dev, long long M, int K, const void* X, long long ldx, int8_t* Q, long long ldq, int fill, float* scale) {
    const long long groups = (M + THREADS / LANES - 1) / (THREADS / LANES), x = groups < 1 << 23 ? groups : 1 << 23;
    hipLaunchKernelGGL((quantize_kernel<TYPE, LANES, PIECES>), dim3((unsigned)x, (unsigned)((groups + x - 1) / x)), dim3(THREADS), 0, dev->stream, M, K, X, ldx,
                       Q, ldq, fill, scale);
}

template <int TYPE>
void by_length(oz_dev* dev, long long M, int K, const void* X, long long ldx, int8_t* Q, long long ldq, int fill, float* scale) {
    const auto with = [&](auto kernel) { kernel(dev, M, K, X, ldx, Q, ldq, fill, scale); };
    if (K <= 128) with(launch<TYPE, 16, 1>);
    else if (K <= 512) with(launch<TYPE, 64, 1>);
    else if (K <= 2048 && M <= 1024) with(launch<TYPE, 256, 1>);  // few rows: 24 x 2048 in 3.3 us, a wave a row in 4.0; many: 4096 x 1024 5.7, 3.6
    else if (K <= 1024) with(launch<TYPE, 64, 2>);
    else if (K <= 2048) with(launch<TYPE, 64, 4>);
    else if (K <= 4096) with(launch<TYPE, 256, 2>);
    else if (K <= 8192) with(launch<TYPE, 256, 4>);
    else if (K <= 16384) with(launch<TYPE, 256, 8>);
    else with(launch<TYPE, 256, 0>);
}

bool misaligned(const void* p, int type) { return ((uintptr_t)p & (size_of(type) - 1)) != 0; }

}  // namespace

int ozq::launch_quantize(oz_dev* dev, int type, long long M, int K, const void* X, long long ldx, int8_t* Q, long long ldq, int fill, float* scale) {
    if (type == OZ_F32) by_length<OZ_F32>(dev, M, K, X, ldx, Q, ldq, fill, scale);
    else if (type == OZ_BF16) by_length<OZ_BF16>(dev, M, K, X, ldx, Q, ldq, fill, scale);
    else by_length<OZ_F16>(dev, M, K, X, ldx, Q, ldq, fill, scale);
    return oz::launch_check(dev, "quantize_kernel");
}

extern "C" int oz_quantize_rows(oz_dev* dev, const oz_quantize_desc* d, const void* X, int8_t* Q, float* scale) {
    const auto bad_ld = [&](long long ld) { return ld != 0 && (ld < d->K || ld > 1ll << 32); };
    const char* e = !d                                                   ? "no descriptor"
                    : d->M < 0 || d->M > 0x7FFFFFFF || d->K < 1 || d->K > 1 << 22 ? "sizes"
                    : d->type != OZ_F32 && !is_16bit(d->type)            ? "the type"
                    : bad_ld(d->ldx) || bad_ld(d->ldq)                   ? "a leading dimension"
                    : d->M && (!X || !Q || !scale)                       ? "null operand"
                    : misaligned(X, d->type) || misaligned(scale, OZ_F32) ? "operands at addresses that their types do not allow"
                                                                         : nullptr;
    if (e) return oz::fail(dev, OZ_ERR_ARG, "oz_quantize_rows: %s", e);
    if (int st = oz::use(dev)) return st;
    if (!d->M) return OZ_OK;
    return ozq::launch_quantize(dev, d->type, d->M, d->K, X, d->ldx ? d->ldx : d->K, Q, d->ldq ? d->ldq : d->K, d->K, scale);
}
