// Rows as 8-bit integers with a scale each (include/oz_hip.h, oz_quantize_rows).
#include "oz_quantize.hpp"

#include "oz_internal.hpp"

namespace {

using namespace ozt;
using namespace ozq;

constexpr int THREADS = 256, V = 8;

// A workgroup a row: the largest value, then the integers, from memory each time.
template <int TYPE>
__global__ void __launch_bounds__(THREADS) quantize_kernel(long long M, int K, const void* __restrict__ X, long long ldx, int8_t* __restrict__ Q, long long ldq,
                                                           int fill, float* __restrict__ scale) {
    __shared__ unsigned part[THREADS / 64];
    const long long row = blockIdx.x + (long long)gridDim.x * blockIdx.y;
    if (row >= M) return;
    auto get = [&](int col, float* x) {
        if (col + V <= K) load8(X, TYPE, row * ldx + col, x);
        else load_some(X, TYPE, row * ldx + col, max(K - col, 0), x);
    };
    unsigned top = 0;
    for (int col = V * threadIdx.x; col < K; col += V * THREADS) {
        float x[V];
        get(col, x);
#pragma unroll
        for (int k = 0; k < V; k++) top = max(top, bits_of(x[k]));
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) top = max(top, __shfl_xor(top, d));
    if (!(threadIdx.x & 63)) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < THREADS / 64; k++) top = max(top, part[k]);
    const Scale s = scale_of(top);
    if (threadIdx.x == 0) scale[row] = s.scale;
    for (int col = V * threadIdx.x; col < fill; col += V * THREADS) {
        float x[V];
        get(col, x);
        const unsigned w[2] = {pack4(x, s.inverse), pack4(x + 4, s.inverse)};
        int8_t* to = Q + row * ldq + col;
        if (col + V <= fill) {
            __builtin_memcpy(to, w, V);
        } else {
#pragma unroll
            for (int k = 0; k < V; k++)
                if (col + k < fill) to[k] = (int8_t)(w[k / 4] >> (8 * (k % 4)));
        }
    }
}

bool misaligned(const void* p, int type) { return ((uintptr_t)p & (size_of(type) - 1)) != 0; }

}  // namespace

int ozq::launch_quantize(oz_dev* dev, int type, long long M, int K, const void* X, long long ldx, int8_t* Q, long long ldq, int fill, float* scale) {
    const long long x = M < 1 << 23 ? M : 1 << 23;
    const dim3 grid((unsigned)x, (unsigned)((M + x - 1) / x)), block(THREADS);
    if (type == OZ_F32) hipLaunchKernelGGL(quantize_kernel<OZ_F32>, grid, block, 0, dev->stream, M, K, X, ldx, Q, ldq, fill, scale);
    else if (type == OZ_BF16) hipLaunchKernelGGL(quantize_kernel<OZ_BF16>, grid, block, 0, dev->stream, M, K, X, ldx, Q, ldq, fill, scale);
    else hipLaunchKernelGGL(quantize_kernel<OZ_F16>, grid, block, 0, dev->stream, M, K, X, ldx, Q, ldq, fill, scale);
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
