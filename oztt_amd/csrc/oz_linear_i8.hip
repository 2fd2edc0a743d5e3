// Product of 8-bit integers with bias, activation and residual (include/oz_hip.h, oz_linear_i8).
#include "oz_internal.hpp"
#include "oz_linear.hpp"
#include "oz_quantize.hpp"

namespace {

using namespace ozt;
using namespace ozl;

typedef int v4i __attribute__((ext_vector_type(4)));

struct Scaled {
    const int8_t *X, *W;
    const float *x_scale, *w_scale;
    long long M, N, ldx, ldw;
    int K, type;
    Epilogue epi;
};

// 64 x 64 outputs by 4 waves of 32 x 32, operands through LDS, 64 of k at a time.
__global__ void __launch_bounds__(256) product_kernel(const Scaled a) {
    constexpr int LD = 80;
    __shared__ __attribute__((aligned(16))) int8_t lx[64 * LD], lw[64 * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long across = (a.N + 63) / 64, tile = blockIdx.x + (long long)gridDim.x * blockIdx.y;
    const long long m0 = 64 * (tile / across), n0 = 64 * (tile % across);
    if (m0 >= a.M) return;
    const int wm = 32 * (wave >> 1), wn = 32 * (wave & 1), r = lane & 15, g = lane >> 4;
    v4i acc[2][2] = {};
    for (int k0 = 0; k0 < a.K; k0 += 64) {
        for (int e = threadIdx.x; e < 64 * 64; e += 256) {
            const int k = e & 63, i = e >> 6;
            lx[i * LD + k] = m0 + i < a.M && k0 + k < a.K ? a.X[(m0 + i) * a.ldx + k0 + k] : 0;
            lw[i * LD + k] = n0 + i < a.N && k0 + k < a.K ? a.W[(n0 + i) * a.ldw + k0 + k] : 0;
        }
        __syncthreads();
        v4i fx[2], fw[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            fx[i] = *reinterpret_cast<const v4i*>(lx + (wm + 16 * i + r) * LD + 16 * g);
            fw[i] = *reinterpret_cast<const v4i*>(lw + (wn + 16 * i + r) * LD + 16 * g);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j], fx[i], acc[i][j], 0, 0, 0);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const long long m = m0 + wm + 16 * i + r;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const long long n = n0 + wn + 16 * j + 4 * g + k;
                if (m < a.M && n < a.N) finish(a.epi, a.type, m, n, (float)acc[i][j][k] * a.w_scale[n] * a.x_scale[m]);
            }
        }
}

constexpr long long kMaxLd = 1ll << 22;
constexpr int kMaxK = 131071;  // 128 * 128 * K < 2^31

bool bad_ld(long long ld, int row) { return ld != 0 && (ld < row || ld > kMaxLd); }
long long or_row(long long ld, int row) { return ld ? ld : row; }
bool misaligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) != 0; }

const char* refuse(const oz_linear_i8_desc* d) {
    if (!d) return "no descriptor";
    if (d->M < 0 || d->N < 1 || d->K < 1) return "sizes";
    if (d->N > kMaxLd) return "rows longer than 2^22 values";
    if (d->K > kMaxK) return "K beyond 131071, where int32 sums could overflow";
    if (!is_16bit(d->type)) return "the type of X and bias";
    if (d->y_type != d->type && d->y_type != OZ_F32) return "the output's type";
    if (d->act < OZ_ACT_NONE || d->act > OZ_ACT_SILU) return "the activation";
    if (d->x_int8 != 0 && d->x_int8 != 1) return "x_int8";
    if (bad_ld(d->ldx, d->K) || bad_ld(d->ldw, d->K) || bad_ld(d->ldy, d->N) || bad_ld(d->ldr, d->N)) return "a leading dimension";
    if (or_row(d->ldw, d->K) % 4 || (d->x_int8 && or_row(d->ldx, d->K) % 4)) return "rows of 8-bit integers at no multiples of 4 bytes";
    return nullptr;
}

size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
int padded(int K) { return (K + 127) / 128 * 128; }
size_t x_bytes(const oz_linear_i8_desc* d) { return d->x_int8 ? 0 : up((size_t)d->M * padded(d->K)); }
size_t scale_bytes(const oz_linear_i8_desc* d) { return d->x_int8 ? 0 : up(4 * (size_t)d->M); }

}  // namespace

extern "C" {

long long oz_linear_i8_workspace(oz_dev* dev, const oz_linear_i8_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: %s", e);
    return (long long)(x_bytes(d) + scale_bytes(d));
}

int oz_linear_i8(oz_dev* dev, const oz_linear_i8_desc* d, const void* X, const float* x_scale, const int8_t* W,
                 const float* w_scale, const void* bias, const void* residual, void* Y, void* work, size_t bytes) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: %s", e);
    if (d->M > 0 && (!X || !W || !w_scale || !Y || (d->x_int8 && !x_scale))) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: null operand");
    if (misaligned(X, d->x_int8 ? 4 : 2) || misaligned(W, 4) || misaligned(x_scale, 4) || misaligned(w_scale, 4) || misaligned(bias, 2) ||
        misaligned(residual, size_of(d->y_type)) || misaligned(Y, size_of(d->y_type)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: operands at addresses that their types do not allow (8-bit integers: multiples of 4)");
    if (residual == Y && residual && or_row(d->ldr, d->N) != or_row(d->ldy, d->N))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: residual is Y with another leading dimension");
    const size_t need = (size_t)oz_linear_i8_workspace(dev, d);
    if (need && (!work || bytes < need || misaligned(work, 16)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
    if (int st = oz::use(dev)) return st;
    if (d->M == 0) return OZ_OK;
    Scaled a{};
    a.X = static_cast<const int8_t*>(X), a.W = W, a.x_scale = x_scale, a.w_scale = w_scale;
    a.M = d->M, a.N = d->N, a.K = d->K, a.ldx = or_row(d->ldx, d->K), a.ldw = or_row(d->ldw, d->K), a.type = d->type;
    a.epi = {Y, or_row(d->ldy, d->N), d->y_type, nullptr, 0, bias, residual, or_row(d->ldr, d->N), d->act};
    if (!d->x_int8) {
        int8_t* q = static_cast<int8_t*>(work);
        float* scale = reinterpret_cast<float*>(q + x_bytes(d));
        const int fill = padded(d->K);
        if (int st = ozq::launch_quantize(dev, d->type, d->M, d->K, X, a.ldx, q, fill, fill, scale)) return st;
        a.X = q, a.x_scale = scale, a.ldx = fill;
    }
    const long long tiles = ((a.M + 63) / 64) * ((a.N + 63) / 64), x = tiles < 1 << 23 ? tiles : 1 << 23;
    hipLaunchKernelGGL(product_kernel, dim3((unsigned)x, (unsigned)((tiles + x - 1) / x)), dim3(256), 0, dev->stream, a);
    return oz::launch_check(dev, "product_kernel");
}

}  // extern "C"
