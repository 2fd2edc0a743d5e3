// Product with bias, activation and residual in its epilogue, and its gradients (include/oz_hip.h,
// oz_linear and oz_linear_grad).
//
//   Y = act(X W^T + bias) + residual;  dZ = dY act'(Z),  dX = dZ W,  dW = dZ^T X,  dbias = sum of dZ's rows
//
// All three products are C(q, p) = sum over c of Q(q, c) P(p, c), with P's index along the rows of the
// output: Y has q = m, p = n, c = k; dX q = m, p = k, c = n; dW q = n, p = k, c = m.
#include "oz_internal.hpp"
#include "oz_linear.hpp"

namespace {

using namespace ozt;

// Any sizes, strides and alignment: 64 x 64 outputs by 4 waves of 32 x 32, operands element by element
// through LDS, 32 of c at a time. Elements outside are zeros.
template <int TYPE>
__global__ void __launch_bounds__(256) product_any_kernel(const ozl::Product a) {
    typedef typename Half<TYPE>::t T;
    typedef typename Half<TYPE>::x8 T8;
    constexpr int LD = 40;  // 16-byte rows, on other banks each
    __shared__ __attribute__((aligned(16))) T lq[64 * LD], lp[64 * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned across = (unsigned)((a.np + 63) / 64);
    const long long q0 = 64ll * (blockIdx.x / across), p0 = 64ll * (blockIdx.x % across);
    const T* Q = static_cast<const T*>(a.Q);
    const T* P = static_cast<const T*>(a.P);
    const int wq = 32 * (wave >> 1), wp = 32 * (wave & 1), r = lane & 15, g = lane >> 4;
    f32x4 acc[2][2] = {};
    for (long long c0 = 0; c0 < a.C; c0 += 32) {
        for (int e = threadIdx.x; e < 64 * 32; e += 256) {
            // consecutive threads along the operand's contiguous index
            const int cq = a.q_major ? e >> 6 : e & 31, iq = a.q_major ? e & 63 : e >> 5;
            const int cp = a.p_major ? e >> 6 : e & 31, ip = a.p_major ? e & 63 : e >> 5;
            lq[iq * LD + cq] = q0 + iq < a.nq && c0 + cq < a.C ? Q[a.q_major ? (c0 + cq) * a.ldq + q0 + iq : (q0 + iq) * a.ldq + c0 + cq] : (T)0.0f;
            lp[ip * LD + cp] = p0 + ip < a.np && c0 + cp < a.C ? P[a.p_major ? (c0 + cp) * a.ldp + p0 + ip : (p0 + ip) * a.ldp + c0 + cp] : (T)0.0f;
        }
        __syncthreads();
        // lane l brings row l % 16 and the 8 values of c from 8 (l / 16) on, of both operands
        T8 fq[2], fp[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            fq[i] = *reinterpret_cast<const T8*>(lq + (wq + 16 * i + r) * LD + 8 * g);
            fp[i] = *reinterpret_cast<const T8*>(lp + (wp + 16 * i + r) * LD + 8 * g);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = Half<TYPE>::mfma(fp[j], fq[i], acc[i][j]);
        __syncthreads();
    }
    // register k of lane l: p = 4 (l / 16) + k, q = l % 16
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const long long q = q0 + wq + 16 * i + r;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const long long p = p0 + wp + 16 * j + 4 * g + k;
                if (q < a.nq && p < a.np) ozl::finish(a.epi, TYPE, q, p, acc[i][j][k]);
            }
        }
}

// dZ = dY act'(Z), rounded for the products (left out where dz is null), and dbias: 64 columns by a workgroup,
// 4 of its waves a row each.
__global__ void __launch_bounds__(256) act_grad_kernel(const void* __restrict__ dY, const void* __restrict__ Z,
                                                       void* __restrict__ dz, void* __restrict__ dbias, int type,
                                                       int dw_type, int act, int accumulate, long long M, int N,
                                                       long long lddy, long long ldz) {
    const int col = blockIdx.x * 64 + (threadIdx.x & 63);
    float sum = 0.0f;
    if (col < N)
        for (long long m = threadIdx.x >> 6; m < M; m += 4) {
            float d = load(dY, type, m * lddy + col);
            if (act != OZ_ACT_NONE) d *= act_grad(load(Z, type, m * ldz + col), act);
            if (dz) store(dz, type, m * N + col, d);
            sum += d;
        }
    __shared__ float part[256];
    part[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < 64 && col < N && dbias) {
        sum = (part[threadIdx.x] + part[64 + threadIdx.x]) + (part[128 + threadIdx.x] + part[192 + threadIdx.x]);
        if (accumulate) sum += load(dbias, dw_type, col);
        store(dbias, dw_type, col, sum);
    }
}

constexpr long long kMaxTiles = 1ll << 23;  // workgroups of 256 threads in one launch

int launch_product(oz_dev* dev, int type, const ozl::Product& a) {
    if (!a.nq || !a.np) return OZ_OK;
    const long long tiles = (long long)oz::ceil_div(a.np, 64) * oz::ceil_div(a.nq, 64);
    if (tiles > kMaxTiles) return oz::fail(dev, OZ_ERR_ARG, "a product of %lld x %lld outputs is too large", a.nq, a.np);
    const dim3 grid((unsigned)tiles);
    if (type == OZ_BF16) hipLaunchKernelGGL(product_any_kernel<OZ_BF16>, grid, dim3(256), 0, dev->stream, a);
    else hipLaunchKernelGGL(product_any_kernel<OZ_F16>, grid, dim3(256), 0, dev->stream, a);
    return oz::launch_check(dev, "product_any_kernel");
}

constexpr long long kMaxLd = 1ll << 22;  // offsets inside a tile's operands are 32-bit

bool bad_ld(long long ld, int row) { return ld != 0 && (ld < row || ld > kMaxLd); }
long long or_row(long long ld, int row) { return ld ? ld : row; }

// What is wrong with a descriptor, or null.
const char* refuse(const oz_linear_desc* d) {
    if (!d) return "no descriptor";
    if (d->M < 0 || d->N < 1 || d->K < 1) return "sizes";
    if (d->N > kMaxLd || d->K > kMaxLd) return "rows longer than 2^22 values";
    if (!is_16bit(d->type)) return "the operands' type";
    if (d->y_type != d->type && d->y_type != OZ_F32) return "the output's type";
    if (d->act < OZ_ACT_NONE || d->act > OZ_ACT_SILU) return "the activation";
    if (bad_ld(d->ldx, d->K) || bad_ld(d->ldw, d->K) || bad_ld(d->ldy, d->N) || bad_ld(d->ldr, d->N) || bad_ld(d->ldz, d->N))
        return "a leading dimension";
    return nullptr;
}

const char* refuse(const oz_linear_grad_desc* d) {
    if (!d) return "no descriptor";
    if (d->M < 0 || d->N < 1 || d->K < 1) return "sizes";
    if (d->N > kMaxLd || d->K > kMaxLd) return "rows longer than 2^22 values";
    if (!is_16bit(d->type)) return "the operands' type";
    if (d->dw_type != d->type && d->dw_type != OZ_F32) return "the type of dW";
    if (d->act < OZ_ACT_NONE || d->act > OZ_ACT_SILU) return "the activation";
    if (d->accumulate != 0 && d->accumulate != 1) return "accumulate";
    if (bad_ld(d->lddy, d->N) || bad_ld(d->ldx, d->K) || bad_ld(d->ldw, d->K) || bad_ld(d->ldz, d->N) ||
        bad_ld(d->lddx, d->K) || bad_ld(d->lddw, d->K))
        return "a leading dimension";
    return nullptr;
}

bool misaligned(const void* p, int type) { return ((uintptr_t)p & (size_of(type) - 1)) != 0; }

size_t dz_bytes(const oz_linear_grad_desc* d) {
    return d->act == OZ_ACT_NONE ? 0 : ((size_t)d->M * d->N * 2 + 255) & ~(size_t)255;
}

}  // namespace

extern "C" {

long long oz_linear_workspace(oz_dev* dev, const oz_linear_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear: %s", e);
    return 0;
}

int oz_linear(oz_dev* dev, const oz_linear_desc* d, const void* X, const void* W, const void* bias,
              const void* residual, void* Y, void* Z, void* work, size_t bytes) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear: %s", e);
    if (d->M > 0 && (!X || !W || !Y)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear: null operand");
    if (misaligned(X, d->type) || misaligned(W, d->type) || misaligned(bias, d->type) || misaligned(Z, d->type) ||
        misaligned(residual, d->y_type) || misaligned(Y, d->y_type))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear: operands at addresses that their types do not allow");
    if (residual == Y && residual && or_row(d->ldr, d->N) != or_row(d->ldy, d->N))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear: residual is Y with another leading dimension");
    if (int st = oz::use(dev)) return st;
    if (d->M == 0) return OZ_OK;
    (void)work, (void)bytes;
    ozl::Product p{};
    p.Q = X, p.P = W, p.nq = d->M, p.np = d->N, p.C = d->K, p.ldq = or_row(d->ldx, d->K), p.ldp = or_row(d->ldw, d->K);
    p.epi = {Y, or_row(d->ldy, d->N), d->y_type, Z, or_row(d->ldz, d->N), bias, residual, or_row(d->ldr, d->N), d->act, 0};
    return launch_product(dev, d->type, p);
}

long long oz_linear_grad_workspace(oz_dev* dev, const oz_linear_grad_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: %s", e);
    return (long long)dz_bytes(d);
}

int oz_linear_grad(oz_dev* dev, const oz_linear_grad_desc* d, const void* dY, const void* X, const void* W,
                   const void* Z, void* dX, void* dW, void* dbias, void* work, size_t bytes) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: %s", e);
    const bool curved = d->act != OZ_ACT_NONE;
    if (d->M > 0 && (dX || dW || dbias) && (!dY || (curved && !Z) || (dX && !W) || (dW && !X)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: null operand");
    if (misaligned(dY, d->type) || misaligned(X, d->type) || misaligned(W, d->type) || misaligned(Z, d->type) ||
        misaligned(dX, d->type) || misaligned(dW, d->dw_type) || misaligned(dbias, d->dw_type))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: operands at addresses that their types do not allow");
    const size_t need = dz_bytes(d);
    if (need && (!work || bytes < need || ((uintptr_t)work & 15)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
    if (int st = oz::use(dev)) return st;
    const void* dz = dY;
    long long lddz = or_row(d->lddy, d->N);
    const bool products = d->M > 0 && (dX || dW);
    if ((curved && products) || dbias) {
        if (curved) dz = work, lddz = d->N;
        hipLaunchKernelGGL(act_grad_kernel, dim3(oz::ceil_div(d->N, 64)), dim3(256), 0, dev->stream, dY, Z,
                           curved && products ? work : nullptr, dbias, d->type, d->dw_type, d->act, d->accumulate,
                           (long long)d->M, d->N, or_row(d->lddy, d->N), or_row(d->ldz, d->N));
        if (int st = oz::launch_check(dev, "act_grad_kernel")) return st;
    }
    if (dX && d->M > 0) {
        ozl::Product p{};
        p.Q = dz, p.P = W, p.nq = d->M, p.np = d->K, p.C = d->N, p.ldq = lddz, p.ldp = or_row(d->ldw, d->K), p.p_major = 1;
        p.epi = {dX, or_row(d->lddx, d->K), d->type, nullptr, 0, nullptr, nullptr, 0, OZ_ACT_NONE, 0};
        if (int st = launch_product(dev, d->type, p)) return st;
    }
    if (dW) {
        ozl::Product p{};
        p.Q = dz, p.P = X, p.nq = d->N, p.np = d->K, p.C = d->M, p.ldq = lddz, p.ldp = or_row(d->ldx, d->K), p.q_major = p.p_major = 1;
        p.epi = {dW, or_row(d->lddw, d->K), d->dw_type, nullptr, 0, nullptr, nullptr, 0, OZ_ACT_NONE, d->accumulate};
        if (int st = launch_product(dev, d->type, p)) return st;
    }
    return OZ_OK;
}

}  // extern "C"
