// Products of few rows (an answering program's tokens): Y = act(X W^T + bias) + residual with M <= 32.
//
// The weights are read once and used M times, so the time is theirs: the waves stream them straight into registers, with
// no LDS and no barrier on the way, as one operand of the matrix instructions (16 rows of W x 32 values of c; M = 1 wastes
// 15 of their 16 columns, and there are still 20 times more than the weights' bandwidth could feed), the rows of X, which
// all workgroups share, come from the L2. A workgroup has 16 NB rows of W and deals c out to its 8 waves, 64 or 128 at a time,
// so that together they read 1 or 2 KB of each row in a piece; the waves' sums are joined in LDS, in order. Few rows of
// W (N small): ranges of c go to several workgroups, joined by a second launch.
#include "oz_internal.hpp"
#include "oz_linear.hpp"

namespace {

using namespace ozl;
using namespace ozt;

constexpr int WAVES = 8;

template <int TYPE, int MB, int NB>
__global__ void __launch_bounds__(64 * WAVES, 4) few_rows_kernel(const Product a, int blocks_p) {
    typedef typename Half<TYPE>::t T;
    typedef typename Half<TYPE>::x8 T8;
    constexpr int F = MB == 1 ? 4 : 2, UNIT = 32 * F;  // values of c that a wave takes at a time
    __shared__ f32x4 sums[WAVES][NB * MB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.x / blocks_p;
    const long long p0 = 16ll * NB * (blockIdx.x - split * blocks_p);
    const int r = lane & 15, g = lane >> 4;
    // rows beyond an operand's last are its last one again; their sums are not used
    const T *pw[NB], *px[MB];
#pragma unroll
    for (int n = 0; n < NB; n++) pw[n] = static_cast<const T*>(a.P) + (p0 + 16 * n + r < a.np ? p0 + 16 * n + r : a.np - 1) * a.ldp + 8 * g;
#pragma unroll
    for (int m = 0; m < MB; m++) px[m] = static_cast<const T*>(a.Q) + (16 * m + r < a.nq ? 16 * m + r : a.nq - 1) * a.ldq + 8 * g;
    const int units = (int)(a.C / UNIT);  // whole ones; what is left behind them goes to one wave of the last range
    const int u0 = (int)((long long)units * split / a.splits), u1 = (int)((long long)units * (split + 1) / a.splits);
    f32x4 acc[NB][MB] = {};
    T8 w[2][NB][F], x[2][MB][F];
    auto ask = [&](int b, int u) {
        if (u < u1) {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int f = 0; f < F; f++) w[b][n][f] = get16<T8>(pw[n] + (long long)u * UNIT + 32 * f);
#pragma unroll
            for (int m = 0; m < MB; m++)
#pragma unroll
                for (int f = 0; f < F; f++) x[b][m][f] = get16<T8>(px[m] + (long long)u * UNIT + 32 * f);
        }
    };
    auto multiply = [&](int b) {
#pragma unroll
        for (int f = 0; f < F; f++)
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int m = 0; m < MB; m++) acc[n][m] = Half<TYPE>::mfma(w[b][n][f], x[b][m][f], acc[n][m]);
    };
    int u = u0 + wave;
    ask(0, u);
    for (; u < u1; u += 2 * WAVES) {
        ask(1, u + WAVES);
        multiply(0);
        ask(0, u + 2 * WAVES);
        if (u + WAVES < u1) multiply(1);
    }
    if (split == a.splits - 1 && wave == WAVES - 1 && a.C % UNIT) {
        for (long long c = (long long)units * UNIT; c < a.C; c += 32) {
            T8 wt[NB], xt[MB];
            auto guarded = [&](const T* p) {  // p: this lane's first chunk of the row
                T8 v;
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = c + 8 * g + k < a.C ? p[c + k] : (T)0.0f;
                return v;
            };
#pragma unroll
            for (int n = 0; n < NB; n++) wt[n] = guarded(pw[n]);
#pragma unroll
            for (int m = 0; m < MB; m++) xt[m] = guarded(px[m]);
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int m = 0; m < MB; m++) acc[n][m] = Half<TYPE>::mfma(wt[n], xt[m], acc[n][m]);
        }
    }
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
        for (int m = 0; m < MB; m++) sums[wave][n * MB + m][lane] = acc[n][m];
    __syncthreads();
    // 16 NB values of p a row, next to each other
    for (int e = threadIdx.x; e < 256 * NB * MB; e += 64 * WAVES) {
        const int i = e % (16 * NB), q = e / (16 * NB);
        if (q >= a.nq || p0 + i >= a.np) continue;
        const int block = (i / 16) * MB + q / 16, from = 16 * (i % 16 / 4) + q % 16, k = i % 4;
        float v = sums[0][block][from][k];
#pragma unroll
        for (int s = 1; s < WAVES; s++) v += sums[s][block][from][k];
        if (a.splits > 1) a.parts[(split * a.nq + q) * a.ldparts + p0 + i] = v;
        else finish(a.epi, TYPE, q, p0 + i, v);
    }
}

// One or two rows of X: a wave streams a row of W, 4 or 2 KB at a time, and multiplies on the vector units. Rows read in long
// pieces come at 5.5 TB/s where 16 rows x 64 bytes at a time, what the matrix instructions take, come at 4.7
// (8192 x 8192: 24 against 29 us by loads alone), and 8 products and 16 conversions for each 16 bytes take a quarter of
// the vector units' time. X comes from the caches, the CU's waves read the same pieces at about the same time. Few rows of W:
// KS waves share a row's c and are joined in LDS, in order.
template <int TYPE, int M>
__global__ void __launch_bounds__(64 * WAVES, 4) stream_rows_kernel(const Product a, int ks) {
    constexpr int U = 4 / M, STEP = 512 * U;
    __shared__ float sums[WAVES][M];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave % ks, rows = WAVES / ks;
    const long long p = (long long)blockIdx.x * rows + wave / ks;
    const uint16_t* pw = static_cast<const uint16_t*>(a.P) + (p < a.np ? p : a.np - 1) * a.ldp + 8 * lane;
    const uint16_t* px[M];
#pragma unroll
    for (int m = 0; m < M; m++) px[m] = static_cast<const uint16_t*>(a.Q) + m * a.ldq + 8 * lane;
    float acc[M] = {};
    auto add = [&](u32x4 w, const u32x4 (&x)[M]) {
        float v[8];
        widen8(w, TYPE, v);
#pragma unroll
        for (int m = 0; m < M; m++) {
            float y[8];
            widen8(x[m], TYPE, y);
#pragma unroll
            for (int k = 0; k < 8; k++) acc[m] = __builtin_fmaf(v[k], y[k], acc[m]);
        }
    };
    const int steps = (int)(a.C / STEP);  // whole ones, dealt out in turn; what is left behind them is the last wave's
    u32x4 w[2][U], x[2][U][M];
    auto ask = [&](int b, int s) {
        if (s < steps) {
#pragma unroll
            for (int u = 0; u < U; u++) w[b][u] = get16<u32x4>(pw + (long long)s * STEP + 512 * u);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int m = 0; m < M; m++) x[b][u][m] = get16<u32x4>(px[m] + (long long)s * STEP + 512 * u);
        }
    };
    int s = part;
    ask(0, s);
    for (; s < steps; s += 2 * ks) {
        ask(1, s + ks);
#pragma unroll
        for (int u = 0; u < U; u++) add(w[0][u], x[0][u]);
        ask(0, s + 2 * ks);
        if (s + ks < steps)
#pragma unroll
            for (int u = 0; u < U; u++) add(w[1][u], x[1][u]);
    }
    if (part == ks - 1)
        for (long long c = (long long)steps * STEP; c + 8 * lane < a.C; c += 512) {
            auto some = [&](const uint16_t* row) {
                union {
                    uint16_t v[8];
                    u32x4 w;
                } t;
                t.w = u32x4{0, 0, 0, 0};
                if (c + 8 * lane + 8 <= a.C) t.w = get16<u32x4>(row + c);
                else
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (c + 8 * lane + k < a.C) t.v[k] = row[c + k];
                return t.w;
            };
            u32x4 y[M];
#pragma unroll
            for (int m = 0; m < M; m++) y[m] = some(px[m]);
            add(some(pw), y);
        }
#pragma unroll
    for (int m = 0; m < M; m++) {
        float v = acc[m];
#pragma unroll
        for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
        if (lane == 0) sums[wave][m] = v;
    }
    __syncthreads();
    if ((int)threadIdx.x < rows * M) {
        const int i = threadIdx.x % rows, m = threadIdx.x / rows;
        const long long at = (long long)blockIdx.x * rows + i;
        if (at >= a.np) return;
        float v = sums[i * ks][m];
        for (int k = 1; k < ks; k++) v += sums[i * ks + k][m];
        finish(a.epi, TYPE, m, at, v);
    }
}

template <int TYPE, int M>
int launch_stream(oz_dev* dev, const Product& a) {
    // waves that share a row: so many that the chip has 16 on each CU, as long as each has something to read
    int ks = 1;
    while (ks < WAVES && a.np * ks < 16ll * dev->cus && (long long)ks * 2048 < a.C) ks *= 2;
    const unsigned grid = oz::ceil_div(a.np, WAVES / ks);
    hipLaunchKernelGGL((stream_rows_kernel<TYPE, M>), dim3(grid), dim3(64 * WAVES), 0, dev->stream, a, ks);
    return oz::launch_check(dev, "stream_rows_kernel");
}

template <int TYPE, int MB, int NB>
int launch(oz_dev* dev, const Product& a) {
    const int blocks_p = (int)oz::ceil_div(a.np, ozl::few_rows_block(a.nq));
    static_assert(NB == (MB == 1 ? 1 : 2), "few_rows_block");
    const dim3 grid((unsigned)blocks_p * a.splits);
    hipLaunchKernelGGL((few_rows_kernel<TYPE, MB, NB>), grid, dim3(64 * WAVES), 0, dev->stream, a, blocks_p);
    if (int st = oz::launch_check(dev, "few_rows_kernel")) return st;
    return a.splits > 1 ? ozl::launch_join(dev, TYPE, a) : OZ_OK;
}

template <int TYPE>
int by_rows(oz_dev* dev, const Product& a) {
    if (a.nq <= kStreamRows) return a.nq == 1 ? launch_stream<TYPE, 1>(dev, a) : launch_stream<TYPE, 2>(dev, a);
    if (a.nq <= 16) return launch<TYPE, 1, 1>(dev, a);
    return launch<TYPE, 2, 2>(dev, a);
}

}  // namespace

int ozl::launch_few_rows(oz_dev* dev, int type, const Product& a) {
    return type == OZ_BF16 ? by_rows<OZ_BF16>(dev, a) : by_rows<OZ_F16>(dev, a);
}
