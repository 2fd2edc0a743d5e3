// Product with bias, activation and residual in its epilogue, and its gradients (include/oz_hip.h,
// oz_linear and oz_linear_grad).
//
//   Y = act(X W^T + bias) + residual;  dZ = dY act'(Z),  dX = dZ W,  dW = dZ^T X,  dbias = sum of dZ's rows
//
// All three products are C(q, p) = sum over c of Q(q, c) P(p, c), with P's index along the rows of the
// output: Y has q = m, p = n, c = k; dX q = m, p = k, c = n; dW q = n, p = k, c = m.
#include "oz_internal.hpp"
#include "oz_linear.hpp"

#include <algorithm>
#include <type_traits>

namespace {

using namespace ozt;
using namespace ozl;

// Any sizes, strides and alignment: 64 x 64 outputs by 4 waves of 32 x 32, operands element by element
// through LDS, 32 of c at a time. Elements outside are zeros.
template <int TYPE>
__global__ void __launch_bounds__(256) product_any_kernel(const ozl::Product a) {
    typedef typename Half<TYPE>::t T;
    typedef typename Half<TYPE>::x8 T8;
    constexpr int LD = 40;  // 16-byte rows, on other banks each
    __shared__ __attribute__((aligned(16))) T lq[64 * LD], lp[64 * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long across = (a.np + 63) / 64, tile = blockIdx.x + (long long)gridDim.x * blockIdx.y;
    const long long q0 = 64 * (tile / across), p0 = 64 * (tile % across);
    if (q0 >= a.nq) return;
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

// dZ = dY act'(Z), rounded for the products (left out where dz is null), and the sums of its columns over `rows` rows each,
// to dbias if one range holds all rows, else to parts (left out where both are null): 8 columns a lane, 8 LANES columns by
// 256 / LANES rows at a time by a workgroup. One pass over dY and Z, which are not read again and pass the caches by.
// The matrix cores read 16 bits. For gradients in 16 bits one rounding of dZ is as large as the outputs' own (8192 x 8192 x 2048
// in BF16: 2.3e-3 of their norm against 1.7e-3 for the outputs' rounding alone) and two products would take twice the time; a dW
// in FP32 would show it, so its products also get what the rounding leaves, rounded in turn, in `rest` (TWO): together 16 bits
// of a BF16 dZ, 22 of an FP16 one, in 720 us for 492. What rounds to an infinity leaves nothing.
template <int LANES, int ACT, bool TWO>
__global__ void __launch_bounds__(256) act_grad_kernel(const void* __restrict__ dY, const void* __restrict__ Z,
                                                       void* __restrict__ dz, void* __restrict__ rest, float* __restrict__ parts,
                                                       void* __restrict__ dbias, int type, int dw_type, int accumulate, long long M, int N,
                                                       long long lddy, long long ldz, long long lddz, int rows, int strips) {
    constexpr int COLS = 8 * LANES, R = 256 / LANES;
    const int strip = blockIdx.x % strips, chunk = blockIdx.x / strips, l = threadIdx.x % LANES, r = threadIdx.x / LANES;
    // a row's last, fewer than 8 values: its last 8, of which the lane beside has the first `twice` too and writes the same
    const int at = strip * COLS + 8 * l, col = at + 8 <= N || N < 8 ? at : N - 8, twice = at - col;
    const long long end = (long long)(chunk + 1) * rows < M ? (long long)(chunk + 1) * rows : M;
    float sum[8] = {};
    if (at < N) {
        auto rows_of = [&](auto WHOLE) {
            constexpr bool whole = decltype(WHOLE)::value;
            auto get = [&](const void* p, long long i, float* x) {
                if constexpr (whole) load8(p, type, i, x);
                else load_some(p, type, i, N, x);
            };
#pragma unroll 4
            for (long long m = (long long)chunk * rows + r; m < end; m += R) {
                float x[8], y[8];
                get(dY, m * lddy + col, x);
                if constexpr (ACT != OZ_ACT_NONE) {
                    get(Z, m * ldz + col, y);
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = act_grad(x[k], y[k], ACT);
                }
                if (dz) store8(dz, type, m * lddz + col, x);
                if constexpr (TWO) {
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const float h = type == OZ_BF16 ? (float)(__bf16)x[k] : (float)(_Float16)x[k];
                        y[k] = fabsf(h) < INFINITY ? x[k] - h : 0.0f;
                    }
                    store8(rest, type, m * lddz + col, y);
                }
#pragma unroll
                for (int k = 0; k < 8; k++) sum[k] += x[k];
            }
        };
        if (N >= 8) rows_of(std::true_type{});
        else rows_of(std::false_type{});
    }
    if (!parts && !dbias) return;
    __shared__ float part[R][COLS];
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (k >= twice) part[r][8 * l + k - twice] = sum[k];
    __syncthreads();
    // R rows of sums to one, halving
    for (int h = R / 2; h > 0; h /= 2) {
        for (int e = threadIdx.x; e < h * COLS; e += 256) part[e / COLS][e % COLS] += part[e / COLS + h][e % COLS];
        __syncthreads();
    }
    const int c = strip * COLS + threadIdx.x;
    if (threadIdx.x < COLS && c < N) {
        float s = part[0][threadIdx.x];
        if (dbias) {
            if (accumulate) s += load(dbias, dw_type, c);
            store(dbias, dw_type, c, s);
        } else {
            parts[(long long)chunk * N + c] = s;
        }
    }
}

template <int LANES>
auto act_grad_of(int act, bool two) {
    return act == OZ_ACT_GELU   ? (two ? act_grad_kernel<LANES, OZ_ACT_GELU, true> : act_grad_kernel<LANES, OZ_ACT_GELU, false>)
           : act == OZ_ACT_SILU ? (two ? act_grad_kernel<LANES, OZ_ACT_SILU, true> : act_grad_kernel<LANES, OZ_ACT_SILU, false>)
           : act == OZ_ACT_RELU ? act_grad_kernel<LANES, OZ_ACT_RELU, false>
                                : act_grad_kernel<LANES, OZ_ACT_NONE, false>;
}

// dbias from the chunks' sums, 16 chunks at a time by 16 lanes: lane k of a column sums chunks k, k + 16, ..., then the lanes.
__global__ void __launch_bounds__(256) bias_grad_kernel(const float* __restrict__ parts, void* __restrict__ dbias, int dw_type,
                                                        int accumulate, int chunks, int N) {
    const int col = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4;
    __shared__ float part[16][16];
    float s = 0.0f;
    if (col < N)
        for (int c = k; c < chunks; c += 16) s += parts[(long long)c * N + col];
    part[k][threadIdx.x & 15] = s;
    __syncthreads();
    if (k == 0 && col < N) {
#pragma unroll
        for (int j = 1; j < 16; j++) s += part[j][threadIdx.x & 15];
        if (accumulate) s += load(dbias, dw_type, col);
        store(dbias, dw_type, col, s);
    }
}

// Operands whose rows begin at odd addresses, laid out anew: rows x cols values at src to rows of `ldd` values, zeros
// behind the last one. Two operands by one launch, 8 values a thread.
struct Layout {
    const uint16_t* src;
    uint16_t* dst;
    long long rows, cols, ld, ldd;
};
__global__ void __launch_bounds__(256) lay_out_kernel(Layout a, Layout b, long long pieces_a, long long pieces_b) {
    long long i = 256 * (blockIdx.x + (long long)gridDim.x * blockIdx.y) + threadIdx.x;
    const bool first = i < pieces_a;
    if (!first) i -= pieces_a;
    if (!first && i >= pieces_b) return;
    const Layout& l = first ? a : b;
    const long long across = l.ldd / 8, row = i / across, col = 8 * (i % across);
    const uint16_t* from = l.src + row * l.ld + col;
    union {
        uint16_t v[8];
        u32x4 w;
    } x;
    if (col + 8 <= l.cols) {
        x.w = get16<u32x4>(from);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) x.v[k] = col + k < l.cols ? from[k] : 0;
    }
    *reinterpret_cast<u32x4*>(l.dst + row * l.ldd + col) = x.w;
}

// A grid of at least `groups` workgroups of 256 threads: along x 2^31 threads, the rest along y. The kernels go by
// blockIdx.x + gridDim.x blockIdx.y and leave what is too much.
dim3 grid_of(long long groups) {
    const long long x = std::min(groups, 1ll << 23);
    return dim3((unsigned)x, (unsigned)((groups + x - 1) / x));
}
constexpr long long kMaxGroups = (1ll << 24) - 1;  // workgroups of 256 threads along x

// Whether rows begin at multiples of 4 bytes, as the tiles' copies need them.
bool even_rows(const void* p, long long ld) { return !((uintptr_t)p & 3) && ld % 2 == 0; }

size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

constexpr int kFewRows = 16, kFewOddRows = 32;  // rows that begin at odd addresses: laid out for the tiles from 33 on

// Estimated us of a tile's launch with its c cut into `splits` ranges: whole rounds of workgroups over the CUs and the last,
// partly filled one, not less than the operands take from memory (4.6 TB/s), and the join's launch and traffic (8 bytes an
// output and range at 4 TB/s).
float estimate(const Shape& t, int cus, long long nq, long long np, long long C, int splits) {
    const long long tiles = tiles_of(t, nq, np, splits), slots = (long long)cus * t.per_cu;
    const float stages = (float)(((C + 63) / 64 + splits - 1) / splits);
    const long long rest = tiles % slots;
    float us = (float)(tiles / slots) * (t.fixed + stages * t.full);
    if (rest) us += t.fixed + stages * (rest <= cus ? t.alone : t.full);
    us = std::max(us, t.fixed + 2.0f * ((float)nq + (float)np) * (float)C / 4.6e6f);
    if (splits > 1) us += 3.0f + (float)splits * (float)nq * (float)np * 8.0f / 4e6f;
    return us;
}

}  // namespace

// Few rows: their own kernels, c in ranges where 16 rows of W each are too few to keep the CUs reading (at least 512 values a
// range). 5 rows, 512 of W, K = 8192: 8.0 us in four ranges, 9.1 in one.
// More: the tile and ranges with the least estimate; 1000 x 704 x 1504 10.1 us by 64 x 64 (17 by 128 x 128), 2048 x 4096 x 4096 62
// by 128 x 128 (70 by 256 x 256 in two ranges, 98 by 64 x 64), 256 x 1024 x 8192 15.5 by 64 x 64 in 4 ranges (38 in one), 3500^3 88 by
// 256 x 256 (120 by 128 x 128), 8192^2 of K = 512 101 by 128 x 128 (124 by 256 x 256). Measured against all other tiles and numbers
// of ranges at 52 sizes, the choice is the fastest or up to 9% slower at 50 of them with operands in the caches and at 46 without.
// It is further off where c is long and tiles are few, as the estimate takes their stages for shorter than they are: without caches
// 512 x 8192^2 96 us for 81 by 256 x 256 in 4 ranges, 256 x 8192^2 73 (estimate: 45) for 64 by 128 x 128 in 4, and of few rows 16 x
// 8192^2 36 for 30 by 32 x 32.
ozl::Route ozl::route_of(int cus, long long nq, long long np, long long C, bool contiguous, bool even, int streamed) {
    Route r{};
    r.splits = 1;
    if (contiguous && (nq <= kFewRows || (!even && nq <= kFewOddRows))) {
        r.few = true;
        const long long groups = (np + few_rows_block(nq) - 1) / few_rows_block(nq);
        while (nq > streamed && r.splits < 16 && groups * r.splits * 4 <= cus && C / (r.splits * 2) >= 512) r.splits *= 2;
    } else {
        float best = 0.0f;
        for (int t = 0; t < TILES; t++)
            for (int s = 1; s <= 16; s *= 2) {
                if ((s > 1 && (C + 63) / 64 / s < 4) || !fits(shape_of((Tile)t), nq, np, s)) break;
                const float us = estimate(shape_of((Tile)t), cus, nq, np, C, s);
                if (best == 0.0f || us < best) best = us, r.tile = (Tile)t, r.splits = s;
            }
    }
    if (r.splits > 1) r.parts = up(4 * (size_t)r.splits * nq * ((np + 7) / 8 * 8));
    return r;
}

namespace {

int launch_any(oz_dev* dev, int type, const Product& a) {
    const dim3 grid = grid_of((long long)oz::ceil_div(a.np, 64) * oz::ceil_div(a.nq, 64));
    if (type == OZ_BF16) hipLaunchKernelGGL(product_any_kernel<OZ_BF16>, grid, dim3(256), 0, dev->stream, a);
    else hipLaunchKernelGGL(product_any_kernel<OZ_F16>, grid, dim3(256), 0, dev->stream, a);
    return oz::launch_check(dev, "product_any_kernel");
}

// Bytes of an operand's copy of whole rows: n rows along c, or C rows along n.
size_t copy_bytes(long long n, long long C, bool major) { return up(2 * (size_t)(major ? C : n) * (((major ? n : C) + 7) / 8 * 8)); }

// Workspace of a product whose operands need copies or not.
size_t product_bytes(int cus, long long nq, long long np, long long C, bool q_major, bool p_major, bool copy_q, bool copy_p) {
    if (!nq || !np || !C) return 0;
    const Route r = route_of(cus, nq, np, C, !q_major && !p_major, !copy_q && !copy_p);
    if (r.few) return r.parts;
    return r.parts + (copy_q ? copy_bytes(nq, C, q_major) : 0) + (copy_p ? copy_bytes(np, C, p_major) : 0);
}

// The same where operands may need copies (their addresses are said to be odd), enough whether they turn out to or not.
size_t reserve(int cus, long long nq, long long np, long long C, bool q_major, bool p_major, bool copy_q, bool copy_p, bool may_q, bool may_p) {
    return std::max(product_bytes(cus, nq, np, C, q_major, p_major, copy_q, copy_p),
                    product_bytes(cus, nq, np, C, q_major, p_major, copy_q || may_q, copy_p || may_p));
}

// Runs a product in `bytes` bytes of workspace. Operands whose rows begin at odd addresses are laid out in it; where that has no room
// (an operand at an odd address of which the descriptor does not say so) few rows take one range, and of more the element by
// element kernel runs.
int launch_product(oz_dev* dev, int type, Product a, void* work, size_t bytes) {
    if (!a.nq || !a.np) return OZ_OK;
    a.splits = 1;
    if (!a.C) return launch_any(dev, type, a);
    const bool copy_q = !even_rows(a.Q, a.ldq), copy_p = !even_rows(a.P, a.ldp);
    Route r = route_of(dev->cus, a.nq, a.np, a.C, !a.q_major && !a.p_major, !copy_q && !copy_p);
    const size_t need = product_bytes(dev->cus, a.nq, a.np, a.C, a.q_major, a.p_major, copy_q, copy_p);
    if (need > bytes) {
        if (!r.few) return launch_any(dev, type, a);
        r.splits = 1, r.parts = 0;
    }
    char* at = static_cast<char*>(work);
    a.splits = r.splits;
    a.parts = reinterpret_cast<float*>(at);
    a.ldparts = (a.np + 7) / 8 * 8;
    at += r.parts;
    if (r.few) return launch_few_rows(dev, type, a);
    if (!fits(shape_of(r.tile), a.nq, a.np, r.splits)) return oz::fail(dev, OZ_ERR_ARG, "a product of %lld x %lld outputs is too large", a.nq, a.np);
    if (copy_q || copy_p) {
        Layout l[2] = {};
        long long pieces[2] = {};
        auto lay = [&](const void*& p, long long& ld, long long n, bool major, int i) {
            const long long rows = major ? a.C : n, cols = major ? n : a.C, ldd = (cols + 7) / 8 * 8;
            l[i] = Layout{static_cast<const uint16_t*>(p), reinterpret_cast<uint16_t*>(at), rows, cols, ld, ldd};
            pieces[i] = rows * (ldd / 8);
            p = at;
            ld = ldd;
            at += copy_bytes(n, a.C, major);
        };
        if (copy_q) lay(a.Q, a.ldq, a.nq, a.q_major, 0);
        if (copy_p) lay(a.P, a.ldp, a.np, a.p_major, 1);
        hipLaunchKernelGGL(lay_out_kernel, grid_of((pieces[0] + pieces[1] + 255) / 256), dim3(256), 0, dev->stream, l[0], l[1], pieces[0], pieces[1]);
        if (int st = oz::launch_check(dev, "lay_out_kernel")) return st;
    }
    return launch_tile(dev, type, r.tile, a);
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
    if (d->odd & ~(OZ_ODD_X | OZ_ODD_W)) return "odd operands";
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
    if (d->odd & ~(OZ_ODD_X | OZ_ODD_W | OZ_ODD_DY)) return "odd operands";
    return nullptr;
}

bool misaligned16(const void* p) { return ((uintptr_t)p & 15) != 0; }
bool misaligned(const void* p, int type) { return ((uintptr_t)p & (size_of(type) - 1)) != 0; }

// Workspace of the gradients: dZ where it is not dY (or dY's rows are not even), what its rounding leaves where dW takes that too,
// the columns' sums, and the larger of the products' own.
struct GradWork {
    bool make_dz;
    bool two;          // dZ in two parts of `part` bytes: ReLU's is dY or 0, exact in one
    long long lddz;
    int lanes;         // act_grad_kernel's
    int rows, chunks;  // of M for the columns' sums
    size_t part, dz, sums, product, bytes;
};
GradWork grad_work(int cus, const oz_linear_grad_desc* d, bool even_dy) {
    GradWork w{};
    w.make_dz = d->act != OZ_ACT_NONE || !even_dy;
    w.lddz = (d->N + 7) / 8 * 8;
    w.two = d->dw_type == OZ_F32 && (d->act == OZ_ACT_GELU || d->act == OZ_ACT_SILU);
    w.part = up(2 * (size_t)d->M * w.lddz);
    w.dz = w.make_dz ? (1 + w.two) * w.part : 0;
    // Strips of 256 columns, 64 of few values, and of the rows so many that the chip is filled four times, 16 to 256 at a time.
    w.lanes = (long long)d->M * d->N <= 1 << 22 ? 8 : 32;
    const long long strips = (d->N + 8 * w.lanes - 1) / (8 * w.lanes), rows = (long long)d->M * strips / (4 * cus), least = 512 / w.lanes;
    w.rows = (int)std::min(256ll, std::max(least, (rows + least - 1) / least * least));
    w.chunks = (int)std::max(1ll, ((long long)d->M + w.rows - 1) / w.rows);
    w.sums = up(4 * (size_t)w.chunks * d->N);
    w.product = std::max(reserve(cus, d->M, d->K, d->N, false, true, false, or_row(d->ldw, d->K) % 2 != 0, false, d->odd & OZ_ODD_W),
                         reserve(cus, d->N, d->K, d->M, true, true, false, or_row(d->ldx, d->K) % 2 != 0, false, d->odd & OZ_ODD_X));
    w.bytes = w.dz + w.sums + w.product;
    return w;
}

// Whether dY's rows begin at even addresses, as the descriptor says it.
bool even_dy(const oz_linear_grad_desc* d) { return or_row(d->lddy, d->N) % 2 == 0 && !(d->odd & OZ_ODD_DY); }

int cus_of(const oz_dev* dev) { return dev && dev->cus > 0 ? dev->cus : 256; }

}  // namespace

extern "C" {

long long oz_linear_workspace(oz_dev* dev, const oz_linear_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear: %s", e);
    return (long long)reserve(cus_of(dev), d->M, d->N, d->K, false, false, or_row(d->ldx, d->K) % 2 != 0, or_row(d->ldw, d->K) % 2 != 0,
                              d->odd & OZ_ODD_X, d->odd & OZ_ODD_W);
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
    if (misaligned16(work)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear: workspace not 16-byte aligned");
    const size_t need = (size_t)oz_linear_workspace(dev, d);
    if (need && (!work || bytes < need)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear: workspace of %zu bytes, %zu needed", bytes, need);
    ozl::Product p{};
    p.Q = X, p.P = W, p.nq = d->M, p.np = d->N, p.C = d->K, p.ldq = or_row(d->ldx, d->K), p.ldp = or_row(d->ldw, d->K);
    p.epi = {Y, or_row(d->ldy, d->N), d->y_type, Z, or_row(d->ldz, d->N), bias, residual, or_row(d->ldr, d->N), d->act};
    return launch_product(dev, d->type, p, work, work ? bytes : 0);
}

long long oz_linear_grad_workspace(oz_dev* dev, const oz_linear_grad_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: %s", e);
    return (long long)grad_work(cus_of(dev), d, even_dy(d)).bytes;
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
    const size_t least = grad_work(cus_of(dev), d, even_dy(d)).bytes;
    if (!work || bytes < least || misaligned16(work))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, least);
    if (int st = oz::use(dev)) return st;
    const long long lddy = or_row(d->lddy, d->N), ldz = or_row(d->ldz, d->N);
    GradWork w = grad_work(cus_of(dev), d, even_rows(dY, lddy));
    if (w.bytes > bytes) w.make_dz = false, w.dz = 0;  // dY at an odd address without room for a copy
    char* at = static_cast<char*>(work);
    const void* dz = dY;
    long long lddz = lddy;
    const bool products = d->M > 0 && (dX || dW);
    if ((w.make_dz && products) || dbias) {
        void* make = w.make_dz && products ? at : nullptr;
        if (make) dz = make, lddz = w.lddz;
        void* rest = make && w.two && dW ? at + w.part : nullptr;
        float* sums = dbias ? reinterpret_cast<float*>(at + w.dz) : nullptr;
        const int strips = (int)oz::ceil_div(d->N, 8 * w.lanes), chunks = d->M ? w.chunks : 0;
        if ((long long)strips * w.chunks > kMaxGroups) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_grad: %d x %d outputs are too many", d->M, d->N);
        const bool one = chunks == 1;
        if (chunks) {
            const dim3 grid((unsigned)(strips * chunks));
            const auto kernel = w.lanes == 8 ? act_grad_of<8>(d->act, rest) : act_grad_of<32>(d->act, rest);
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, dev->stream, dY, Z, make, rest, one ? nullptr : sums,
                               one ? dbias : nullptr, d->type, d->dw_type, d->accumulate, (long long)d->M, d->N, lddy, ldz, w.lddz, w.rows, strips);
            if (int st = oz::launch_check(dev, "act_grad_kernel")) return st;
        }
        if (dbias && !one) {
            hipLaunchKernelGGL(bias_grad_kernel, dim3(oz::ceil_div(d->N, 16)), dim3(256), 0, dev->stream, sums, dbias, d->dw_type,
                               d->accumulate, chunks, d->N);
            if (int st = oz::launch_check(dev, "bias_grad_kernel")) return st;
        }
    }
    char* room = at + w.dz + w.sums;
    const size_t left = bytes - w.dz - w.sums;
    if (dX && d->M > 0) {
        ozl::Product p{};
        p.Q = dz, p.P = W, p.nq = d->M, p.np = d->K, p.C = d->N, p.ldq = lddz, p.ldp = or_row(d->ldw, d->K), p.p_major = 1;
        p.epi = {dX, or_row(d->lddx, d->K), d->type, nullptr, 0, nullptr, nullptr, 0, OZ_ACT_NONE};
        if (int st = launch_product(dev, d->type, p, room, left)) return st;
    }
    if (dW) {
        ozl::Product p{};
        p.Q = dz, p.P = X, p.nq = d->N, p.np = d->K, p.C = d->M, p.ldq = lddz, p.ldp = or_row(d->ldx, d->K), p.q_major = p.p_major = 1;
        p.epi = {dW, or_row(d->lddw, d->K), d->dw_type, nullptr, 0, nullptr, d->accumulate ? dW : nullptr, or_row(d->lddw, d->K), OZ_ACT_NONE};
        if (w.two && d->M > 0) {  // the smaller part's product first, the other's added to it
            ozl::Product r = p;
            r.Q = at + w.part;
            if (int st = launch_product(dev, d->type, r, room, left)) return st;
            p.epi.residual = dW;
        }
        if (int st = launch_product(dev, d->type, p, room, left)) return st;
    }
    return OZ_OK;
}

}  // extern "C"

// The route of a product of nq x np outputs over C, for tests: -1 for the kernels of few rows, else the tile; *splits its ranges of c.
extern "C" int oz_rule_linear_route(int cus, long long nq, long long np, long long C, int contiguous, int even, int* splits) {
    const Route r = route_of(cus, nq, np, C, contiguous != 0, even != 0);
    if (splits) *splits = r.splits;
    return r.few ? -1 : (int)r.tile;
}
