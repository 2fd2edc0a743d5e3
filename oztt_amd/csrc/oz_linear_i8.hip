// Product of 8-bit integers with bias, activation and residual (include/oz_hip.h, oz_linear_i8).
//
//   Y = act(w_scale_n x_scale_m sum_k Xq_mk Wq_nk + bias_n) + residual
//
// The tiles are the linear layers' (oz_linear_tiles.hpp): a stage's 128 bytes of a row are 128 integers in place of 64 values, and the
// matrix instruction of 16 x 16 x 64 integers takes a lane's 16 bytes as the one of 16 x 16 x 32 values does, so everything
// but the epilogue's scales is the same at twice the rate, the choice of a tile included. The sums are int32 and exact, so ranges of k
// and waves join them in any order.
#include "oz_internal.hpp"
#include "oz_linear_tiles.hpp"
#include "oz_quantize.hpp"

#include <algorithm>

namespace {

using namespace ozt;
using namespace ozl;

constexpr int WAVES = 8;

// ---- tiles ------------------------------------------------------------------------------------------

// Rows of X that the call quantized end in zeros; a caller's end in what is there, which is cleared in LDS. What stands behind W's
// rows is multiplied by those zeros.
__device__ __forceinline__ int ragged_tail(const ScaledProduct& a, int split) { return split == a.splits - 1 && !a.q_zeros ? a.K % (2 * BC) : 0; }

template <int TYPE, int TI, int TJ, int WQ, int WP, int NSTG>
__global__ void __launch_bounds__(64 * WQ * WP, NSTG * 16 * BC * 2 * (TI * WQ + TJ * WP) <= 81920 ? 2 : 1)
    scaled_tile_kernel(const ScaledProduct a, int tiles_q, int tiles_p) {
    typedef TileLoop<Int8, false, false, TI, TJ, WQ, WP, NSTG> Loop;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Loop::LDS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work w = work_of(a, tiles_q, tiles_p, Loop::QR, Loop::PR);
    typename Loop::OQ oq;
    typename Loop::OP op;
    oq.init(a.Q, a.ldq, a.nq, a.C, w.q0, w.c0, w.nst, lane, wave);
    op.init(a.P, a.ldp, a.np, a.C, w.p0, w.c0, w.nst, lane, wave);
    i32x4 acc[TI][TJ];
    Loop::template run<int8_t>(lds, oq, op, w.nst, ragged_tail(a, w.split), lane, wave, acc);
    put_sums<TYPE, TI, TJ, Loop::ROOM>(a, acc, reinterpret_cast<float*>(lds) + wave * Loop::ROOM, lane, w.split, w.q0 + 16 * (wave / WP) * TI,
                                       w.p0 + 16 * (wave % WP) * TJ);
}

template <int TYPE>
__global__ void __launch_bounds__(256) scaled_big_kernel(const ScaledProduct a, int tiles_q, int tiles_p) {
    typedef BigLoop<Int8, false, false> Loop;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Loop::LDS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work w = work_of(a, tiles_q, tiles_p, 256, 256);
    typename Loop::OQ oq;
    typename Loop::OP op;
    oq.init(a.Q, a.ldq, a.nq, a.C, w.q0, w.c0, w.nst, lane, wave);
    op.init(a.P, a.ldp, a.np, a.C, w.p0, w.c0, w.nst, lane, wave);
    i32x4 acc[8][8];
    Loop::template run<int8_t>(lds, oq, op, w.nst, ragged_tail(a, w.split), lane, wave, acc);
    put_sums<TYPE, 8, 8, Loop::ROOM>(a, acc, reinterpret_cast<float*>(lds) + wave * Loop::ROOM, lane, w.split, w.q0 + 128 * (wave >> 1), w.p0 + 128 * (wave & 1));
}

// Joins the ranges' int32 sums.
template <int TYPE>
__global__ void __launch_bounds__(256) scaled_join_kernel(const ScaledProduct a) {
    const long long across = (a.np + 7) / 8, i = 256ll * blockIdx.x + threadIdx.x;
    const long long q = i / across, p = 8 * (i % across);
    if (q >= a.nq) return;
    float v[8], x[8];
    load8(a.parts, OZ_F32, q * a.ldparts + p, v);
#pragma unroll 8
    for (int s = 1; s < a.splits; s++) {
        load8(a.parts, OZ_F32, (s * a.nq + q) * a.ldparts + p, x);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = __int_as_float(__float_as_int(v[k]) + __float_as_int(x[k]));
    }
    scale8(a, q, p, v);
    finish8<TYPE>(a.epi, a.np, q, p, v);
}

int launch_join(oz_dev* dev, const ScaledProduct& a) {
    if (a.splits == 1) return OZ_OK;
    const dim3 grid(oz::ceil_div(a.nq * ((a.np + 7) / 8), 256)), block(256);
    if (a.type == OZ_BF16) hipLaunchKernelGGL(scaled_join_kernel<OZ_BF16>, grid, block, 0, dev->stream, a);
    else hipLaunchKernelGGL(scaled_join_kernel<OZ_F16>, grid, block, 0, dev->stream, a);
    return oz::launch_check(dev, "scaled_join_kernel");
}

template <int TYPE, int TI, int TJ, int WQ, int WP, int NSTG>
void launch_tiles(oz_dev* dev, const ScaledProduct& a) {
    const int tiles_q = (int)oz::ceil_div(a.nq, 16 * TI * WQ), tiles_p = (int)oz::ceil_div(a.np, 16 * TJ * WP);
    hipLaunchKernelGGL((scaled_tile_kernel<TYPE, TI, TJ, WQ, WP, NSTG>), dim3((unsigned)tiles_q * tiles_p * a.splits), dim3(64 * WQ * WP), 0, dev->stream, a,
                       tiles_q, tiles_p);
}

template <int TYPE>
int by_tile(oz_dev* dev, Tile t, const ScaledProduct& a) {
    switch (t) {
        case T256: {
            const int tiles_q = (int)oz::ceil_div(a.nq, 256), tiles_p = (int)oz::ceil_div(a.np, 256);
            hipLaunchKernelGGL(scaled_big_kernel<TYPE>, dim3((unsigned)tiles_q * tiles_p * a.splits), dim3(256), 0, dev->stream, a, tiles_q, tiles_p);
            break;
        }
        case T128: launch_tiles<TYPE, 2, 4, 4, 2, 2>(dev, a); break;
        case T64: launch_tiles<TYPE, 2, 2, 2, 2, 4>(dev, a); break;
        case T64X32: launch_tiles<TYPE, 2, 2, 2, 1, 6>(dev, a); break;
        default: launch_tiles<TYPE, 1, 2, 2, 1, 8>(dev, a); break;
    }
    if (int st = oz::launch_check(dev, "scaled_tile_kernel")) return st;
    return launch_join(dev, a);
}

// ---- few rows of X ----------------------------------------------------------------------------------

// The 16 bytes of a row from k on, of those in front of K; whole words are read (rows begin at multiples of 4 bytes, so a row's last
// word is its own). MASK: nothing behind K is in them.
template <bool MASK>
__device__ __forceinline__ i32x4 guarded16(const int8_t* row, int k, int K) {
    i32x4 v;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const int left = K - k - 4 * w;
        int x = left > 0 ? *reinterpret_cast<const int*>(row + k + 4 * w) : 0;
        if (MASK && left > 0 && left < 4) x &= (1 << (8 * left)) - 1;
        v[w] = x;
    }
    return v;
}

// Up to 16 rows of X, 16 of W a workgroup: the waves stream W straight into registers as one operand of the matrix instructions, 256
// bytes of a row at a time, and read the rows of X, which all workgroups share, from the L2. k is dealt out to the 8 waves,
// whose sums are joined in LDS. Few rows of W: ranges of k go to several workgroups, joined by a second launch.
__global__ void __launch_bounds__(64 * WAVES, 4) scaled_few_rows_kernel(const ScaledProduct a, int blocks_p) {
    constexpr int F = 4, UNIT = 64 * F;
    __shared__ i32x4 sums[WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.x / blocks_p;
    const long long p0 = 16ll * (blockIdx.x - split * blocks_p);
    const int r = lane & 15, g = lane >> 4;
    // rows beyond an operand's last are its last one again; their sums are not used
    const int8_t* pw = static_cast<const int8_t*>(a.P) + (p0 + r < a.np ? p0 + r : a.np - 1) * 2 * a.ldp;
    const int8_t* px = static_cast<const int8_t*>(a.Q) + (r < a.nq ? r : a.nq - 1) * 2 * a.ldq;
    const int units = a.K / UNIT, u0 = (int)((long long)units * split / a.splits), u1 = (int)((long long)units * (split + 1) / a.splits);
    i32x4 acc = {0, 0, 0, 0};
    i32x4 w[2][F], x[2][F];
    auto ask = [&](int b, int u) {
        if (u < u1) {
#pragma unroll
            for (int f = 0; f < F; f++) w[b][f] = get16<i32x4>(pw + (long long)u * UNIT + 64 * f + 16 * g);
#pragma unroll
            for (int f = 0; f < F; f++) x[b][f] = get16<i32x4>(px + (long long)u * UNIT + 64 * f + 16 * g);
        }
    };
    auto multiply = [&](int b) {
#pragma unroll
        for (int f = 0; f < F; f++) acc = Int8::mfma(w[b][f], x[b][f], acc);
    };
    int u = u0 + wave;
    ask(0, u);
    for (; u < u1; u += 2 * WAVES) {
        ask(1, u + WAVES);
        multiply(0);
        ask(0, u + 2 * WAVES);
        if (u + WAVES < u1) multiply(1);
    }
    if (split == a.splits - 1 && wave == WAVES - 1)
        for (int k = units * UNIT; k < a.K; k += 64)
            acc = Int8::mfma(guarded16<false>(pw, k + 16 * g, a.K), guarded16<true>(px, k + 16 * g, a.K), acc);
    sums[wave][lane] = acc;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    // 16 values of p a row, next to each other
    const int i = threadIdx.x % 16, q = threadIdx.x / 16;
    if (q >= a.nq || p0 + i >= a.np) return;
    int v = 0;
#pragma unroll
    for (int s = 0; s < WAVES; s++) v += sums[s][16 * (i / 4) + q][i % 4];
    if (a.splits > 1) a.parts[(split * a.nq + q) * a.ldparts + p0 + i] = __int_as_float(v);
    else finish(a.epi, a.type, q, p0 + i, (float)v * a.p_scale[p0 + i] * a.q_scale[q]);
}

// One or two rows of X, values or integers: a wave streams rows of W, 4 KB at a time and two such ahead, and multiplies on the vector units, four products an
// instruction. X is quantized by every workgroup for itself into LDS, while the first 8 KB of its waves' rows are on
// the way: a launch of its own in front would cost more than that. Few rows of W: KS waves share a row's k.
constexpr int kStreamK = 16384;  // X in LDS, by each workgroup
struct Tokens {
    const void* X;  // values of `type`, or integers with scales
    long long ldx;
    int type;
    bool int8;
};
template <int M>
constexpr int kStreamGroups = M == 1 ? 4 : 3;  // of a CU, as registers allow: their first reads are all of 8192 x 8192 weights
template <int M, int TYPE, bool INT8>
__global__ void __launch_bounds__(64 * WAVES, 2 * kStreamGroups<M>) scaled_stream_kernel(const ScaledProduct a, const Tokens t, int ks) {
    constexpr int U = 4, THREADS = 64 * WAVES, V = 8;
    extern __shared__ __attribute__((aligned(16))) int8_t xs[];  // M rows of whole KB, zeros behind K
    __shared__ unsigned tops[WAVES][M];
    __shared__ int sums[WAVES][M];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave % ks, rows = WAVES / ks, kbs = (a.K + 1023) / 1024, width = 1024 * kbs;
    const int groups = (kbs + U * ks - 1) / (U * ks);  // of U pieces of a KB, dealt out to the waves of a row
    const int turns = (int)((a.np + rows - 1) / rows);
    auto row_of = [&](int turn) {
        const long long p = (long long)turn * rows + wave / ks;
        return static_cast<const int8_t*>(a.P) + (p < a.np ? p : a.np - 1) * 2 * a.ldp;
    };
    i32x4 w[2][U];
    auto ask = [&](int b, const int8_t* row, int group) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = 1024 * ((group * U + u) * ks + part);
            if (k + 1024 <= a.K) w[b][u] = get16<i32x4>(row + k + 16 * lane);
            else w[b][u] = guarded16<false>(row, k + 16 * lane, a.K);
        }
    };
    // the group to ask for next, of this row or a next one's first
    int next_turn = blockIdx.x, next_group = 0;
    const int8_t* next_row = row_of(next_turn);
    auto ask_next = [&](int b) {
        if (next_turn >= turns) return;
        ask(b, next_row, next_group);
        if (++next_group == groups) {
            next_group = 0;
            next_turn += gridDim.x;
            next_row = row_of(next_turn);
        }
    };
    ask_next(0);
    ask_next(1);
    float scale[M];
    if constexpr (INT8) {
#pragma unroll
        for (int m = 0; m < M; m++) {
            const int8_t* x = static_cast<const int8_t*>(t.X) + m * t.ldx;
            for (int k = 16 * threadIdx.x; k < width; k += 16 * THREADS) *reinterpret_cast<i32x4*>(xs + m * width + k) = guarded16<true>(x, k, a.K);
            scale[m] = a.q_scale[m];
        }
    } else {
        // X is read twice, from memory and out of the caches: kept, it would take the registers of a fourth workgroup
        auto get = [&](int m, int k, float* v) {
            if (k + V <= a.K) load8(t.X, TYPE, m * t.ldx + k, v);
            else load_some(t.X, TYPE, m * t.ldx + k, max(a.K - k, 0), v);
        };
        unsigned top[M] = {};
#pragma unroll
        for (int m = 0; m < M; m++) {
#pragma unroll 2
            for (int k = V * threadIdx.x; k < a.K; k += V * THREADS) {
                float v[V];
                get(m, k, v);
#pragma unroll
                for (int e = 0; e < V; e++) top[m] = max(top[m], ozq::bits_of(v[e]));
            }
#pragma unroll
            for (int d = 32; d > 0; d /= 2) top[m] = max(top[m], (unsigned)__shfl_xor(top[m], d));
            if (lane == 0) tops[wave][m] = top[m];
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < M; m++) {
#pragma unroll
            for (int s = 0; s < WAVES; s++) top[m] = max(top[m], tops[s][m]);
            const ozq::Scale s = ozq::scale_of(top[m]);
            scale[m] = s.scale;
#pragma unroll 2
            for (int k = V * threadIdx.x; k < width; k += V * THREADS) {
                float v[V];
                get(m, k, v);
                *reinterpret_cast<u32x2*>(xs + m * width + k) = u32x2{ozq::pack4(v, s.inverse), ozq::pack4(v + 4, s.inverse)};
            }
        }
    }
    __syncthreads();
    int acc[M] = {};
    auto add = [&](int b, int group) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int piece = (group * U + u) * ks + part;
            if (piece >= kbs) continue;
#pragma unroll
            for (int m = 0; m < M; m++) {
                const i32x4 x = *reinterpret_cast<const i32x4*>(xs + m * width + 1024 * piece + 16 * lane);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[m] = __builtin_amdgcn_sdot4(w[b][u][e], x[e], acc[m], false);
            }
        }
    };
    auto put = [&](long long p, int m, int v) {
        if (p < a.np) finish(a.epi, a.type, m, p, (float)v * a.p_scale[p] * scale[m]);
    };
    int turn = blockIdx.x, group = 0;
    auto one = [&](auto B) {
        constexpr int b = decltype(B)::value;
        add(b, group);
        ask_next(b);
        if (++group == groups) {  // the row's last group
#pragma unroll
            for (int m = 0; m < M; m++) {
#pragma unroll
                for (int d = 32; d > 0; d /= 2) acc[m] += __shfl_xor(acc[m], d);
            }
            if (ks == 1) {
#pragma unroll
                for (int m = 0; m < M; m++)
                    if (lane == m) put((long long)turn * rows + wave, m, acc[m]);
            } else {  // a workgroup has one turn
                if (lane == 0)
#pragma unroll
                    for (int m = 0; m < M; m++) sums[wave][m] = acc[m];
                __syncthreads();
#pragma unroll
                for (int m = 0; m < M; m++)
                    if ((int)threadIdx.x < rows) {
                        int v = 0;
                        for (int k = 0; k < ks; k++) v += sums[threadIdx.x * ks + k][m];
                        put((long long)turn * rows + threadIdx.x, m, v);
                    }
            }
#pragma unroll
            for (int m = 0; m < M; m++) acc[m] = 0;
            turn += gridDim.x, group = 0;
        }
    };
    while (turn < turns) {
        one(std::integral_constant<int, 0>{});
        if (turn < turns) one(std::integral_constant<int, 1>{});
    }
}

// Waves that share a row: so many that the chip has 16 on each CU, as long as each has something to read.
int waves_of_a_row(int cus, long long np, int K) {
    int ks = 1;
    while (ks < WAVES && np * ks < 16ll * cus && ks * 4096 < K) ks *= 2;
    return ks;
}

template <int M, int TYPE, bool INT8>
int launch_stream(oz_dev* dev, const ScaledProduct& a, const Tokens& t) {
    const int ks = waves_of_a_row(dev->cus, a.np, a.K), rows = WAVES / ks;
    const long long turns = (a.np + rows - 1) / rows, grid = ks > 1 ? turns : std::min<long long>(turns, kStreamGroups<M> * dev->cus);
    hipLaunchKernelGGL((scaled_stream_kernel<M, TYPE, INT8>), dim3((unsigned)grid), dim3(64 * WAVES), M * ((a.K + 1023) / 1024 * 1024), dev->stream, a, t, ks);
    return oz::launch_check(dev, "scaled_stream_kernel");
}

int launch_few_rows(oz_dev* dev, const ScaledProduct& a) {
    const int blocks_p = (int)oz::ceil_div(a.np, 16);
    hipLaunchKernelGGL(scaled_few_rows_kernel, dim3((unsigned)blocks_p * a.splits), dim3(64 * WAVES), 0, dev->stream, a, blocks_p);
    if (int st = oz::launch_check(dev, "scaled_few_rows_kernel")) return st;
    return launch_join(dev, a);
}

// ---- calls ------------------------------------------------------------------------------------------

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

// Few rows by the kernel of few rows: with integers for X 8 x 2048 x 2048 4.2 us (5.8 in tiles), 16 x 512 x 8192 8.5 (10.7), 4 x 4096 x 16384 15.4
// (17.3), 4 x 8192 x 8192 13.9 (14.1). Tiles read X once for more rows of W, and long rows in more ranges: 16 x 8192 x 8192 14.1 us (17.9), 8 x
// 8192 x 8192 14.2 (15.4), 3 x 1024 x 131000 30 (46).
bool few_rows(int M, int N, int K) { return K <= 32768 && (M <= 4 || N <= 4096); }

// How a call runs, and its workspace: the integers of X in rows of whole stages, their scales, the ranges' sums.
struct Plan {
    bool stream;
    Route route;
    int width;
    size_t x, scale;
    size_t bytes() const { return x + scale + route.parts; }
};
Plan plan_of(int cus, const oz_linear_i8_desc* d) {
    Plan p{};
    p.stream = d->M <= kStreamRows && d->K <= kStreamK;
    if (p.stream || !d->M) return p;
    // one and two rows too long to be streamed are cut into ranges as others are: 1 x 64 x 32768 9.4 us in 16 (19.7 in one), 1 x 1024 x
    // 28672 13.2 in 2 (17.7)
    p.route = route_of(cus, d->M, d->N, (d->K + 1) / 2, few_rows(d->M, d->N, d->K), true, 0);
    p.width = (d->K + 2 * BC - 1) / (2 * BC) * (2 * BC);
    if (!d->x_int8) p.x = up((size_t)d->M * p.width), p.scale = up(4 * (size_t)d->M);
    return p;
}

int cus_of(const oz_dev* dev) { return dev && dev->cus > 0 ? dev->cus : 256; }

template <int M, int TYPE>
int stream(oz_dev* dev, const ScaledProduct& a, const Tokens& t) {
    return t.int8 ? launch_stream<M, TYPE, true>(dev, a, t) : launch_stream<M, TYPE, false>(dev, a, t);
}

}  // namespace

extern "C" {

long long oz_linear_i8_workspace(oz_dev* dev, const oz_linear_i8_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: %s", e);
    return (long long)plan_of(cus_of(dev), d).bytes();
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
    if (int st = oz::use(dev)) return st;
    if (d->M == 0) return OZ_OK;
    const Plan plan = plan_of(cus_of(dev), d);
    const size_t need = plan.bytes();
    if (need && (!work || bytes < need || misaligned(work, 16)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
    if (!plan.stream && !plan.route.few && !fits(shape_of(plan.route.tile), d->M, d->N, plan.route.splits))
        return oz::fail(dev, OZ_ERR_ARG, "oz_linear_i8: a product of %d x %d outputs is too large", d->M, d->N);
    const long long ldx = or_row(d->ldx, d->K);
    ScaledProduct a{};
    a.Q = X, a.P = W, a.q_scale = x_scale, a.p_scale = w_scale;
    a.nq = d->M, a.np = d->N, a.K = d->K, a.C = (d->K + 1) / 2, a.ldq = ldx / 2, a.ldp = or_row(d->ldw, d->K) / 2, a.type = d->type;
    a.splits = std::max(plan.route.splits, 1);
    a.epi = {Y, or_row(d->ldy, d->N), d->y_type, nullptr, 0, bias, residual, or_row(d->ldr, d->N), d->act};
    if (plan.stream) {
        const Tokens t{X, ldx, d->type, d->x_int8 != 0};
        if (d->M == 1) return d->type == OZ_BF16 ? stream<1, OZ_BF16>(dev, a, t) : stream<1, OZ_F16>(dev, a, t);
        return d->type == OZ_BF16 ? stream<2, OZ_BF16>(dev, a, t) : stream<2, OZ_F16>(dev, a, t);
    }
    char* at = static_cast<char*>(work);
    if (!d->x_int8) {
        int8_t* q = reinterpret_cast<int8_t*>(at);
        float* scale = reinterpret_cast<float*>(at + plan.x);
        if (int st = ozq::launch_quantize(dev, d->type, d->M, d->K, X, ldx, q, plan.width, plan.width, scale)) return st;
        a.Q = q, a.q_scale = scale, a.ldq = plan.width / 2, a.q_zeros = true;
    }
    a.parts = reinterpret_cast<float*>(at + plan.x + plan.scale);
    a.ldparts = (a.np + 7) / 8 * 8;
    if (plan.route.few) return launch_few_rows(dev, a);
    return d->type == OZ_BF16 ? by_tile<OZ_BF16>(dev, plan.route.tile, a) : by_tile<OZ_F16>(dev, plan.route.tile, a);
}

}  // extern "C"

// The way of a product, for tests: -2 streamed, -1 the kernel of few rows, else the tile; *splits its ranges of k.
extern "C" int oz_rule_linear_i8(int cus, int M, int N, int K, int* splits) {
    oz_linear_i8_desc d{};
    d.M = M, d.N = N, d.K = K, d.x_int8 = 1;
    const Plan p = plan_of(cus, &d);
    if (splits) *splits = p.route.splits;
    return p.stream ? -2 : p.route.few ? -1 : (int)p.route.tile;
}
