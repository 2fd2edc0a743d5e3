// Tiled products of the Newton-Schulz iteration (oz_newton_schulz.hpp), on the linear layers' loops over a tile
// (oz_linear_tiles.hpp).
//
// A and A^2 are symmetric: only tiles on and above the diagonal are computed and written twice, as they are and transposed. X's
// product with the symmetric B takes X as it lies, B X with X read transposed out of LDS, X B for a tall matrix. All sides in the
// workspace are multiples of 64 with zeros behind the matrices, so no stage is ragged and every access of 8 values is whole.
#pragma once
#include "oz_linear_tiles.hpp"
#include "oz_newton_schulz.hpp"

namespace ozn {

using namespace ozt;
using ozl::Operand;

// Tile `u` of the T (T + 1) / 2 with row <= column: groups of 4 rows column by column, as the tiles of a whole product.
__device__ __forceinline__ void triangle(int u, int T, int& row, int& col) {
    int first = 0;
    for (;; first += 4) {
        const int g = min(T - first, 4), here = g * (T - first) - g * (g - 1) / 2;
        if (u < here) {
            const int head = g * (g + 1) / 2;  // columns first .. first + g - 1 have 1, 2, ... rows
            if (u < head) {
                int c = 0;
                while (u > c) u -= ++c;
                row = first + u, col = first + c;
            } else {
                row = first + (u - head) % g, col = first + g + (u - head) / g;
            }
            return;
        }
        u -= here;
    }
}

// Workgroup `first` + i of the P that a shape has -> its place in the shape's sequence of tiles: XCD x runs workgroups x, x + 8, ..., and gets a
// run of their number, the XCDs' runs one behind the other. A bijection for any first and P.
__device__ __forceinline__ int xcd_run(int first, int i, int P) {
    constexpr int N = ozg::XCDS;
    const int x = (first + i) % N, s = first % N;   // its XCD, and that of the shape's first
    const int k = (x - s) & (N - 1);                // the XCD's first workgroup of the shape
    const int q = P / N, r = P % N, wrap = max(s + r - N, 0);  // XCDs s .. s + r - 1 (modulo N) have q + 1
    return x * q + min(x, wrap) + min(max(x - s, 0), r - wrap) + (i - k) / N;
}

// Workgroup -> shape, matrix and tile; false where there is nothing for it. Shapes come one after the other (the long ones first, as they
// differ in length), within a shape each XCD takes one contiguous run of the tiles, so that what it runs at a time shares rows and columns
// in its L2. A launch may have the first or the last tiles of a sequence of larger ones (Pass): `parent` / T by as many tiles in each.
template <Phase PHASE, int T>
__device__ __forceinline__ bool tile_place(const Shapes& m, const Pass& pass, int w, int& shape, int& matrix, int& tq, int& tp) {
    const Places& p = pass.places;
    shape = __builtin_amdgcn_readfirstlane(shape_of(p, m.n, w));
    const Shape& s = m.s[shape];
    const int split = pass.parent / T, sub = split * split, P = pass.parent;
    int j = xcd_run(p.first[shape], w - p.first[shape], p.first[shape + 1] - p.first[shape]);
    const int inside = __builtin_amdgcn_readfirstlane(j % sub);
    j = __builtin_amdgcn_readfirstlane(j / sub + pass.begin[shape]);
    matrix = __builtin_amdgcn_readfirstlane(j / p.per[shape]);
    const int u = j - matrix * p.per[shape];
    if constexpr (PHASE == UPDATE) {
        // groups of rows column by column: what an XCD runs at a time is 8 x 8 tiles of 128 (4 x 16: 782 for 750 us) or 4 x 8 of 256
        const int G = P == 256 ? 4 : 8;
        const int rows = (s.R + P - 1) / P, cols = (s.C + P - 1) / P;
        const int group = u / (G * cols), first = G * group, g = min(rows - first, G), v = u - group * G * cols;
        tq = first + v % g, tp = v / g;
    } else {
        triangle(u, (side_of(s) + P - 1) / P, tq, tp);
    }
    tq = __builtin_amdgcn_readfirstlane(tq * split + inside / split);
    tp = __builtin_amdgcn_readfirstlane(tp * split + inside % split);
    if (split == 1) return true;
    if (PHASE != UPDATE) return tq <= tp && T * tp < side_of(s);
    return T * tq < s.R && T * tp < s.C;
}

// ---- from sums to values ------------------------------------------------------------------------------

union Half8 {
    u32x4 w;
    f16x8 v;
};
// v in one or two parts to h and l. PAST: past the caches, which the products' operands need more.
template <bool PAST>
__device__ __forceinline__ void put8(_Float16* h, _Float16* l, long long at, const float* v) {
    f16x8 x, y;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        x[k] = (_Float16)v[k];
        y[k] = (_Float16)(v[k] - (float)x[k]);
    }
    if constexpr (PAST) {
        __builtin_nontemporal_store(x, reinterpret_cast<f16x8*>(h + at));
        __builtin_nontemporal_store(y, reinterpret_cast<f16x8*>(l + at));
    } else {
        *reinterpret_cast<f16x8*>(h + at) = x;
        if (l) *reinterpret_cast<f16x8*>(l + at) = y;
    }
}

// How a wave's sums go through LDS: RI bands of 16 rows at a time, turns of RT rows, a lane 8 values in a row; pieces of what they
// are added to are asked for in batches.
template <bool THREE, int TI, int TJ, int ROOM>
struct Bands {
    static constexpr int ROW = 16 * TJ;
    static constexpr int RI = TI * 16 * ROW <= ROOM ? TI : TI * 8 * ROW <= ROOM ? TI / 2 : TI / 4;
    static_assert(RI >= 1 && RI * 16 * ROW <= ROOM && TI % RI == 0, "staging room");
    static constexpr int RT = 32 / TJ, NT = 16 * RI / RT;
    static constexpr int BATCH = NT < 8 ? NT : 8, ALL = TI / RI * NT / BATCH;  // of a turn's pieces; batches of a tile
    static_assert(NT % BATCH == 0, "whole batches");
    // With one batch the pieces that products of first parts are added to are asked for before them and wait in registers (four large
    // blocks' update in tiles of 128 x 128: 693 us for 752). Products of both parts have none left over: there they cost (matrices of
    // 700 x 1500 and others in tiles of 128 x 128: 40 us for 37). More do not fit: two in turn, a batch ahead.
    static constexpr bool AHEAD = ALL == 1 && !THREE;
    static constexpr int BUFFERS = ALL == 1 ? 1 : 2;
};

// The sums of a wave, as in ozl::put_sums: ask(P, t, row) loads what the t-th piece of a batch wants, use(P, t, row, v) finishes its 8
// values (P: the batch's buffer; rows and columns are the wave's own). With TWICE use()'s values go back to LDS, and across(row, col, v)
// gets 8 values of a column from `row` on.
template <bool THREE, int TI, int TJ, int ROOM, class Ask, class P>
__device__ __forceinline__ void ask_batch(int lane, Ask&& ask, int b, P p) {
    typedef Bands<THREE, TI, TJ, ROOM> S;
    ozl::each<S::BATCH>([&](auto T) { ask(p, T, (b * S::BATCH + decltype(T)::value) * S::RT + lane / (2 * TJ)); });
}
template <bool THREE, int TI, int TJ, int ROOM, bool TWICE, class Ask, class Use, class Across>
__device__ __forceinline__ void put_rows(const f32x4 (&acc)[TI][TJ], float* tile, int lane, bool twice, Ask&& ask, Use&& use, Across&& across) {
    typedef Bands<THREE, TI, TJ, ROOM> S;
    constexpr int ROW = S::ROW, RI = S::RI, RT = S::RT, BATCHES = S::NT / S::BATCH;
    static_assert(TJ >= 2, "8 pieces of a row");
    // a row's pieces of 4 values swizzled so that 8 rows in a row, and every eighth row, have a column on other banks
    const auto swizzle = [](int row) { return (row ^ (row >> 3)) & 7; };
    const int r = lane & 15, g = lane >> 4, piece = 2 * (lane % (2 * TJ)), rr = lane / (2 * TJ);
    if constexpr (!S::AHEAD) ask_batch<THREE, TI, TJ, ROOM>(lane, ask, 0, std::integral_constant<int, 0>{});
    ozl::each<TI / RI>([&](auto H) {
        constexpr int h = decltype(H)::value;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < RI; i++)
#pragma unroll
            for (int j = 0; j < TJ; j++) *reinterpret_cast<f32x4*>(tile + (16 * i + r) * ROW + 4 * ((4 * j + g) ^ swizzle(16 * i + r))) = acc[h * RI + i][j];
        __builtin_amdgcn_wave_barrier();
        ozl::each<BATCHES>([&](auto C) {
            constexpr int c = decltype(C)::value, b = h * BATCHES + c;
            if constexpr (b + 1 < S::ALL) ask_batch<THREE, TI, TJ, ROOM>(lane, ask, b + 1, std::integral_constant<int, (b + 1) & 1>{});
            ozl::each<S::BATCH>([&](auto T) {
                constexpr int t = decltype(T)::value;
                const int row = (c * S::BATCH + t) * RT + rr;
                float v[8];
                f32x4* at[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    at[k] = reinterpret_cast<f32x4*>(tile + row * ROW + 4 * ((piece + k) ^ swizzle(row)));
                    const f32x4 x = *at[k];
#pragma unroll
                    for (int m = 0; m < 4; m++) v[4 * k + m] = x[m];
                }
                // X's row made anew, so that no addresses wait in registers from asking until here: 256 x 256 tiles have none left, products
                // of both parts in tiles of 128 x 128 21.7 us for 21.0. (Tiles that are written twice lose by it: 130 us for 137)
                int turn = 16 * RI * h + (c * S::BATCH + t) * RT;
                if constexpr (!TWICE) asm volatile("" : "+s"(turn));
                use(std::integral_constant<int, b % S::BUFFERS>{}, T, turn + rr, v);
                if constexpr (TWICE) {
#pragma unroll
                    for (int k = 0; k < 2; k++) *at[k] = f32x4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
                }
            });
        });
        if constexpr (TWICE) {
            if (twice) {
                // 8 rows a lane, so that neighbouring lanes' 16 bytes of a column lie next to each other: whole lines (with a column a
                // lane the 64 pieces of a store went to 64 lines: two rounds of 256 x 256 tiles of 8192^2's A 423 us for 402)
                constexpr int CHUNKS = 2 * RI < 8 ? 2 * RI : 8, COLS = 64 / CHUNKS;
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int r0 = 0; r0 < 16 * RI; r0 += 8 * CHUNKS)
#pragma unroll 2
                    for (int c0 = 0; c0 < ROW; c0 += COLS) {
                        const int col = c0 + lane / CHUNKS, row = r0 + 8 * (lane % CHUNKS);
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) v[k] = tile[(row + k) * ROW + 4 * ((col >> 2) ^ swizzle(row + k)) + (col & 3)];
                        across(16 * RI * h + row, col, v);
                    }
                __builtin_amdgcn_wave_barrier();
            }
        }
    });
}

// What a wave's sums become: its first row and column q0 and p0, the lane's column. SQUARE adds to A, UPDATE to X.
template <Phase PHASE, bool THREE, int TI, int TJ, int ROOM>
struct Finish {
    typedef Bands<THREE, TI, TJ, ROOM> S;
    const Shape s;
    const Factors f;
    const int from, last;
    int i, lane, q0, p0, col, side;
    u32x4 hs[S::BUFFERS][S::BATCH], ls[S::BUFFERS][S::BATCH];
    const float* diagonal;  // B's in LDS: of the wave's columns, or of its rows, each four times
    int by_row, by_half;
    static constexpr int D = (16 * TI + 63) / 64;  // of it, a lane's values

    __device__ __forceinline__ Finish(const Shape& s, const Pass& pass, int i, int lane, int q0, int p0)
        : s(s), f(pass.f), from(pass.from), last(pass.last), i(i), lane(lane), q0(q0), p0(p0), col(p0 + 8 * (lane % (2 * TJ))), side(side_of(s)) {}

    template <class P, class T>
    __device__ __forceinline__ void ask(P, T, int row) {
        if constexpr (PHASE == GRAM) return;
        constexpr int b = P::value, t = T::value;
        const int rows = PHASE == SQUARE ? side : s.R, cols = PHASE == SQUARE ? side : s.C;
        const _Float16* h = PHASE == SQUARE ? square_of(s, s.a, i) : h_of(s, from, i);
        const _Float16* l = PHASE == SQUARE ? h + (long long)side * side : l_of(s, from, i);
        const long long at = (long long)(q0 + row) * cols + col;
        if (q0 + row < rows && col < cols) {
            hs[b][t] = *reinterpret_cast<const u32x4*>(h + at);
            if constexpr (PHASE == UPDATE && !THREE) ls[b][t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(l + at));
            else if constexpr (THREE) ls[b][t] = *reinterpret_cast<const u32x4*>(l + at);
        }
    }
    __device__ __forceinline__ void ahead() {
        if constexpr (S::AHEAD) ask_batch<THREE, TI, TJ, ROOM>(lane, [&](auto P, auto T, int row) { ask(P, T, row); }, 0, std::integral_constant<int, 0>{});
    }
    // v = factor times what it is added to, and `of` v
    template <class P, class T>
    __device__ __forceinline__ void add(P, T, int row, float factor, float of, float* v) const {
        Half8 x, y;
        x.w = hs[P::value][T::value], y.w = ls[P::value][T::value];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            f32x4 f = {factor, factor, factor, factor};
            if constexpr (PHASE == UPDATE && !THREE) f += *reinterpret_cast<const f32x4*>(diagonal + by_row * (row - lane / (2 * TJ)) + by_half * half);
#pragma unroll
            for (int k = 4 * half; k < 4 * half + 4; k++) {
                float z = (float)x.v[k];
                if constexpr (THREE || PHASE == UPDATE) z += (float)y.v[k];
                v[k] = __builtin_fmaf(of, v[k], f[k & 3] * z);
            }
        }
    }

    __device__ __forceinline__ void put(const Ends& ends, bool mirror, const f32x4 (&acc)[TI][TJ], float* tile, const float (&d)[D]) {
        const auto get = [&](auto P, auto T, int row) { ask(P, T, row); };
        if constexpr (PHASE != UPDATE) {
            _Float16* to = PHASE == GRAM ? square_of(s, s.a, i) : square_of(s, s.b, i);
            _Float16* rest = THREE ? to + (long long)side * side : nullptr;
            put_rows<THREE, TI, TJ, ROOM, true>(
                acc, tile, lane, mirror, get,
                [&](auto P, auto T, int row, float* v) {
                    if constexpr (PHASE == GRAM) {
#pragma unroll
                        for (int k = 0; k < 8; k++) v[k] *= f.gram;
                    } else {
                        add(P, T, row, f.b, f.c, v);
                        if (!THREE && !mirror) {  // a tile on the diagonal
                            float* d = diagonal_of(s, i);
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                if (q0 + row == col + k && col < side) d[col + k] = v[k] * f.update, v[k] = 0.0f;
                        }
                    }
                    if (q0 + row < side && col < side) put8<false>(to, rest, (long long)(q0 + row) * side + col, v);
                },
                [&](int row, int c, const float* v) {
                    if (q0 + row < side && p0 + c < side) put8<false>(to, rest, (long long)(p0 + c) * side + q0 + row, v);
                });
        } else {
            auto none = [](int, int, const float*) {};
            if constexpr (!THREE) {
                constexpr int AT = 16 * S::RI * S::ROW;  // behind the staged sums
                static_assert(AT + 64 * TI <= ROOM, "room for the diagonal");
#pragma unroll
                for (int k = 0; k < D; k++) {
                    const int j = 64 * k + lane;
                    if (is_tall(s) && j < 16 * TI) tile[AT + j] = d[k];
                    else if (j < 16 * TI) *reinterpret_cast<f32x4*>(tile + AT + 4 * j) = f32x4{d[k], d[k], d[k], d[k]};
                }
                diagonal = tile + AT + (is_tall(s) ? col - p0 : 4 * (lane / (2 * TJ)));
                by_row = is_tall(s) ? 0 : 4, by_half = is_tall(s) ? 4 : 0;
            }
            if (!last) {
                _Float16 *to = h_of(s, from ^ 1, i), *rest = l_of(s, from ^ 1, i);
                put_rows<THREE, TI, TJ, ROOM, false>(
                    acc, tile, lane, false, get,
                    [&](auto P, auto T, int row, float* v) {
                        add(P, T, row, f.a, f.update, v);
                        if (q0 + row < s.R && col < s.C) put8<!THREE>(to, rest, (long long)(q0 + row) * s.C + col, v);
                    },
                    none);
            } else if (ends.tensors) {
                const oz_muon_tensor t = ends.tensors[s.first + i];
                const float keep = 1.0f - ends.lr * t.weight_decay, rate = ends.lr * t.lr_scale * (1.0f / kScale);
                put_rows<THREE, TI, TJ, ROOM, false>(
                    acc, tile, lane, false, get,
                    [&](auto P, auto T, int row, float* v) {
                        add(P, T, row, f.a, f.update, v);
                        const int q = q0 + row, count = q < s.rows ? min(s.cols - col, 8) : 0;
                        if (count <= 0) return;
                        const long long at = (long long)q * s.cols + col;
                        const void* from = t.master ? t.master : t.param;
                        const int type = t.master ? OZ_F32 : t.param_type;
                        float x[8];
                        if (count == 8) load8(from, type, at, x);
                        else load_some(from, type, at, count, x);
#pragma unroll
                        for (int k = 0; k < 8; k++) x[k] = x[k] * keep - v[k] * rate;
                        if (count == 8) {
                            if (t.master) store8(t.master, OZ_F32, at, x);
                            store8(t.param, t.param_type, at, x);
                        } else {
                            if (t.master) store_some(t.master, OZ_F32, at, count, x);
                            store_some(t.param, t.param_type, at, count, x);
                        }
                    },
                    none);
            } else {
                put_rows<THREE, TI, TJ, ROOM, false>(
                    acc, tile, lane, false, get,
                    [&](auto P, auto T, int row, float* v) {
                        add(P, T, row, f.a, f.update, v);
                        const int q = q0 + row, count = q < s.rows ? min(s.cols - col, 8) : 0;
                        if (count <= 0) return;
                        const long long at = (s.first + i) * ends.stride_o + q * ends.ldo + col;
#pragma unroll
                        for (int k = 0; k < 8; k++) v[k] *= 1.0f / kScale;
                        if (count == 8) store8(ends.O, ends.type, at, v);
                        else store_some(ends.O, ends.type, at, count, v);
                    },
                    none);
            }
        }
    }
};

// ---- kernels ------------------------------------------------------------------------------------------

// Products of both parts: h h + h l + l h in one loop, which brings each part of an operand once for the two products that read it
// (one after the other they would be brought, and read out of LDS, half as often again: three matrices of
// 700 x 1500 in 306 us for 265). As ozl::BigLoop, with pairs of units: 4 waves
// of 16 B x 16 B outputs, a ring of five pairs, the copies of stage k + 2 of Q in stage k's first step, those of P in its second.
template <bool QM, bool PM, int B>
struct PairLoop {
    typedef Half<OZ_F16> M;
    typedef typename M::x8 T8;
    typedef Operand<QM, 32 * B, 4> OQ;
    typedef Operand<PM, 32 * B, 4> OP;
    static constexpr int UNIT = 2 * ozl::BC * 32 * B, PAIR = 2 * UNIT, RING = 5 * PAIR, LD = OQ::N, LDS = RING, ROOM = RING / 4 / 4;
    static_assert(OQ::N == OP::N, "copies of a unit");
    struct Parts {
        T8 h[B], l[B];
    };

    __device__ static __forceinline__ void run(uint8_t* lds, OQ (&oq)[2], OP (&op)[2], int nst, int lane, int wave, f32x4 (&out)[B][B]) {
        const int wq = B * (wave >> 1), wp = B * (wave & 1);
        const int lq = OQ::lane_offset(lane), lp = OP::lane_offset(lane);
        f32x4 acc[B][B];
#pragma unroll
        for (int i = 0; i < B; i++)
#pragma unroll
            for (int j = 0; j < B; j++) acc[i][j] = f32x4{0, 0, 0, 0};
        auto copy_q = [&](int to, int j) { oq[j / LD].copy(lds + to + UNIT * (j / LD), j % LD, wave); };
        auto copy_p = [&](int to, int j) { op[j / LD].copy(lds + to + UNIT * (j / LD), j % LD, wave); };
        auto landed = [&](auto LEFT) {
            ozl::wait_vmcnt_lgkm0<decltype(LEFT)::value>();
            ozl::stage_barrier();
        };
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int j = 0; j < 2 * LD; j++) copy_q(2 * s * PAIR, j);
#pragma unroll
            for (int j = 0; j < 2 * LD; j++) copy_p((2 * s + 1) * PAIR, j);
            oq[0].next(), oq[1].next(), op[0].next(), op[1].next();
        }
        // fragment t of a step, in the order its instructions want them
        auto read = [&](Parts& q, Parts& p, int t, int h, int uq, int up) {
            if (t == 0) q.h[0] = OQ::template fragment<T8>(lds + uq, h, wq, lq);
            else if (t <= B) p.h[t - 1] = OP::template fragment<T8>(lds + up, h, wp + t - 1, lp);
            else if (t < 2 * B) q.h[t - B] = OQ::template fragment<T8>(lds + uq, h, wq + t - B, lq);
            else if (t < 3 * B) p.l[t - 2 * B] = OP::template fragment<T8>(lds + up + UNIT, h, wp + t - 2 * B, lp);
            else q.l[t - 3 * B] = OQ::template fragment<T8>(lds + uq + UNIT, h, wq + t - 3 * B, lq);
        };
        Parts fq, fp, gq, gp;
        landed(std::integral_constant<int, 4 * LD>{});
#pragma unroll
        for (int t = 0; t < 4 * B; t++) read(fq, fp, t, 0, 0, PAIR);
        // One step: 3 B B matrix instructions on (xq, xp), the 4 B fragments (yq, yp) of step H of the pairs at uq and up, the copies of a pair
        // of Q (in a stage's first step) or P to `to`.
        auto step = [&](auto H, Parts& xq, Parts& xp, Parts& yq, Parts& yp, int uq, int up, int to) {
            constexpr int h = decltype(H)::value, R = B == 4 ? 3 : 1, C = B == 4 ? 3 : 2;
#pragma unroll
            for (int n = 0; n < 3 * B * B; n++) {
                const int part = n / (B * B), i = n / B % B, j = n % B;
                const T8 p = part == 1 ? xp.l[j] : xp.h[j], q = part == 2 ? xq.l[i] : xq.h[i];
                // (written as in the large loop only where a sum comes up again late enough)
                if constexpr (B * B >= ozl::kLeastSums) ozl::mfma_acc<M>(acc[i][j], p, q);
                else acc[i][j] = M::mfma(p, q, acc[i][j]);
                if (n % R == 0 && n / R < 4 * B) read(yq, yp, n / R, h, uq, up);
                if (n % C == C - 1 && n / C < 2 * LD) {
                    if constexpr (h == 1) copy_q(to, n / C);
                    else copy_p(to, n / C);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        int at = 0;
        auto wrap = [](int b) { return b >= RING ? b - RING : b; };
        for (int k = 0; k < nst; k++) {
            const int u1 = wrap(at + PAIR), u2 = wrap(at + 2 * PAIR), u3 = wrap(at + 3 * PAIR), u4 = wrap(at + 4 * PAIR);
            step(std::integral_constant<int, 1>{}, fq, fp, gq, gp, at, u1, u4);
            oq[0].next(), oq[1].next();
            landed(std::integral_constant<int, 2 * LD>{});
            step(std::integral_constant<int, 0>{}, gq, gp, fq, fp, u2, u3, at);
            op[0].next(), op[1].next();
            at = u2;
        }
        ozl::settle_sums();
        ozl::wait_vmcnt<0>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < B; i++)
#pragma unroll
            for (int j = 0; j < B; j++) out[i][j] = acc[i][j];
    }
};

// Tiles of products of the first parts (ONE) and of both. BLOCKS: bands of 16 rows and columns of a wave.
struct Tile64 {
    static constexpr int T = 64, BLOCKS = 2, PER_SIMD = 2;
    template <bool QM, bool PM>
    using One = ozl::TileLoop<Half<OZ_F16>, QM, PM, 2, 2, 2, 2, 4>;
    template <bool QM, bool PM>
    using Both = PairLoop<QM, PM, 2>;
};
struct Tile128 {
    static constexpr int T = 128, BLOCKS = 4, PER_SIMD = 2;
    template <bool QM, bool PM>
    using One = ozl::BigLoop<Half<OZ_F16>, QM, PM, 4>;
    template <bool QM, bool PM>
    using Both = PairLoop<QM, PM, 4>;
};
struct Tile256 {
    static constexpr int T = 256, BLOCKS = 8, PER_SIMD = 1;
    template <bool QM, bool PM>
    using One = ozl::BigLoop<Half<OZ_F16>, QM, PM>;
};
template <class TILE, bool THREE, bool QM, bool PM>
struct LoopOf {
    typedef typename TILE::template One<QM, PM> type;
};
template <class TILE, bool QM, bool PM>
struct LoopOf<TILE, true, QM, PM> {
    typedef typename TILE::template Both<QM, PM> type;
};

template <Phase PHASE, class TILE, bool THREE>
__global__ void __launch_bounds__(256, THREE && TILE::T == 128 ? 1 : TILE::PER_SIMD) newton_schulz_kernel(const Shapes m, const Ends ends, const Pass pass) {
    constexpr int T = TILE::T, B = TILE::BLOCKS;
    typedef typename LoopOf<TILE, THREE, false, false>::type Any;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Any::LDS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int shape, i, tq, tp;
    if (!tile_place<PHASE, T>(m, pass, blockIdx.x, shape, i, tq, tp)) return;
    const Shape s = m.s[shape];
    const int side = side_of(s), q0 = T * tq, p0 = T * tp;
    const long long nx = (long long)s.R * s.C, nn = (long long)side * side;  // values of a plane
    f32x4 acc[B][B];
    // sum over c < C of Q(q, c) P(p, c)
    auto run = [&](auto QM, auto PM, const _Float16* Q, int nq, int ldq, long long plane_q, const _Float16* P, int np, int ldp, long long plane_p, int C) {
        typedef typename LoopOf<TILE, THREE, decltype(QM)::value, decltype(PM)::value>::type Loop;
        const int stages = C / ozl::BC;
        if constexpr (THREE) {
            typename Loop::OQ oq[2];
            typename Loop::OP op[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                oq[k].init(Q + k * plane_q, ldq, nq, C, q0, 0, stages, lane, wave);
                op[k].init(P + k * plane_p, ldp, np, C, p0, 0, stages, lane, wave);
            }
            Loop::run(lds, oq, op, stages, lane, wave, acc);
        } else {
            typename Loop::OQ oq;
            typename Loop::OP op;
            oq.init(Q, ldq, nq, C, q0, 0, stages, lane, wave);
            op.init(P, ldp, np, C, p0, 0, stages, lane, wave);
            Loop::template run<uint16_t>(lds, oq, op, stages, 0, lane, wave, acc);
        }
    };
    constexpr std::false_type no{};
    constexpr std::true_type yes{};
    const _Float16* x = h_of(s, pass.from, i);
    typedef Finish<PHASE, THREE, B, B, Any::ROOM> Put;
    const int q1 = q0 + 16 * B * (wave / 2), p1 = p0 + 16 * B * (wave % 2);
    Put put(s, pass, i, lane, q1, p1);
    put.ahead();
    float d[Put::D] = {};
    if constexpr (PHASE == UPDATE && !THREE) {
#pragma unroll
        for (int k = 0; k < Put::D; k++) {
            const int j = (is_tall(s) ? p1 : q1) + 64 * k + lane;
            if (j < side) d[k] = diagonal_of(s, i)[j];
        }
    }
    if constexpr (PHASE == GRAM) {
        if (is_tall(s)) run(yes, yes, x, s.C, s.C, nx, x, s.C, s.C, nx, s.R);
        else run(no, no, x, s.R, s.C, nx, x, s.R, s.C, nx, s.C);
    } else if constexpr (PHASE == SQUARE) {
        const _Float16* a = square_of(s, s.a, i);
        run(no, no, a, side, side, nn, a, side, side, nn, side);
    } else {
        const _Float16* b = square_of(s, s.b, i);
        if (is_tall(s)) run(no, no, x, s.R, s.C, nx, b, side, side, nn, side);
        else run(no, yes, b, side, side, nn, x, s.C, s.C, nx, side);
    }
    float* room = reinterpret_cast<float*>(lds) + wave * Any::ROOM;
    if constexpr (Put::S::AHEAD) put.put(ends, tq != tp, acc, room, d);
    else Put(s, pass, i, lane, q1, p1).put(ends, tq != tp, acc, room, d);
}

template <bool THREE>
void launch_products(hipStream_t stream, Phase phase, int tile, const Shapes& m, const Ends& ends, const Pass& pass) {
    const dim3 grid((unsigned)pass.places.first[m.n]), block(256);
    auto with = [&](auto TILE) {
        typedef decltype(TILE) Tile;
        if (phase == GRAM) hipLaunchKernelGGL((newton_schulz_kernel<GRAM, Tile, THREE>), grid, block, 0, stream, m, ends, pass);
        else if (phase == SQUARE) hipLaunchKernelGGL((newton_schulz_kernel<SQUARE, Tile, THREE>), grid, block, 0, stream, m, ends, pass);
        else hipLaunchKernelGGL((newton_schulz_kernel<UPDATE, Tile, THREE>), grid, block, 0, stream, m, ends, pass);
    };
    if (tile == 64) return with(Tile64{});
    if constexpr (!THREE)
        if (tile == 256) return with(Tile256{});
    with(Tile128{});
}

}  // namespace ozn
