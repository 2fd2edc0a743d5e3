// Tiles of the products with an epilogue: operands staged in LDS by direct copies, matrix instructions of
// 16 x 16 x 32, sums in FP32.
//
// A stage is 64 values of c of both operands, two steps of the matrix instructions. An operand whose rows run along c
// (row-major activations and weights) is staged as 1 KB blocks of 8 rows x 128 bytes, one copy each: whole cache lines
// (with 64 bytes a row all CUs together get 70 GB/s each out of the L2, with 128 they get 128). Their 16-byte chunks
// are swizzled so that the 64 lanes of a fragment read fall on all banks equally: lane l reads row l % 16, chunk l / 16 of
// a step. An operand whose rows run along its own index (the gradients' transposed ones) is staged as 64 rows
// of c, and a fragment is read by the transposing LDS read: 16 lanes read 4 rows of c x 16 columns, and lane i gets column
// i's 4 values; the columns' 32-byte pieces are swizzled by the row, so that the rows that a read takes at once fall on
// different banks. Both give a lane the same 8 values of c.
//
// The copies are buffer loads, whose range is checked by the 4-byte word: what lies outside an operand is outside its
// buffer's range and reads as zero, so no load is guarded and nothing beyond the word with an operand's last value is
// touched. Rows may begin at any multiple of 4 bytes.
#pragma once
#include "oz_gemm_common.hpp"
#include "oz_linear.hpp"

#include <type_traits>
#include <utility>

namespace ozl {

using namespace ozt;
using ozg::stage_barrier;
using ozg::wait_vmcnt;
using ozg::wait_vmcnt_lgkm0;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int BC = 64;                       // c of a stage, two steps of 32
constexpr unsigned OUTSIDE = 0x80000000u;    // an offset beyond every range

// Copies 16 bytes a lane from buffer rs at offset voff to LDS byte lbase + 16 lane. M0 carries the LDS base;
// the wait state between its write and the copy is the s_nop.
__device__ __forceinline__ void lds_copy(v4i rs, void* lbase, unsigned voff) {
    const unsigned l = (unsigned)(uintptr_t)(lds_u8*)lbase;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(l), "v"(voff), "s"(rs) : "memory");
}

// One operand of a tile of ROWS rows: its copies (wave `wave` of W brings blocks wave, wave + W, ...) and fragments.
template <bool MAJOR, int ROWS, int W>
struct Operand {
    static constexpr int BLOCKS = ROWS / 8;   // 1 KB blocks of a stage
    static constexpr int N = BLOCKS / W;      // copies of a wave
    static_assert(N * W == BLOCKS, "whole blocks per wave");
    static constexpr int RB = 2 * ROWS;       // MAJOR: bytes of a row of c
    static constexpr int PIECES = RB / 32;    // 32-byte pieces of it
    v4i rs;          // buffer of the stage to load next: its address, and what of the operand lies from there on (of this stage)
    unsigned range;  // !MAJOR: from its address to the end of the tile's last row; MAJOR: of a whole stage
    unsigned last;   // MAJOR: of the last stage
    unsigned step;   // bytes of a stage's advance
    unsigned off[N]; // of this lane's copies
    int steps;       // stages left to load

    // a row's swizzle in 32-byte pieces: rows 8 g + j and 8 g + 4 + j (j < 4) of g and g + 1 differ
    __device__ static int piece_swizzle(int row) { return ((row & 3) | ((row >> 3) & 1) << 2) & (PIECES - 1); }

    __device__ __forceinline__ void init(const void* p, long long ld, long long n, long long C, long long row0, long long c0, int stages,
                                         int lane, int wave) {
        steps = stages;
        const long long ldb = 2 * ld;
        unsigned long long base;
        if constexpr (MAJOR) {
            base = (unsigned long long)p + c0 * ldb + 2 * row0;
            step = (unsigned)(BC * ldb);
            const long long end = C - c0 - (long long)BC * (stages - 1);  // rows of the last stage
            range = (unsigned)(BC * ldb);
            last = (unsigned)((end < BC ? end - 1 : BC - 1) * ldb + ((2 * (n - row0) + 3) & ~3ll));
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int byte = 1024 * (W * j + wave) + 16 * lane, row = byte / RB;
                const int chunk = ((byte % RB) / 16) ^ (piece_swizzle(row) << 1);
                off[j] = row0 + 8 * chunk < n ? (unsigned)(row * ldb + 16 * chunk) : OUTSIDE;
            }
        } else {
            base = (unsigned long long)p + row0 * ldb + 2 * c0;
            step = 2 * BC;
            range = (unsigned)(((n - row0 < ROWS ? n - row0 : ROWS) - 1) * ldb + ((2 * (C - c0) + 3) & ~3ll));
            last = 0;
            const int r = lane >> 3, chunk = (lane & 7) ^ r;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int row = 8 * (W * j + wave) + r;
                off[j] = row0 + row < n ? (unsigned)(row * ldb + 16 * chunk) : OUTSIDE;
            }
        }
        rs[0] = __builtin_amdgcn_readfirstlane((int)base);
        rs[1] = __builtin_amdgcn_readfirstlane((int)(base >> 32) & 0xFFFF);
        rs[3] = 0x00020000;
        range = __builtin_amdgcn_readfirstlane(range);
        last = __builtin_amdgcn_readfirstlane(last);
        step = __builtin_amdgcn_readfirstlane(step);
        limit();
    }
    // A few scalar instructions a stage: whatever more there was showed (85 cycles a stage, 2% of 8192^3, 15% of small
    // products, for 64-bit ranges and a mask of the last chunks).
    __device__ __forceinline__ void limit() {
        if constexpr (MAJOR) rs[2] = steps > 1 ? range : steps == 1 ? last : 0u;
        else rs[2] = steps > 0 ? range : 0u;
    }
    __device__ __forceinline__ void copy(uint8_t* stage, int j, int wave) const { lds_copy(rs, stage + 1024 * (W * j + wave), off[j]); }
    __device__ __forceinline__ void next() {
        steps--;
        const unsigned long long base = ((unsigned long long)(unsigned)rs[1] << 32 | (unsigned)rs[0]) + step;
        rs[0] = (int)base;
        rs[1] = (int)(base >> 32);
        if constexpr (!MAJOR) range -= step;
        limit();
    }

    // Zeros for what lies behind the `valid` last values of c in a stage: there stand a window's other columns or the next
    // row (rows of c beyond the last are zeros).
    __device__ static void zero_tail(uint8_t* stage, int valid, int thread) {
        if constexpr (!MAJOR) {
            const v4i none = {0, 0, 0, 0};
            for (int row = thread; row < ROWS; row += 64 * W) {
                uint8_t* at = stage + 128 * row;
                uint16_t* cut = reinterpret_cast<uint16_t*>(at + 16 * ((valid >> 3) ^ (row & 7)));
                for (int e = valid & 7; e < 8; e++) cut[e] = 0;
                for (int c = (valid >> 3) + 1; c < 8; c++) *reinterpret_cast<v4i*>(at + 16 * (c ^ (row & 7))) = none;
            }
        }
    }

    // Fragment of rows 16 blk .. 16 blk + 15 in step h (0, 1) of the stage.
    __device__ static int lane_offset(int lane) {
        if constexpr (MAJOR) {
            const int row = 8 * (lane >> 4) + ((lane >> 2) & 3);
            return row * RB + 8 * (lane & 3) + 32 * piece_swizzle(row);  // piece 0; piece b is this xor 32 b
        } else {
            const int r = lane & 15, g = lane >> 4;
            return 128 * r + 16 * (g ^ (r & 7));  // step 0; step 1 is this xor 64
        }
    }
    template <class T8>
    __device__ static __forceinline__ T8 fragment(const uint8_t* stage, int h, int blk, int loff) {
        if constexpr (MAJOR) {
            typedef __attribute__((address_space(3))) v4s lds_v4s;
            union {
                v4s h[2];
                T8 v;
            } u;
            const uint8_t* at = stage + 32 * RB * h + (loff ^ (32 * blk));
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 4 * RB));
            return u.v;
        } else {
            return *reinterpret_cast<const T8*>(stage + 2048 * blk + (loff ^ (64 * h)));
        }
    }
};

// Workgroup -> tile, in the XCD-aware order of the exact products' kernels, and range of c.
__device__ __forceinline__ void place_of(const Product& a, int tiles_q, int tiles_p, int& split, int& tq, int& tp) {
    ozg::tile_of(blockIdx.x, tiles_q, tiles_p, a.splits, split, tq, tp);
    split = __builtin_amdgcn_readfirstlane(split);
    tq = __builtin_amdgcn_readfirstlane(tq);
    tp = __builtin_amdgcn_readfirstlane(tp);
}

// f(0), ..., f(N - 1), the numbers as types: what indexes registers is a constant whatever the compiler unrolls.
template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

// The sums of a wave to the outputs. Register k of lane l holds p = 4 (l / 16) + k, q = l % 16. They go through LDS (`tile`,
// ROOM floats of the wave's own), RI bands of 16 rows at a time, in rows of 16 TJ values whose 16-byte pieces are swizzled
// by the row; then a lane takes 8 values in a row, the same columns each time, so that outputs, residual
// and Z move in whole 16-byte pieces and whole rows. The residual's pieces are asked for a batch ahead: with one wave
// on a SIMD nothing else would hide their latency (8192^3 with everything in the epilogue: 1003 us with a
// wait for each piece).
template <int TYPE, int TI, int TJ, int ROOM>
__device__ __forceinline__ void put_sums(const Product& a, const f32x4 (&acc)[TI][TJ], float* tile, int lane, int split, long long q0, long long p0) {
    constexpr int ROW = 16 * TJ;
    constexpr int RI = TI * 16 * ROW <= ROOM ? TI : TI * 8 * ROW <= ROOM ? TI / 2 : TI / 4;
    static_assert(RI >= 1 && RI * 16 * ROW <= ROOM && TI % RI == 0, "staging room");
    constexpr int XM = TJ * 4 >= 8 ? 7 : TJ * 4 - 1;
    constexpr int RT = 32 / TJ, NT = 16 * RI / RT;            // rows of a turn, turns of RI bands
    constexpr int BATCH = NT < 4 ? NT : 4, BATCHES = NT / BATCH;
    const Epilogue& e = a.epi;
    const int r = lane & 15, g = lane >> 4, piece = 2 * (lane % (2 * TJ)), rr = lane / (2 * TJ);
    const long long p = p0 + 4 * piece;
    auto write = [&](auto H) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < RI; i++)
#pragma unroll
            for (int j = 0; j < TJ; j++)
                *reinterpret_cast<f32x4*>(tile + (16 * i + r) * ROW + 4 * ((4 * j + g) ^ (r & XM))) = acc[decltype(H)::value * RI + i][j];
        __builtin_amdgcn_wave_barrier();
    };
    auto read = [&](int row, float* v) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(tile + row * ROW + 4 * ((piece + k) ^ (row & XM)));
#pragma unroll
            for (int m = 0; m < 4; m++) v[4 * k + m] = x[m];
        }
    };
    if (a.splits > 1) {
        each<TI / RI>([&](auto H) {
            constexpr int h = decltype(H)::value;
            write(H);
#pragma unroll 4
            for (int turn = 0; turn < NT; turn++) {
                const long long q = q0 + 16 * h * RI + RT * turn + rr;
                float v[8];
                read(RT * turn + rr, v);
                if (q < a.nq && p < a.np) store8(a.parts, OZ_F32, (split * a.nq + q) * a.ldparts + p, v);
            }
        });
        return;
    }
    // A row's last, fewer than 8 values: the lane takes the row's last 8 instead, of which its neighbour has the first ones too
    // and writes the same. (Only where fewer than 8 are left for the wave are they written one by one.)
    const long long pl = p + 8 <= a.np || a.np - 8 < p0 ? p : a.np - 8;
    const bool in = p < a.np && pl + 8 <= a.np;
    float bias[8] = {};
    if (e.bias && in) load8(e.bias, TYPE, pl, bias);
    const int wide = e.y_type == OZ_F32;
    const char* pr = static_cast<const char*>(e.residual) + ((q0 + rr) * e.ldr + pl) * (wide ? 4 : 2);
    char* py = static_cast<char*>(e.Y) + ((q0 + rr) * e.ldy + pl) * (wide ? 4 : 2);
    char* pz = static_cast<char*>(e.Z) + ((q0 + rr) * e.ldz + pl) * 2;
    const long long dr = RT * e.ldr * (wide ? 4 : 2), dy = RT * e.ldy * (wide ? 4 : 2), dz = RT * e.ldz * 2;
    u32x4 res[2][BATCH][2] = {};
    auto ask = [&](auto B) {  // batch B of all TI / RI * BATCHES
        constexpr int b = decltype(B)::value;
        if (!e.residual) return;
#pragma unroll
        for (int t = 0; t < BATCH; t++) {
            if (!in || q0 + (b * BATCH + t) * RT + rr >= a.nq) continue;
            const char* from = pr + (b * BATCH + t) * dr;
            res[b & 1][t][0] = get16<u32x4>(from);
            if (wide) res[b & 1][t][1] = get16<u32x4>(from + 16);
        }
    };
    ask(std::integral_constant<int, 0>{});
    each<TI / RI>([&](auto H) {
        constexpr int h = decltype(H)::value;
        write(H);
        each<BATCHES>([&](auto C) {
            constexpr int c = decltype(C)::value, b = h * BATCHES + c;
            if constexpr (b + 1 < TI / RI * BATCHES) ask(std::integral_constant<int, b + 1>{});
#pragma unroll
            for (int t = 0; t < BATCH; t++) {
                const int turn = c * BATCH + t;
                if (!in || q0 + (h * NT + turn) * RT + rr >= a.nq) continue;
                float v[8];
                if (pl == p) {
                    read(RT * turn + rr, v);
                } else {
                    const int row = RT * turn + rr, col = (int)(pl - p0);
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] = tile[row * ROW + 4 * (((col + k) >> 2) ^ (row & XM)) + ((col + k) & 3)];
                }
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] += bias[k];
                if (e.Z) store8(pz + (h * NT + turn) * dz, TYPE, 0, v);
                act8(v, e.act);
                if (e.residual) {
                    float x[8];
                    if (wide) {
#pragma unroll
                        for (int k = 0; k < 8; k++) x[k] = __uint_as_float(res[b & 1][t][k >> 2][k & 3]);
                    } else {
                        widen8(res[b & 1][t][0], TYPE, x);
                    }
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] += x[k];
                }
                store8(py + (h * NT + turn) * dy, e.y_type, 0, v);
            }
        });
        if (!in && p < a.np) {
#pragma unroll 1
            for (int turn = 0; turn < NT; turn++) {
                const long long q = q0 + (h * NT + turn) * RT + rr;
                float v[8];
                read(RT * turn + rr, v);
                if (q < a.nq) finish8<TYPE>(e, a.np, q, p, v);
            }
        }
    });
}

// The values of c in the last stage where they do not fill it, else 0 (of the last range only).
__device__ __forceinline__ int ragged_tail(const Product& a, int split) {
    return split == a.splits - 1 ? (int)(a.C % BC) : 0;
}

// WQ x WP waves of 16 TI x 16 TJ outputs each; a ring of NSTG stages, one barrier a stage. The fragments of the next
// step are read while this one's multiply.
template <int TYPE, bool QM, bool PM, int TI, int TJ, int WQ, int WP, int NSTG>
__global__ void __launch_bounds__(64 * WQ * WP, NSTG * 16 * BC * 2 * (TI * WQ + TJ * WP) <= 81920 ? 2 : 1)
    product_tile_kernel(const Product a, int tiles_q, int tiles_p) {
    typedef typename Half<TYPE>::x8 T8;
    constexpr int W = WQ * WP, QR = 16 * TI * WQ, PR = 16 * TJ * WP;
    typedef Operand<QM, QR, W> OQ;
    typedef Operand<PM, PR, W> OP;
    constexpr int STG_Q = 2 * BC * QR, STG = STG_Q + 2 * BC * PR, LD = OQ::N + OP::N;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[NSTG * STG];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int split, tq, tp;
    place_of(a, tiles_q, tiles_p, split, tq, tp);
    const long long q0 = (long long)tq * QR, p0 = (long long)tp * PR;
    const long long all = (a.C + BC - 1) / BC, s0 = all * split / a.splits;
    const int nst = (int)(all * (split + 1) / a.splits - s0);
    OQ oq;
    OP op;
    oq.init(a.Q, a.ldq, a.nq, a.C, q0, s0 * BC, nst, lane, wave);
    op.init(a.P, a.ldp, a.np, a.C, p0, s0 * BC, nst, lane, wave);
    auto issue = [&](uint8_t* to) {
#pragma unroll
        for (int j = 0; j < OQ::N; j++) oq.copy(to, j, wave);
#pragma unroll
        for (int j = 0; j < OP::N; j++) op.copy(to + STG_Q, j, wave);
        oq.next();
        op.next();
    };
    const int wq = wave / WP, wp = wave % WP;
    const int lq = OQ::lane_offset(lane), lp = OP::lane_offset(lane);
    f32x4 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; i++)
#pragma unroll
        for (int j = 0; j < TJ; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    const int tail = ragged_tail(a, split);
    // Stage k, at `at`, has landed for every wave: all but the copies of the NSTG - 2 stages behind it are complete (in the
    // beginning, of NSTG - 1); this wave's reads before are too.
    auto landed = [&](auto LEFT, int k, uint8_t* at) {
        wait_vmcnt_lgkm0<LD * decltype(LEFT)::value>();
        stage_barrier();
        if (!(QM && PM) && tail && k == nst - 1) {
            OQ::zero_tail(at, tail, threadIdx.x);
            OP::zero_tail(at + STG_Q, tail, threadIdx.x);
            wait_vmcnt_lgkm0<LD * decltype(LEFT)::value>();
            stage_barrier();
        }
    };
    T8 fq[2][TI], fp[2][TJ];
    auto read = [&](const uint8_t* at, int h) {
#pragma unroll
        for (int i = 0; i < TI; i++) fq[h][i] = OQ::template fragment<T8>(at, h, wq * TI + i, lq);
#pragma unroll
        for (int j = 0; j < TJ; j++) fp[h][j] = OP::template fragment<T8>(at + STG_Q, h, wp * TJ + j, lp);
    };
    auto multiply = [&](int h) {
#pragma unroll
        for (int i = 0; i < TI; i++)
#pragma unroll
            for (int j = 0; j < TJ; j++) acc[i][j] = Half<TYPE>::mfma(fp[h][j], fq[h][i], acc[i][j]);
    };
#pragma unroll
    for (int s = 0; s < NSTG; s++) issue(lds + s * STG);
    landed(std::integral_constant<int, NSTG - 1>{}, 0, lds);
    read(lds, 0);
    // The two steps of stage k. Before the second one multiplies stage k + 1 has landed, and behind that barrier nobody reads
    // stage k's buffer any more, which stage k + NSTG takes.
    uint8_t* at = lds;
    for (int k = 0; k < nst; k++) {
        uint8_t* next = at + STG == lds + NSTG * STG ? lds : at + STG;
        read(at, 1);
        multiply(0);
        landed(std::integral_constant<int, NSTG - 2>{}, k + 1, next);
        issue(at);
        read(next, 0);
        multiply(1);
        at = next;
    }
    wait_vmcnt<0>();
    __syncthreads();
    constexpr int ROOM = NSTG * STG / W / 4;
    put_sums<TYPE, TI, TJ, ROOM>(a, acc, reinterpret_cast<float*>(lds) + wave * ROOM, lane, split, q0 + 16 * wq * TI, p0 + 16 * wp * TJ);
}

// c += a b with c in accumulation registers. Left to itself the compiler moves sums between the two halves of the
// register file inside the loop (up to 184 moves for its 128 matrix instructions); written so, c stays. Nothing else
// touches the registers while the loop runs, the same c comes up every 64 instructions, and settle_sums() stands
// between the loop and the first use of the sums, so that no result is read early.
template <int TYPE>
__device__ __forceinline__ void mfma_acc(f32x4& c, typename Half<TYPE>::x8 a, typename Half<TYPE>::x8 b) {
    if constexpr (TYPE == OZ_BF16) asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void settle_sums() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// 256 x 256 outputs by 4 waves of 128 x 128, one a SIMD, each with 256 sums' registers. The fragments of the next
// step are read while this one's multiply, one or two reads per four matrix instructions. LDS holds five operands'
// stages, two of each and a spare: the copies of stage k + 2 of Q go out in stage k's first step and those of P in its second,
// where Q's stage k is free, and have one and a half or two and a half steps to land. (With two whole stages all copies go out
// in the second step and have one and a half: 852 against 763 us at 8192^3.)
template <int TYPE, bool QM, bool PM>
__global__ void __launch_bounds__(256) product_big_kernel(const Product a, int tiles_q, int tiles_p) {
    typedef typename Half<TYPE>::x8 T8;
    typedef Operand<QM, 256, 4> OQ;
    typedef Operand<PM, 256, 4> OP;
    constexpr int UNIT = 2 * BC * 256, RING = 5 * UNIT, LD = OQ::N;
    static_assert(OQ::N == OP::N, "copies of a unit");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[RING];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int split, tq, tp;
    place_of(a, tiles_q, tiles_p, split, tq, tp);
    const long long q0 = 256ll * tq, p0 = 256ll * tp;
    const long long all = (a.C + BC - 1) / BC, s0 = all * split / a.splits;
    const int nst = (int)(all * (split + 1) / a.splits - s0);
    OQ oq;
    OP op;
    oq.init(a.Q, a.ldq, a.nq, a.C, q0, s0 * BC, nst, lane, wave);
    op.init(a.P, a.ldp, a.np, a.C, p0, s0 * BC, nst, lane, wave);
    const int wq = wave >> 1, wp = wave & 1;
    const int lq = OQ::lane_offset(lane), lp = OP::lane_offset(lane);
    f32x4 acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    const int tail = ragged_tail(a, split);
    // Unit 2 k is Q's stage k, unit 2 k + 1 P's; unit u is at u UNIT modulo RING.
    auto landed = [&](auto LEFT, int k, int uq, int up) {  // stage k, whose units are at uq and up
        wait_vmcnt_lgkm0<decltype(LEFT)::value>();
        stage_barrier();
        if (!(QM && PM) && tail && k == nst - 1) {
            OQ::zero_tail(lds + uq, tail, threadIdx.x);
            OP::zero_tail(lds + up, tail, threadIdx.x);
            wait_vmcnt_lgkm0<decltype(LEFT)::value>();
            stage_barrier();
        }
    };
#pragma unroll
    for (int s = 0; s < 2; s++) {
#pragma unroll
        for (int j = 0; j < LD; j++) oq.copy(lds + 2 * s * UNIT, j, wave);
#pragma unroll
        for (int j = 0; j < LD; j++) op.copy(lds + (2 * s + 1) * UNIT, j, wave);
        oq.next();
        op.next();
    }
    T8 fq[8], fp[8], gq[8], gp[8];
    landed(std::integral_constant<int, 2 * LD>{}, 0, 0, UNIT);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        fq[i] = OQ::template fragment<T8>(lds, 0, wq * 8 + i, lq);
        fp[i] = OP::template fragment<T8>(lds + UNIT, 0, wp * 8 + i, lp);
    }
    // One step: 64 matrix instructions on (xq, xp); the 16 fragments (yq, yp) of step H of the units at uq and up, in the order
    // their instructions want them; the copies of a unit of Q (in a stage's first step) or P to `to`.
    auto step = [&](auto H, T8* xq, T8* xp, T8* yq, T8* yp, int uq, int up, int to) {
        constexpr int h = decltype(H)::value;
        const uint8_t *rq = lds + uq, *rp = lds + up;
#pragma unroll
        for (int n = 0; n < 64; n++) {
            const int i = n >> 3, j = n & 7;
            mfma_acc<TYPE>(acc[i][j], xp[j], xq[i]);
            if (n % 4 == 0) {
                const int t = n / 4;
                if (t == 0) yq[0] = OQ::template fragment<T8>(rq, h, wq * 8, lq);
                else if (t <= 8) yp[t - 1] = OP::template fragment<T8>(rp, h, wp * 8 + t - 1, lp);
                else yq[t - 8] = OQ::template fragment<T8>(rq, h, wq * 8 + t - 8, lq);
            }
            if (n % 4 == 2 && n / 4 < LD) {
                if constexpr (h == 1) oq.copy(lds + to, n / 4, wave);
                else op.copy(lds + to, n / 4, wave);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The two steps of stage k. Before the second one stage k + 1 has landed and every wave has read all of stage k. What
    // is read behind the last stage is not used.
    int at = 0;
    auto wrap = [](int b) { return b >= RING ? b - RING : b; };
    for (int k = 0; k < nst; k++) {
        const int u1 = wrap(at + UNIT), u2 = wrap(at + 2 * UNIT), u3 = wrap(at + 3 * UNIT), u4 = wrap(at + 4 * UNIT);
        step(std::integral_constant<int, 1>{}, fq, fp, gq, gp, at, u1, u4);
        oq.next();
        landed(std::integral_constant<int, LD>{}, k + 1, u2, u3);
        step(std::integral_constant<int, 0>{}, gq, gp, fq, fp, u2, u3, at);
        op.next();
        at = u2;
    }
    settle_sums();
    wait_vmcnt<0>();
    __syncthreads();
    constexpr int ROOM = RING / 4 / 4;
    put_sums<TYPE, 8, 8, ROOM>(a, acc, reinterpret_cast<float*>(lds) + wave * ROOM, lane, split, q0 + 128 * wq, p0 + 128 * wp);
}

}  // namespace ozl
