// Products of the Newton-Schulz iteration (oz_newton_schulz.hpp).
#include "oz_internal.hpp"
#include "oz_newton_schulz.hpp"

namespace {

using namespace ozt;
using namespace ozn;

enum Phase { GRAM, SQUARE, UPDATE, LAST };  // A, B, X, the result

struct Pass {
    Places places;
    Factors f;
    int from;  // X's buffer, its values go to the other one
};

__device__ __forceinline__ void put_parts(_Float16* h, _Float16* l, long long at, float v) {
    const _Float16 x = (_Float16)v;
    h[at] = x;
    if (l) l[at] = (_Float16)(v - (float)x);
}

template <int PHASE>
__device__ __forceinline__ void finish(const Shape& s, const Ends& e, const Factors& f, int from, int i, int q, int p, float v) {
    const int side = side_of(s);
    const long long nn = (long long)side * side;
    if constexpr (PHASE == GRAM) {
        _Float16* a = square_of(s, s.a, i);
        put_parts(a, s.three ? a + nn : nullptr, (long long)q * side + p, v * (1.0f / kScale / kScale));
    } else if constexpr (PHASE == SQUARE) {
        const _Float16* a = square_of(s, s.a, i);
        _Float16* b = square_of(s, s.b, i);
        const long long at = (long long)q * side + p;
        float x = (float)a[at];
        if (s.three) x += (float)a[nn + at];
        put_parts(b, s.three ? b + nn : nullptr, at, f.b * x + f.c * v);
    } else {
        const long long at = (long long)q * s.C + p;
        const float x = f.a * ((float)h_of(s, from, i)[at] + (float)l_of(s, from, i)[at]) + v;
        if constexpr (PHASE == UPDATE) {
            put_parts(h_of(s, from ^ 1, i), l_of(s, from ^ 1, i), at, x);
        } else if (q < s.rows && p < s.cols) {
            const float o = x * (1.0f / kScale);
            if (e.tensors) {
                const oz_muon_tensor& t = e.tensors[s.first + i];
                const long long to = (long long)q * s.cols + p;
                const float old = t.master ? t.master[to] : load(t.param, t.param_type, to);
                const float now = old * (1.0f - e.lr * t.weight_decay) - o * (e.lr * t.lr_scale);
                if (t.master) t.master[to] = now;
                store(t.param, t.param_type, to, now);
            } else {
                store(e.O, e.type, (s.first + i) * e.stride_o + q * e.ldo + p, o);
            }
        }
    }
}

// 64 x 64 values by 4 waves of 32 x 32, operands through LDS, 32 of c at a time.
template <int PHASE>
__global__ void __launch_bounds__(256) product_kernel(const Shapes m, const Ends ends, const Pass pass) {
    constexpr int LD = 40;  // 16-byte rows, on other banks each
    __shared__ __attribute__((aligned(16))) _Float16 lq[64 * LD], lp[64 * LD];
    const Place w = place_of(pass.places, m.n, blockIdx.x);
    const Shape& s = m.s[w.shape];
    const int side = side_of(s), tall = is_tall(s);
    const int across = (PHASE == GRAM || PHASE == SQUARE ? side : s.C) / 64, q0 = 64 * (w.index / across), p0 = 64 * (w.index % across);
    const long long nx = (long long)s.R * s.C, nn = (long long)side * side;
    // X' = a X + B X, or a X + X B: (q, c) of one operand, (c, p) of the other; B is symmetric
    const _Float16 *Q, *P;
    long long q_plane = nx, p_plane = nx;
    int C, q_row, q_col, p_row, p_col;  // strides of an operand's own index and of c
    if constexpr (PHASE == GRAM) {
        Q = P = h_of(s, pass.from, w.matrix);
        C = tall ? s.R : s.C;
        q_row = p_row = tall ? 1 : s.C, q_col = p_col = tall ? s.C : 1;
    } else if constexpr (PHASE == SQUARE) {
        Q = P = square_of(s, s.a, w.matrix);
        C = q_row = p_row = side, q_col = p_col = 1;
        q_plane = p_plane = nn;
    } else {
        const _Float16 *x = h_of(s, pass.from, w.matrix), *b = square_of(s, s.b, w.matrix);
        C = side;
        Q = tall ? x : b, P = tall ? b : x;
        q_row = tall ? s.C : side, q_col = 1;
        p_row = tall ? side : 1, p_col = tall ? 1 : s.C;
        (tall ? p_plane : q_plane) = nn;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wq = 32 * (wave >> 1), wp = 32 * (wave & 1), r = lane & 15, g = lane >> 4;
    f32x4 acc[2][2] = {};
    for (int part = 0; part < (s.three ? 3 : 1); part++) {  // h h, h l, l h
        const _Float16 *Qs = Q + (part == 2 ? q_plane : 0), *Ps = P + (part == 1 ? p_plane : 0);
        for (int c0 = 0; c0 < C; c0 += 32) {
            for (int e = threadIdx.x; e < 64 * 32; e += 256) {
                const int cq = q_col == 1 ? e & 31 : e >> 6, iq = q_col == 1 ? e >> 5 : e & 63;
                const int cp = p_col == 1 ? e & 31 : e >> 6, ip = p_col == 1 ? e >> 5 : e & 63;
                lq[iq * LD + cq] = Qs[(long long)(q0 + iq) * q_row + (long long)(c0 + cq) * q_col];
                lp[ip * LD + cp] = Ps[(long long)(p0 + ip) * p_row + (long long)(c0 + cp) * p_col];
            }
            __syncthreads();
            f16x8 fq[2], fp[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                fq[i] = *reinterpret_cast<const f16x8*>(lq + (wq + 16 * i + r) * LD + 8 * g);
                fp[i] = *reinterpret_cast<const f16x8*>(lp + (wp + 16 * i + r) * LD + 8 * g);
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = Half<OZ_F16>::mfma(fp[j], fq[i], acc[i][j]);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int k = 0; k < 4; k++) finish<PHASE>(s, ends, pass.f, pass.from, w.matrix, q0 + wq + 16 * i + r, p0 + wp + 16 * j + 4 * g + k, acc[i][j][k]);
}

// The workgroups of a launch of 64 x 64 tiles, or 0 where they are too many.
long long places(const Shapes& m, bool square, Places* p) {
    long long at = 0;
    for (int k = 0; k < m.n; k++) {
        const Shape& s = m.s[k];
        const long long side = side_of(s) / 64, per = square ? side * side : (long long)(s.R / 64) * (s.C / 64);
        if (per >> 24 || at + per * s.count >= 1 << 24) return -1;
        p->first[k] = (int)at;
        p->per[k] = (int)per;
        at += per * s.count;
    }
    p->first[m.n] = (int)at;
    return at;
}

}  // namespace

int ozn::iterate(oz_dev* dev, const Shapes& m, const Ends& ends, const Factors& f, int steps) {
    Pass square{}, whole{};
    square.f = whole.f = f;
    const long long ns = places(m, true, &square.places), nw = places(m, false, &whole.places);
    if (ns < 0 || nw < 0) return oz::fail(dev, OZ_ERR_ARG, "too many values in matrices");
    for (int k = 0; k < steps; k++) {
        square.from = whole.from = k & 1;
        hipLaunchKernelGGL(product_kernel<GRAM>, dim3((unsigned)ns), dim3(256), 0, dev->stream, m, ends, square);
        hipLaunchKernelGGL(product_kernel<SQUARE>, dim3((unsigned)ns), dim3(256), 0, dev->stream, m, ends, square);
        if (k + 1 < steps) hipLaunchKernelGGL(product_kernel<UPDATE>, dim3((unsigned)nw), dim3(256), 0, dev->stream, m, ends, whole);
        else hipLaunchKernelGGL(product_kernel<LAST>, dim3((unsigned)nw), dim3(256), 0, dev->stream, m, ends, whole);
        if (int st = oz::launch_check(dev, "Newton-Schulz product")) return st;
    }
    return OZ_OK;
}
