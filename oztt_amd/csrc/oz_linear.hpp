// Products with an epilogue: what the kernels of oz_linear*.hip take.
#pragma once
#include "oz_types.hpp"

struct oz_dev;

namespace ozl {

// v = sum + bias[p]; Z(q, p) = v; Y(q, p) = act(v) + residual(q, p). The residual may be Y itself.
struct Epilogue {
    void* Y;
    long long ldy;
    int y_type;
    void* Z;
    long long ldz;
    const void* bias;
    const void* residual;
    long long ldr;
    int act;
};

// C(q, p) = sum over c < C of Q(q, c) P(p, c), q < nq, p < np. Q(q, c) is at q ldq + c, or at c ldq + q where
// q_major; P alike. With splits > 1 range s of c goes to parts + s nq ldparts as FP32, for join_kernel.
struct Product {
    const void *Q, *P;
    long long nq, np, C, ldq, ldp;
    int q_major, p_major;
    Epilogue epi;
    float* parts;
    long long ldparts;
    int splits;
};

// The same of 8-bit integers, sums in int32 (parts too): what goes to the epilogue is sum p_scale[p] q_scale[q]. Sizes along c
// count pairs of integers; Z is not taken.
struct ScaledProduct : Product {
    const float *q_scale, *p_scale;
    int K;         // integers along c
    int type;      // oz_type of the bias
    bool q_zeros;  // zeros behind the K integers of Q's rows, to the end of a stage
};

// Eight sums in a row from p on to values, of those below np.
__device__ __forceinline__ void scale8(const ScaledProduct& a, long long q, long long p, float* v) {
    const float s = a.q_scale[q];
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (p + k < a.np) v[k] = (float)__float_as_int(v[k]) * a.p_scale[p + k] * s;
}

// One value. bias, Z in the operands' type, residual and Y in y_type.
__device__ __forceinline__ void finish(const Epilogue& e, int type, long long q, long long p, float v) {
    if (e.bias) v += ozt::load(e.bias, type, p);
    if (e.Z) ozt::store(e.Z, type, q * e.ldz + p, v);
    v = ozt::act(v, e.act);
    if (e.residual) v += ozt::load(e.residual, e.y_type, q * e.ldr + p);
    ozt::store(e.Y, e.y_type, q * e.ldy + p, v);
}

// Eight values in a row from p on, of them those below np. Everything is read before anything is written: with one
// wave on a SIMD every wait for memory counts.
template <int TYPE>
__device__ __forceinline__ void finish8(const Epilogue& e, long long np, long long q, long long p, float* v) {
    const int count = p + 8 <= np ? 8 : (int)(np - p);
    float b[8] = {}, r[8] = {};
    if (count == 8) {
        if (e.bias) ozt::load8(e.bias, TYPE, p, b);
        if (e.residual) ozt::load8(e.residual, e.y_type, q * e.ldr + p, r);
    } else {
        if (e.bias) ozt::load_some(e.bias, TYPE, p, count, b);
        if (e.residual) ozt::load_some(e.residual, e.y_type, q * e.ldr + p, count, r);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] += b[k];
    if (e.Z) {
        if (count == 8) ozt::store8(e.Z, TYPE, q * e.ldz + p, v);
        else ozt::store_some(e.Z, TYPE, q * e.ldz + p, count, v);
    }
    ozt::act8(v, e.act);
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] += r[k];
    if (count == 8) ozt::store8(e.Y, e.y_type, q * e.ldy + p, v);
    else ozt::store_some(e.Y, e.y_type, q * e.ldy + p, count, v);
}

// Tiles of a product whose operands' rows begin at multiples of 4 bytes; rows x columns of outputs.
enum Tile { T256, T128, T64, T64X32, T32, TILES };
struct Shape {
    int q, p;            // outputs
    int threads;         // of a workgroup
    int per_cu;          // workgroups that a CU holds (LDS)
    float alone, full;   // us for a stage of 64 values of c: one workgroup on a CU, per_cu of them
    float fixed;         // us from the first copy to the first product, and from the last to the outputs
};
// Fitted to times of passes over the same operands on 256 CUs in BF16: 4096^2 of K = 256 and 1024 and 8192^2 of 512 by 256 x 256 tiles (25.8, 42.8 and 124 us) and
// by 128 x 128 (18.4, 38.5 and 101), 2048^2 of K = 512 and 2048 by 128 x 128 (10.2, 24.1; one workgroup a CU) and by 64 x 64 (13.2,
// 28.7), 1024^3 by 64 x 64 (7.5), 64 rows of 2048^2 by 32 x 32.
inline const Shape& shape_of(Tile t) {
    static const Shape shapes[TILES] = {
        {256, 256, 256, 1, 1.42f, 1.42f, 20.0f}, {128, 128, 512, 2, 0.58f, 0.85f, 5.8f}, {64, 64, 256, 2, 0.21f, 0.32f, 4.0f},
        {64, 32, 128, 2, 0.20f, 0.28f, 3.9f},    {32, 32, 128, 2, 0.18f, 0.22f, 3.4f}};
    return shapes[t];
}
// A launch takes fewer than 2^32 threads along a dimension of its grid. The products of 2^31 - 1 rows that memory holds fit it with
// the largest tile.
inline long long tiles_of(const Shape& t, long long nq, long long np, int splits) { return (nq + t.q - 1) / t.q * ((np + t.p - 1) / t.p) * splits; }
inline bool fits(const Shape& t, long long nq, long long np, int splits) { return tiles_of(t, nq, np, splits) * t.threads < 1ll << 32; }
// How a product runs, from its sizes alone: `contiguous` operands along c, whose rows all begin at `even` addresses.
struct Route {
    bool few;       // the kernels of few rows
    Tile tile;
    int splits;
    size_t parts;   // bytes of the ranges' sums
};
// Up to `streamed` rows have a kernel of their own, which takes no ranges.
constexpr int kStreamRows = 2;
Route route_of(int cus, long long nq, long long np, long long C, bool contiguous, bool even, int streamed = kStreamRows);
int launch_tile(oz_dev* dev, int type, Tile tile, const Product& a);
// At most 32 rows of Q, operands along c at any address; splits as in Product (1 for at most kStreamRows). A workgroup has
// few_rows_block rows of P.
inline int few_rows_block(long long nq) { return nq <= 16 ? 16 : 32; }
int launch_few_rows(oz_dev* dev, int type, const Product& a);
// Joins the ranges of c in order.
int launch_join(oz_dev* dev, int type, const Product& a);

}  // namespace ozl
