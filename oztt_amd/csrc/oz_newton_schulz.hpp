// The Newton-Schulz iteration over matrices of several sizes at once: what its kernels take (oz_muon.hip, oz_newton_schulz.hip).
//
//   X0 = U / (|U|_F + eps);  A = X X^T,  B = b A + c A^2,  X <- a X + B X, `steps` times
//
// and from the right (A = X^T X, X <- a X + X B) where a matrix has more rows than columns, so that A has the shorter side.
// Every singular value s of X0 goes through s <- a s + b s^3 + c s^5; with the usual factors all but the smallest end within 0.7
// to 1.2.
//
// X is held as two FP16 parts, X = h + l, times kScale: together 22 bits. The products read h alone, the term a X both. A gradient has
// a few strong directions and many weak ones that each step makes a times larger, so what rounding does to X there
// grows with them: with X in BF16 the result is off by 1e-2 of its norm for a Gaussian matrix and by 0.2 to 0.6 for one of
// low rank, in FP16 by 1e-3 and 2e-2 to 7e-2. The products do not have that weakness, as B is nearly zero in the directions of small
// singular values. Once most of them are near 1, B is near -2.7 times the identity, and rounding h and B to 11 bits is what shows:
// B's diagonal is therefore kept in FP32 and multiplies both parts of X in the product's epilogue, X <- (a + diag B) X + (B - diag B) h,
// which costs 1% (for Gaussian matrices of 513 to 1500 rows off by 1.3e-3 to 1.8e-3 without it, 4e-4 to 8.5e-4 with it). The
// result is off by 2e-4 to 1.5e-3 where values differ (against 64 bits). Where rows or values do not, their roundings do not average: an identity of
// 513 rows by up to 5e-3, equal rows and matrices of one value by 3e-3 to 8e-3, some blocks of one value by 1.8e-2; to first order by up to 6.2e-2.
// Where a side is short (the rounding errors of A and B then average over few values: up to 1e-2 at one to four rows) or the result
// is kept in more than BF16's 8 bits, or the caller asks for it, the products take both parts of both operands, h h + h l + l h: off by 1e-6 to 4e-6,
// and by up to 3e-4 where thousands of values are alike and so are the roundings of their FP32 sums.
#pragma once
#include <hip/hip_runtime.h>

#include "oz_types.hpp"

struct oz_dev;

namespace ozn {

constexpr float kScale = 4096.0f;  // X's values are at most about 1: 16 times as large ones still are FP16 numbers
// A and B are kept times powers of two as well (Factors), as large as the singular values' range allows: their values are about the side's
// reciprocal, and FP16 ends at 2^-24, so that second parts of unscaled ones had lost most of their bits (FP32 matrices of four blocks of one value, 1020 x 672: off
// by 7.3e-5 of their norm, 5.5e-6 with the scales; with a gradient's spectrum, 4096^2, 3.7e-6 and 1.9e-6, for 3% of the time).
constexpr double kLargest = 32768.0;  // of them, half of FP16's
constexpr double kMaxSingular = 8.0;  // what callers promise
constexpr int kPad = 64;           // sides in the workspace are multiples of it, the rest zeros, which the iteration keeps
constexpr int kShapes = OZ_MUON_SHAPES;
// Up to this shorter side the products take both parts of X. There launches and their latency count more than products: 64^2 takes 74 us
// for 70, 256 x 1024 130 for 98, 512^2 132 for 101, twelve of 512 x 2048 496 for 308; 1024^2 188 for 140 and twelve 933 for 466.
constexpr int kThreeSide = 512;

// `count` matrices of one size. Buffers hold them one after the other, each as one plane of R x C (h) or two (h, l).
struct Shape {
    int rows, cols;  // of a matrix
    int R, C;        // in the workspace
    int count, first;
    int three;       // products of both parts
    int chunks;      // of a matrix, for the sum of its squares
    _Float16 *x[2], *l, *a, *b;
    float* d;        // products of the first parts: B's diagonals, where b has zeros
    double* sums;
};
struct Shapes {
    int n;
    Shape s[kShapes];
};
// A launch's workgroups: per[s] for each matrix of shape s, the first of shape s is first[s].
struct Places {
    int first[kShapes + 1], per[kShapes];
};
struct Place {
    int shape, matrix, index;
};
__device__ __forceinline__ int shape_of(const Places& p, int n, int w) {
    int s = 0;
    while (s + 1 < n && w >= p.first[s + 1]) s++;
    return s;
}
__device__ __forceinline__ Place place_of(const Places& p, int n, int w) {
    const int s = shape_of(p, n, w), i = w - p.first[s];
    return {s, i / p.per[s], i % p.per[s]};
}

__host__ __device__ inline int side_of(const Shape& s) { return s.R < s.C ? s.R : s.C; }
__host__ __device__ inline bool is_tall(const Shape& s) { return s.rows > s.cols; }
__device__ __forceinline__ _Float16* h_of(const Shape& s, int b, int i) { return (b ? s.x[1] : s.x[0]) + (long long)(1 + s.three) * i * s.R * s.C; }
__device__ __forceinline__ _Float16* l_of(const Shape& s, int b, int i) {
    const long long n = (long long)s.R * s.C;
    return s.three ? (b ? s.x[1] : s.x[0]) + (2 * i + 1) * n : s.l + i * n;
}
// A or B of a matrix
__device__ __forceinline__ _Float16* square_of(const Shape& s, _Float16* p, int i) { return p + (long long)(1 + s.three) * i * side_of(s) * side_of(s); }

__device__ __forceinline__ float* diagonal_of(const Shape& s, int i) { return s.d + (long long)i * side_of(s); }

// Where the matrices come from and the results go: one array each (orthogonalize), or a list of tensors (Muon).
struct Ends {
    const void* G;
    void* O;
    int type;
    long long ldg, ldo, stride_g, stride_o;
    const oz_muon_tensor* tensors;
    float momentum, fresh, lr;  // fresh = 1 - momentum
    int nesterov;
    const float* grad_scale;
};
// The iteration's factors with the scales of what they multiply and of what becomes of it: X <- a X + update B X, B = b A + c A^2, A = gram X X^T.
struct Factors {
    float a, b, c, update, gram;
};

// The products of a step. X' goes to the ends in the last one.
enum Phase { GRAM, SQUARE, UPDATE };
struct Pass {
    Places places;       // per: tiles of `parent` x `parent` outputs
    int parent;
    int begin[kShapes];  // of a shape's tiles, the first that the launch has
    Factors f;
    int from;  // X's buffer, its values go to the other one
    int last;
};
// Tiles of `tile` x `tile` outputs of a phase's products, 64, 128 or (of the first parts) 256, for shapes that are alike in `three`.
template <bool THREE>
void launch_products(hipStream_t stream, Phase phase, int tile, const Shapes& m, const Ends& ends, const Pass& pass);

Factors factors_of(double a, double b, double c, int steps);

// The launches of a step, of the shapes whose products take one part of their operands and of those that take both: prepared, and
// refused where they are too many, before anything runs.
struct Launches {
    Shapes order[3];  // the shapes as a phase's sequence of tiles has them
    Pass pass[3][2];
    int tile[3][2];
};
struct Iteration {
    Launches of[2];
};
int prepare(oz_dev* dev, const Shapes& m, const Factors& f, Iteration* it);
// The iteration on X0 in the shapes' x[0] (and l), the last step's results to the ends.
int iterate(oz_dev* dev, Iteration* it, const Ends& ends, int steps);

}  // namespace ozn
