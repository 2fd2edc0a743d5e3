// Products with an epilogue: what the kernels of oz_linear*.hip take.
#pragma once
#include "oz_types.hpp"

namespace ozl {

// v = sum + bias[p]; Z(q, p) = v; Y(q, p) = act(v) + residual(q, p), or added to Y with accumulate.
struct Epilogue {
    void* Y;
    long long ldy;
    int y_type;
    void* Z;
    long long ldz;
    const void* bias;
    const void* residual;
    long long ldr;
    int act, accumulate;
};

// C(q, p) = sum over c < C of Q(q, c) P(p, c), q < nq, p < np. Q(q, c) is at q ldq + c, or at c ldq + q where
// q_major; P alike.
struct Product {
    const void *Q, *P;
    long long nq, np, C, ldq, ldp;
    int q_major, p_major;
    Epilogue epi;
};

// One value. bias, Z in the operands' type, residual and Y in y_type.
__device__ __forceinline__ void finish(const Epilogue& e, int type, long long q, long long p, float v) {
    if (e.bias) v += ozt::load(e.bias, type, p);
    if (e.Z) ozt::store(e.Z, type, q * e.ldz + p, v);
    v = ozt::act(v, e.act);
    if (e.residual) v += ozt::load(e.residual, e.y_type, q * e.ldr + p);
    if (e.accumulate) v += ozt::load(e.Y, e.y_type, q * e.ldy + p);
    ozt::store(e.Y, e.y_type, q * e.ldy + p, v);
}

}  // namespace ozl
