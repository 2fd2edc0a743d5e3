// Launches of the tiled products (oz_linear_tiles.hpp).
#include "oz_internal.hpp"
#include "oz_linear_tiles.hpp"

namespace {

using namespace ozl;

// Joins the ranges of c in order.
template <int TYPE>
__global__ void __launch_bounds__(256) join_kernel(const Product a) {
    const long long across = (a.np + 7) / 8, i = 256ll * blockIdx.x + threadIdx.x;
    const long long q = i / across, p = 8 * (i % across);
    if (q >= a.nq) return;
    float v[8], x[8];
    load8(a.parts, OZ_F32, q * a.ldparts + p, v);
#pragma unroll 8
    for (int s = 1; s < a.splits; s++) {
        load8(a.parts, OZ_F32, (s * a.nq + q) * a.ldparts + p, x);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] += x[k];
    }
    finish8<TYPE>(a.epi, a.np, q, p, v);
}

template <int TYPE, bool QM, bool PM, int TI, int TJ, int WQ, int WP, int NSTG>
int launch(oz_dev* dev, const Product& a) {
    const int tiles_q = (int)oz::ceil_div(a.nq, 16 * TI * WQ), tiles_p = (int)oz::ceil_div(a.np, 16 * TJ * WP);
    const dim3 grid((unsigned)tiles_q * tiles_p * a.splits), block(64 * WQ * WP);
    hipLaunchKernelGGL((product_tile_kernel<TYPE, QM, PM, TI, TJ, WQ, WP, NSTG>), grid, block, 0, dev->stream, a, tiles_q, tiles_p);
    if (int st = oz::launch_check(dev, "product_tile_kernel")) return st;
    return a.splits > 1 ? ozl::launch_join(dev, TYPE, a) : OZ_OK;
}

template <int TYPE, bool QM, bool PM>
int launch_big(oz_dev* dev, const Product& a) {
    const int tiles_q = (int)oz::ceil_div(a.nq, 256), tiles_p = (int)oz::ceil_div(a.np, 256);
    hipLaunchKernelGGL((product_big_kernel<TYPE, QM, PM>), dim3((unsigned)tiles_q * tiles_p * a.splits), dim3(256), 0, dev->stream, a, tiles_q, tiles_p);
    if (int st = oz::launch_check(dev, "product_big_kernel")) return st;
    return a.splits > 1 ? ozl::launch_join(dev, TYPE, a) : OZ_OK;
}

template <int TYPE, bool QM, bool PM>
int by_tile(oz_dev* dev, Tile t, const Product& a) {
    switch (t) {
        case T256: return launch_big<TYPE, QM, PM>(dev, a);
        case T128: return launch<TYPE, QM, PM, 2, 4, 4, 2, 2>(dev, a);
        case T64: return launch<TYPE, QM, PM, 2, 2, 2, 2, 4>(dev, a);
        case T64X32: return launch<TYPE, QM, PM, 2, 2, 2, 1, 6>(dev, a);
        default: return launch<TYPE, QM, PM, 1, 2, 2, 1, 8>(dev, a);
    }
}

template <int TYPE>
int by_layout(oz_dev* dev, Tile t, const Product& a) {
    if (a.q_major) return by_tile<TYPE, true, true>(dev, t, a);
    return a.p_major ? by_tile<TYPE, false, true>(dev, t, a) : by_tile<TYPE, false, false>(dev, t, a);
}

}  // namespace

int ozl::launch_tile(oz_dev* dev, int type, Tile tile, const Product& a) {
    return type == OZ_BF16 ? by_layout<OZ_BF16>(dev, tile, a) : by_layout<OZ_F16>(dev, tile, a);
}

int ozl::launch_join(oz_dev* dev, int type, const Product& a) {
    const dim3 grid(oz::ceil_div(a.nq * ((a.np + 7) / 8), 256)), block(256);
    if (type == OZ_BF16) hipLaunchKernelGGL(join_kernel<OZ_BF16>, grid, block, 0, dev->stream, a);
    else hipLaunchKernelGGL(join_kernel<OZ_F16>, grid, block, 0, dev->stream, a);
    return oz::launch_check(dev, "join_kernel");
}
