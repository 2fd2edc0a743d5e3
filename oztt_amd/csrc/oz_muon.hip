// Orthogonalized matrices and Muon's step (include/oz_hip.h, oz_orthogonalize and oz_muon_step): what stands before the
// iteration's products (oz_newton_schulz.hip).
//
// The first pass reads gradients and momenta, writes the momenta and sums the squares of what is to be orthogonalized, the
// second reads them again and writes X0 = U / (|U| + eps) in two FP16 parts with the padding's zeros. Both are bound by memory:
// 10 bytes a value each with an FP32 momentum and a BF16 gradient.
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

#include "oz_internal.hpp"
#include "oz_newton_schulz.hpp"

namespace {

using namespace ozt;
using namespace ozn;

constexpr int THREADS = 256, V = 8;
constexpr int kChunk = V * THREADS;      // least values of a chunk
constexpr int kMaxChunks = 512;          // of a matrix: each workgroup of the second pass adds them all
constexpr int kRounds = 8;               // pieces of a thread in the second pass, where they are many

// Eight values in a row, `count` of them there.
__device__ __forceinline__ void get(const void* p, int type, long long i, int count, float* x) {
    if (count == V) load8(p, type, i, x);
    else load_some(p, type, i, count, x);
}

// The sum of v over the workgroup, in every thread, in an order that does not change.
__device__ __forceinline__ double sum_all(double v) {
    __shared__ double part[THREADS / 64];
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
    if (!(threadIdx.x & 63)) part[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = part[0];
#pragma unroll
    for (int k = 1; k < THREADS / 64; k++) s += part[k];
    return s;
}

__device__ __forceinline__ void update_of(const Ends& e, const float* m, const float* g, float gs, float* u) {
#pragma unroll
    for (int k = 0; k < V; k++) u[k] = e.nesterov ? e.momentum * m[k] + e.fresh * (g[k] * gs) : m[k];
}

// Muon: m' and the sum of the squares of u; else the sum of the squares of G.
__global__ void __launch_bounds__(THREADS) squares_kernel(const Shapes shapes, const Ends e, const Places places) {
    const Place w = place_of(places, shapes.n, blockIdx.x);
    const Shape& s = shapes.s[w.shape];
    const long long step = (long long)THREADS * s.chunks;  // pieces that all chunks take in a round
    double sum = 0.0;
    auto add = [&](const float* u) {
#pragma unroll
        for (int k = 0; k < V; k++) sum = __builtin_fma((double)u[k], (double)u[k], sum);
    };
    if (e.tensors) {
        const oz_muon_tensor& t = e.tensors[s.first + w.matrix];
        const long long n = (long long)s.rows * s.cols;
        const float gs = e.grad_scale ? *e.grad_scale : 1.0f;
        auto all = [&](auto TYPE) {
            for (long long j = (long long)THREADS * w.index + threadIdx.x; V * j < n; j += step) {
                const long long i = V * j;
                const int count = (int)(n - i < V ? n - i : V);
                float g[V], m[V], u[V];
                get(t.grad, decltype(TYPE)::value, i, count, g);
                get(t.m, OZ_F32, i, count, m);
#pragma unroll
                for (int k = 0; k < V; k++) m[k] = e.momentum * m[k] + e.fresh * (g[k] * gs);
                if (count == V) store8(t.m, OZ_F32, i, m);
                else store_some(t.m, OZ_F32, i, count, m);
                update_of(e, m, g, gs, u);
                add(u);
            }
        };
        if (t.grad_type == OZ_F32) all(std::integral_constant<int, OZ_F32>{});
        else if (t.grad_type == OZ_BF16) all(std::integral_constant<int, OZ_BF16>{});
        else all(std::integral_constant<int, OZ_F16>{});
    } else {
        const unsigned across = (s.cols + V - 1) / V;
        const long long n = (long long)across * s.rows;
        for (long long j = (long long)THREADS * w.index + threadIdx.x; j < n; j += step) {
            const unsigned row = (unsigned)j / across, col = V * ((unsigned)j % across);
            float u[V];
            get(e.G, e.type, (s.first + w.matrix) * e.stride_g + row * e.ldg + col, min((int)(s.cols - col), V), u);
            add(u);
        }
    }
    sum = sum_all(sum);
    if (threadIdx.x == 0) s.sums[(long long)w.matrix * s.chunks + w.index] = sum;
}

// X0 in the shapes' x[0].
__global__ void __launch_bounds__(THREADS) start_kernel(const Shapes shapes, const Ends e, const Places places, double eps, int rounds) {
    const Place w = place_of(places, shapes.n, blockIdx.x);
    const Shape& s = shapes.s[w.shape];
    double sum = 0.0;
    for (int c = threadIdx.x; c < s.chunks; c += THREADS) sum += s.sums[(long long)w.matrix * s.chunks + c];
    // In FP64, as U's squares are: no factor that a finite U needs is out of its range. Zeros stay zeros, a norm that is not finite makes
    // all values NaN.
    const double norm = sqrt(sum_all(sum));
    const double factor = norm == 0.0 ? 0.0 : norm < INFINITY ? (double)kScale / (norm + eps) : (double)NAN;
    const unsigned across = s.C / V;
    const long long n = (long long)across * s.R;
    _Float16 *h = h_of(s, 0, w.matrix), *l = l_of(s, 0, w.matrix);
    const float gs = e.grad_scale ? *e.grad_scale : 1.0f;
    for (int round = 0; round < rounds; round++) {
        const long long j = THREADS * ((long long)rounds * w.index + round) + threadIdx.x;
        if (j >= n) return;
        const unsigned row = (unsigned)j / across, col = V * ((unsigned)j % across);
        const int count = (int)row < s.rows ? min(max((int)(s.cols - col), 0), V) : 0;
        float u[V] = {};
        if (e.tensors) {
            const oz_muon_tensor& t = e.tensors[s.first + w.matrix];
            const long long i = (long long)row * s.cols + col;
            float g[V] = {}, m[V];
            if (count) {
                get(t.m, OZ_F32, i, count, m);
                if (e.nesterov) get(t.grad, t.grad_type, i, count, g);
                update_of(e, m, g, gs, u);
            }
        } else if (count) {
            get(e.G, e.type, (s.first + w.matrix) * e.stride_g + row * e.ldg + col, count, u);
        }
        f16x8 hi, lo;
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float x = k < count ? (float)((double)u[k] * factor) : 0.0f;
            hi[k] = (_Float16)x;
            lo[k] = (_Float16)(x - (float)hi[k]);
        }
        *reinterpret_cast<f16x8*>(h + V * j) = hi;
        *reinterpret_cast<f16x8*>(l + V * j) = lo;
    }
}

size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
int pad(int n) { return (n + kPad - 1) / kPad * kPad; }

// A shape with its buffers laid out from `at` on (null: to count them); the first byte behind them. `exact`: products of both parts
// whatever the size.
size_t lay_out(Shape* s, int rows, int cols, int count, int first, bool exact, char* base, size_t at) {
    *s = Shape{};
    s->rows = rows, s->cols = cols, s->count = count, s->first = first;
    s->R = pad(rows), s->C = pad(cols);
    s->three = exact || std::min(rows, cols) <= kThreeSide;
    const long long values = (long long)rows * cols, side = side_of(*s);
    s->chunks = (int)std::min<long long>(kMaxChunks, (values + kChunk - 1) / kChunk);
    const size_t x = 2 * (size_t)count * s->R * s->C, a = 2 * (size_t)count * side * side * (1 + s->three);
    auto take = [&](size_t bytes) {
        char* p = base + at;
        at += up(bytes);
        return base ? p : nullptr;
    };
    s->x[0] = reinterpret_cast<_Float16*>(take(x * (1 + s->three)));
    s->x[1] = reinterpret_cast<_Float16*>(take(x * (1 + s->three)));
    if (!s->three) s->l = reinterpret_cast<_Float16*>(take(x));
    s->a = reinterpret_cast<_Float16*>(take(a));
    s->b = reinterpret_cast<_Float16*>(take(a));
    if (!s->three) s->d = reinterpret_cast<float*>(take(4 * (size_t)count * side));
    s->sums = reinterpret_cast<double*>(take(8 * (size_t)count * s->chunks));
    return at;
}

// Both passes and the iteration.
int orthogonalize(oz_dev* dev, const Shapes& m, const Ends& e, const Factors& f, double eps, int steps) {
    Places squares{}, start{};
    long long a = 0, b = 0, all = 0;
    for (int k = 0; k < m.n; k++) all += (long long)m.s[k].R * m.s[k].C * m.s[k].count;
    const int rounds = all >= (long long)V * THREADS * kRounds * 4 * dev->cus ? kRounds : 1;
    for (int k = 0; k < m.n; k++) {
        const Shape& s = m.s[k];
        const long long pieces = (long long)s.R * s.C / V, per = (pieces + THREADS * rounds - 1) / (THREADS * rounds);
        squares.first[k] = (int)a, squares.per[k] = s.chunks;
        start.first[k] = (int)b, start.per[k] = (int)per;
        a += (long long)s.chunks * s.count;
        b += per * s.count;
        if (pieces >> 31 || a >= 1 << 23 || b >= 1 << 23) return oz::fail(dev, OZ_ERR_ARG, "too many values in matrices");
    }
    squares.first[m.n] = (int)a, start.first[m.n] = (int)b;
    Iteration it;
    if (int st = prepare(dev, m, f, &it)) return st;
    hipLaunchKernelGGL(squares_kernel, dim3((unsigned)a), dim3(THREADS), 0, dev->stream, m, e, squares);
    if (int st = oz::launch_check(dev, "squares_kernel")) return st;
    hipLaunchKernelGGL(start_kernel, dim3((unsigned)b), dim3(THREADS), 0, dev->stream, m, e, start, eps, rounds);
    if (int st = oz::launch_check(dev, "start_kernel")) return st;
    return iterate(dev, &it, e, steps);
}

constexpr int kMaxSide = 1 << 20;
constexpr long long kMaxValues = 1ll << 33;  // of a matrix

bool known(int type) { return type == OZ_F32 || is_16bit(type); }
bool misaligned(const void* p, int type) { return ((uintptr_t)p & (size_of(type) - 1)) != 0; }
bool finite(double x) { return std::fabs(x) < INFINITY; }

const char* refuse(int steps, double a, double b, double c, double eps) {
    if (steps < 1 || steps > 100) return "steps";
    if (!finite((float)a) || !finite((float)b) || !finite((float)c)) return "the iteration's factors";
    if (!(eps >= 0.0 && eps < INFINITY)) return "eps";
    return nullptr;
}

long long or_else(long long x, long long y) { return x ? x : y; }

const char* refuse(const oz_orthogonalize_desc* d) {
    if (!d) return "no descriptor";
    if (d->rows < 1 || d->cols < 1 || d->count < 0) return "sizes";
    if (d->rows > kMaxSide || d->cols > kMaxSide || (long long)d->rows * d->cols > kMaxValues || d->count > 1 << 20) return "too many values";
    if (!known(d->type)) return "the type";
    if (const char* e = refuse(d->steps, d->a, d->b, d->c, d->eps)) return e;
    for (const auto& [ld, stride] : {std::pair(d->ldg, d->stride_g), std::pair(d->ldo, d->stride_o)}) {
        if (ld && (ld < d->cols || ld > 1ll << 32)) return "a leading dimension";
        const long long matrix = (d->rows - 1) * or_else(ld, d->cols) + d->cols;
        if (stride && d->count > 1 && (stride < matrix || stride > 1ll << 53)) return "a distance of matrices";
    }
    return nullptr;
}

size_t shape_of(const oz_orthogonalize_desc* d, Shape* s, char* base) {
    return lay_out(s, d->rows, d->cols, d->count, 0, d->exact || d->type != OZ_BF16, base, 0);
}

// The plan's shapes in `base`, and the workspace's size.
size_t shapes_of(const oz_muon_plan* p, Shapes* m, char* base) {
    size_t at = 0;
    m->n = p->shapes;
    for (int k = 0; k < p->shapes; k++)
        at = lay_out(&m->s[k], p->shape[k].rows, p->shape[k].cols, p->shape[k].count, p->shape[k].first, p->exact >> k & 1, base, at);
    return at;
}

static_assert(kShapes <= 32, "bits of a plan's exact");
bool bad_plan(const oz_muon_plan* p) {
    if (!p || !p->memory || p->count < 0 || p->shapes < 0 || p->shapes > kShapes) return true;
    for (int k = 0; k < p->shapes; k++) {
        const oz_muon_shape& s = p->shape[k];
        if (s.rows < 1 || s.cols < 1 || s.rows > kMaxSide || s.cols > kMaxSide || s.count < 1 || s.first < 0 || s.count > p->count - s.first) return true;
    }
    return false;
}

}  // namespace

extern "C" {

long long oz_orthogonalize_workspace(oz_dev* dev, const oz_orthogonalize_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_orthogonalize: %s", e);
    Shape s;
    return d->count ? (long long)shape_of(d, &s, nullptr) : 0;
}

int oz_orthogonalize(oz_dev* dev, const oz_orthogonalize_desc* d, const void* G, void* O, void* work, size_t bytes) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_orthogonalize: %s", e);
    if (d->count && (!G || !O)) return oz::fail(dev, OZ_ERR_ARG, "oz_orthogonalize: null operand");
    if (misaligned(G, d->type) || misaligned(O, d->type)) return oz::fail(dev, OZ_ERR_ARG, "oz_orthogonalize: operands at addresses that their type does not allow");
    const size_t need = (size_t)oz_orthogonalize_workspace(dev, d);
    if (need && (!work || bytes < need || ((uintptr_t)work & 15)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_orthogonalize: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
    if (int st = oz::use(dev)) return st;
    if (!d->count) return OZ_OK;
    Shapes m{};
    m.n = 1;
    shape_of(d, &m.s[0], static_cast<char*>(work));
    Ends e{};
    e.G = G, e.O = O, e.type = d->type;
    e.ldg = or_else(d->ldg, d->cols), e.ldo = or_else(d->ldo, d->cols);
    e.stride_g = or_else(d->stride_g, d->rows * e.ldg), e.stride_o = or_else(d->stride_o, d->rows * e.ldo);
    if (G == O && (e.ldg != e.ldo || (d->count > 1 && e.stride_g != e.stride_o)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_orthogonalize: O is G with other strides");
    return orthogonalize(dev, m, e, factors_of(d->a, d->b, d->c, d->steps), d->eps, d->steps);
}

long long oz_muon_plan_bytes(const oz_muon_tensor* tensors, int count) {
    if (count < 0 || (count && !tensors) || count > 1 << 20) return OZ_ERR_ARG;
    for (int k = 0; k < count; k++)
        if (tensors[k].rows < 0 || tensors[k].cols < 0 || tensors[k].rows > kMaxSide || tensors[k].cols > kMaxSide ||
            (long long)tensors[k].rows * tensors[k].cols > kMaxValues)
            return OZ_ERR_ARG;
    return (long long)count * sizeof(oz_muon_tensor) + 16;
}

int oz_muon_make_plan(oz_dev* dev, const oz_muon_tensor* tensors, int count, void* memory, size_t bytes, oz_muon_plan* plan) {
    if (!plan) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: no plan to fill");
    *plan = oz_muon_plan{};
    const long long need = oz_muon_plan_bytes(tensors, count);
    if (need < 0) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: sizes of the matrices");
    for (int k = 0; k < count; k++) {
        const oz_muon_tensor& t = tensors[k];
        if (!known(t.param_type) || !known(t.grad_type) || (t.master && t.param_type == OZ_F32))
            return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: types of matrix %d", k);
        if (t.rows && t.cols && (!t.param || !t.grad || !t.m)) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: arrays of matrix %d", k);
        if (misaligned(t.param, t.param_type) || misaligned(t.grad, t.grad_type) || misaligned(t.master, OZ_F32) || misaligned(t.m, OZ_F32))
            return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: matrix %d at an address that its type does not allow", k);
        if (!(t.weight_decay >= 0.0f && t.weight_decay < INFINITY) || !(t.lr_scale >= 0.0f && t.lr_scale < INFINITY))
            return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: weight decay or lr_scale of matrix %d", k);
    }
    if (!memory || (long long)bytes < need || ((uintptr_t)memory & 15))
        return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: %zu bytes, %lld needed (16-byte aligned)", bytes, need);
    oz_muon_plan p{};
    try {
        std::vector<oz_muon_tensor> list;
        list.reserve((size_t)count + 1);
        std::vector<char> done((size_t)count, 0);
        for (int k = 0; k < count; k++) {
            const oz_muon_tensor& t = tensors[k];
            if (done[k] || !t.rows || !t.cols) continue;
            if (p.shapes == kShapes) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_make_plan: more than %d different sizes", kShapes);
            oz_muon_shape& s = p.shape[p.shapes++];
            s = {t.rows, t.cols, 0, (int)list.size()};
            for (int j = k; j < count; j++)
                if (tensors[j].rows == t.rows && tensors[j].cols == t.cols) {
                    list.push_back(tensors[j]);
                    done[j] = 1;
                    if (tensors[j].param_type == OZ_F32) p.exact |= 1u << (p.shapes - 1);
                    s.count++;
                }
        }
        p.count = (int)list.size();
        // The memory may come from an allocator that hands out again what kernels of its own stream still write: the kernels
        // take their addresses from here, so the copy waits for the device.
        if (int st = oz::use(dev)) return st;
        if (int st = oz::hip_check(dev, hipDeviceSynchronize(), "hipDeviceSynchronize")) return st;
        if (int st = oz_memcpy_h2d(dev, memory, list.data(), list.size() * sizeof(oz_muon_tensor))) return st;
    } catch (const std::bad_alloc&) {
        return oz::fail(dev, OZ_ERR_NOMEM, "oz_muon_make_plan: host memory");
    }
    p.memory = memory;
    *plan = p;
    return OZ_OK;
}

long long oz_muon_workspace(oz_dev* dev, const oz_muon_plan* plan) {
    if (bad_plan(plan)) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_workspace: no plan");
    Shapes m{};
    return (long long)shapes_of(plan, &m, nullptr);
}

int oz_muon_step(oz_dev* dev, const oz_muon_plan* plan, const oz_muon_options* o, void* work, size_t bytes) {
    if (bad_plan(plan) || !o) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_step: no plan or options");
    if (!(o->lr >= 0.0 && o->lr < INFINITY) || !(o->momentum >= 0.0 && o->momentum < 1.0) || (o->nesterov != 0 && o->nesterov != 1))
        return oz::fail(dev, OZ_ERR_ARG, "oz_muon_step: lr %g, momentum %g, nesterov %d", o->lr, o->momentum, o->nesterov);
    if (const char* e = refuse(o->steps, o->a, o->b, o->c, o->eps)) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_step: %s", e);
    if ((uintptr_t)o->grad_scale & 3) return oz::fail(dev, OZ_ERR_ARG, "oz_muon_step: grad_scale at an odd address");
    Shapes m{};
    const size_t need = shapes_of(plan, &m, static_cast<char*>(work));
    if (need && (!work || bytes < need || ((uintptr_t)work & 15)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_muon_step: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
    if (int st = oz::use(dev)) return st;
    if (!m.n) return OZ_OK;
    Ends e{};
    e.tensors = static_cast<const oz_muon_tensor*>(plan->memory);
    e.momentum = (float)o->momentum, e.fresh = (float)(1.0 - o->momentum), e.lr = (float)o->lr;
    e.nesterov = o->nesterov, e.grad_scale = o->grad_scale;
    return orthogonalize(dev, m, e, factors_of(o->a, o->b, o->c, o->steps), o->eps, o->steps);
}

}  // extern "C"
