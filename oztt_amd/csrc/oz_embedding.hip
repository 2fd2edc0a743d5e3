// Embedding rows by token and the table's gradient (include/oz_hip.h, oz_embedding, oz_embedding_grad).
//
// The lookup is a copy of T rows. The gradient is the transposed one-hot matrix times dOut: the tokens are sorted
// by a radix sort that keeps the order of equal ones, so that each row of the table is the sum of consecutive entries
// of the sorted list. The list is cut into runs of equal length, whatever the tokens (a frequent word may
// be a tenth of a text); a wave sums the rows of its run token by token in registers, writes the tokens
// that lie inside it, and leaves the sums of those that its ends cut, which a last launch joins in order. No atomics:
// the order of every sum follows from ids alone.
#include "oz_internal.hpp"
#include "oz_types.hpp"

namespace {

using namespace ozt;

constexpr long long kMaxD = 1ll << 22;
constexpr long long kMaxGroups = 1ll << 23;  // workgroups of 256 threads in one launch

struct Shape {
    long long T, vocab, ldt, ldo, padding;
    int D, type, grad_type, wide, accumulate;
    float scale;
};

__device__ __forceinline__ long long token(const void* ids, int wide, long long t) {
    return wide ? static_cast<const long long*>(ids)[t] : static_cast<const int*>(ids)[t];
}

// Rows by tokens: a wave takes one row's 512 columns at a time. VEC: rows of whole 16-byte pieces (8
// values, of FP32 two pieces), otherwise value by value.
template <bool VEC>
__global__ void __launch_bounds__(256) embedding_kernel(const void* __restrict__ table, const void* __restrict__ ids,
                                                        void* __restrict__ out, uint32_t* __restrict__ flags, Shape s, unsigned slices) {
    const unsigned lane = threadIdx.x & 63;
    const long long item = 4ll * blockIdx.x + (threadIdx.x >> 6), t = item / slices;
    if (t >= s.T) return;
    const int c0 = (int)(item % slices) * 512;
    const long long v = token(ids, s.wide, t);
    const bool known = v >= 0 && v < s.vocab;
    if (!known && flags && c0 == 0 && lane == 0) atomicOr(flags, 1u);
    if constexpr (VEC) {
        const int c = c0 + 8 * lane;
        if (c >= s.D) return;
        float x[8] = {};
        if (known) load8(table, s.type, v * s.ldt + c, x);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] *= s.scale;
        if (!known)
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = 0.0f;
        store8(out, s.type, t * s.ldo + c, x);
    } else {
        for (int c = c0 + lane; c < s.D && c < c0 + 512; c += 64)
            store(out, s.type, t * s.ldo + c, known ? load(table, s.type, v * s.ldt + c) * s.scale : 0.0f);
    }
}

// ---- sort ---------------------------------------------------------------------------------------------
// Least digit first, DIGITS values a digit; keys are the tokens, those without a gradient as `vocab`, behind all
// others. A tile is TILE consecutive entries, a quarter for each of 4 waves.
constexpr int TILE = 4096, MAX_BITS = 9, DIGITS = 1 << MAX_BITS;

__device__ __forceinline__ uint32_t key_of(const void* ids, const Shape& s, long long t, uint32_t* flags) {
    const long long v = token(ids, s.wide, t);
    if (v < 0 || v >= s.vocab) {
        if (flags) atomicOr(flags, 1u);
        return (uint32_t)s.vocab;
    }
    return v == s.padding ? (uint32_t)s.vocab : (uint32_t)v;
}

// Lanes of the wave with this lane's digit, among those of `among`.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, uint64_t among) {
    for (int b = 0; b < bits; b++) {
        const bool one = (d >> b) & 1;
        const uint64_t ones = __ballot(one);
        among &= one ? ones : ~ones;
    }
    return among;
}

// counts[digit][tile]
template <bool FIRST>
__global__ void __launch_bounds__(256) count_kernel(const void* __restrict__ ids, const uint32_t* __restrict__ keys, Shape s, int shift,
                                                    int bits, uint32_t* __restrict__ counts, unsigned tiles, uint32_t* __restrict__ flags) {
    __shared__ uint32_t n[DIGITS];
    for (int d = threadIdx.x; d < DIGITS; d += 256) n[d] = 0;
    __syncthreads();
    for (int e = threadIdx.x; e < TILE; e += 256) {
        const long long t = (long long)blockIdx.x * TILE + e;
        if (t < s.T) atomicAdd(&n[((FIRST ? key_of(ids, s, t, flags) : keys[t]) >> shift) & ((1 << bits) - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < 1 << bits; d += 256) counts[(size_t)d * tiles + blockIdx.x] = n[d];
}

// Exclusive prefix sums of n counts in place, by one workgroup: 8 a thread and round.
__global__ void __launch_bounds__(1024) scan_kernel(uint32_t* __restrict__ counts, long long n) {
    __shared__ uint32_t waves[17];
    uint32_t before = 0;
    for (long long b = 0; b < n; b += 8192) {
        const long long i = b + 8 * threadIdx.x;
        uint32_t x[8], sum = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            x[k] = i + k < n ? counts[i + k] : 0;
            sum += x[k];
        }
        uint32_t upto = sum;
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t y = __shfl_up(upto, d);
            if ((threadIdx.x & 63) >= d) upto += y;
        }
        if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = upto;
        __syncthreads();
        uint32_t at = before + upto - sum, total = 0;
        for (int w = 0; w < 16; w++) {
            if (w < (int)(threadIdx.x >> 6)) at += waves[w];
            total += waves[w];
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (i + k < n) counts[i + k] = at;
            at += x[k];
        }
        before += total;
        __syncthreads();
    }
}

// Every entry of a tile to its place: first the waves' counts of each digit, from them where each
// wave's entries of a digit begin, then 64 entries at a time in order.
template <bool FIRST>
__global__ void __launch_bounds__(256) scatter_kernel(const void* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                      const uint32_t* __restrict__ order, Shape s, int shift, int bits,
                                                      const uint32_t* __restrict__ starts, unsigned tiles,
                                                      uint32_t* __restrict__ keys_out, uint32_t* __restrict__ order_out) {
    __shared__ volatile uint32_t at[4][DIGITS];  // written by one lane of the owning wave, read by its others
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < 4 * DIGITS; d += 256) at[d / DIGITS][d % DIGITS] = 0;
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * TILE + wave * (TILE / 4);
    const uint64_t below = (1ull << lane) - 1;
    for (int round = 0; round < 2; round++) {
        for (int e = 0; e < TILE / 4; e += 64) {
            const long long t = t0 + e + lane;
            const bool in = t < s.T;
            const uint32_t key = in ? (FIRST ? key_of(ids, s, t, nullptr) : keys[t]) : 0;
            const uint32_t d = (key >> shift) & ((1 << bits) - 1);
            const uint64_t same = same_digit(d, bits, __ballot(in));
            if (in) {
                const uint32_t first = at[wave][d];
                __builtin_amdgcn_wave_barrier();
                if (!(same & below)) at[wave][d] = first + __popcll(same);
                if (round) {
                    const uint32_t place = first + __popcll(same & below);
                    keys_out[place] = key;
                    order_out[place] = FIRST ? (uint32_t)t : order[t];
                }
            }
        }
        __syncthreads();
        if (!round) {
            for (int d = threadIdx.x; d < 1 << bits; d += 256) {
                uint32_t a = starts[(size_t)d * tiles + blockIdx.x];
                for (int w = 0; w < 4; w++) {
                    const uint32_t n = at[w][d];
                    at[w][d] = a;
                    a += n;
                }
            }
            __syncthreads();
        }
    }
}

// ---- sums ---------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(256) zero_rows_kernel(void* __restrict__ table, Shape s) {
    const long long n = s.vocab * s.D, stride = 256ll * gridDim.x;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += stride) store(table, s.grad_type, i / s.D * s.ldt + i % s.D, 0.0f);
}

// Eight columns of a lane: c0 + 8 lane + k (VEC), or c0 + lane + 64 k.
template <bool VEC>
struct Columns {
    int c, D;
    __device__ Columns(int c0, int lane, int D) : c(VEC ? c0 + 8 * lane : c0 + lane), D(D) {}
    __device__ void get(const void* p, int type, long long row, float* x) const {
        if constexpr (VEC) {
            if (c < D) load8(p, type, row + c, x);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = c + 64 * k < D ? load(p, type, row + c + 64 * k) : 0.0f;
        }
    }
    __device__ void put(void* p, int type, long long row, const float* x) const {
        if constexpr (VEC) {
            if (c < D) store8(p, type, row + c, x);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (c + 64 * k < D) store(p, type, row + c + 64 * k, x[k]);
        }
    }
    // the table's row v from its sum
    __device__ void finish(void* table, const Shape& s, long long v, float* x) const {
        float old[8] = {};
        if (s.accumulate) get(table, s.grad_type, v * s.ldt, old);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = s.accumulate ? old[k] + x[k] * s.scale : x[k] * s.scale;
        put(table, s.grad_type, v * s.ldt, x);
    }
};

// A wave sums run r of R sorted entries, 512 columns. Sums of tokens that the run's beginning cuts go to
// parts[2 r], of those that its end cuts to parts[2 r + 1] (a token that fills the run: parts[2 r]).
template <bool VEC>
__global__ void __launch_bounds__(256) sums_kernel(const void* __restrict__ dOut, const uint32_t* __restrict__ keys,
                                                   const uint32_t* __restrict__ order, void* __restrict__ table,
                                                   float* __restrict__ parts, Shape s, int R, unsigned slices) {
    const long long item = 4ll * blockIdx.x + (threadIdx.x >> 6), r = item / slices;
    const long long begin = r * R, end = begin + R < s.T ? begin + R : s.T;
    if (begin >= s.T) return;
    const Columns<VEC> cols((int)(item % slices) * 512, threadIdx.x & 63, s.D);
    uint32_t key = keys[begin];
    const uint32_t none = (uint32_t)s.vocab;
    bool cut = begin > 0 && keys[begin - 1] == key;
    float sum[8] = {};
    for (long long i = begin; i < end && key != none; i++) {
        float x[8] = {};
        cols.get(dOut, s.type, order[i] * s.ldo, x);
#pragma unroll
        for (int k = 0; k < 8; k++) sum[k] += x[k];
        const uint32_t next = i + 1 < s.T ? keys[i + 1] : none;
        if (next == key && i + 1 < end) continue;
        if (cut) cols.put(parts, OZ_F32, 2 * r * s.D, sum);
        else if (next == key) cols.put(parts, OZ_F32, (2 * r + 1) * s.D, sum);
        else cols.finish(table, s, key, sum);
        cut = false;
        key = next;
#pragma unroll
        for (int k = 0; k < 8; k++) sum[k] = 0.0f;
    }
}

// Joins the sums of a token that run r's end cuts and that begins in run r.
template <bool VEC>
__global__ void __launch_bounds__(256) join_kernel(const uint32_t* __restrict__ keys, void* __restrict__ table,
                                                   const float* __restrict__ parts, Shape s, int R, unsigned slices) {
    const long long item = 4ll * blockIdx.x + (threadIdx.x >> 6), r = item / slices;
    const long long begin = r * R, end = begin + R;
    if (end >= s.T) return;
    const uint32_t key = keys[end - 1];
    if (key == (uint32_t)s.vocab || keys[end] != key || (begin > 0 && keys[begin - 1] == key)) return;
    const Columns<VEC> cols((int)(item % slices) * 512, threadIdx.x & 63, s.D);
    float sum[8] = {}, x[8] = {};
    cols.get(parts, OZ_F32, (2 * r + 1) * s.D, sum);
    for (long long q = r + 1;; q++) {
        cols.get(parts, OZ_F32, 2 * q * s.D, x);
#pragma unroll
        for (int k = 0; k < 8; k++) sum[k] += x[k];
        if ((q + 1) * R >= s.T || keys[(q + 1) * R] != key) break;
    }
    cols.finish(table, s, key, sum);
}

const char* refuse(const oz_embedding_desc* d) {
    if (!d) return "no descriptor";
    const long long most = (1ll << 31) - 1;
    if (d->T < 0 || d->T > most || d->vocab < 1 || d->vocab > most || d->D < 1 || d->D > kMaxD) return "sizes";
    if (d->type != OZ_F32 && !is_16bit(d->type)) return "the table's type";
    if (d->grad_type != d->type && d->grad_type != OZ_F32) return "the gradient's type";
    if (d->id_bits != 32 && d->id_bits != 64) return "the ids' type";
    if (d->accumulate != 0 && d->accumulate != 1) return "accumulate";
    for (long long ld : {d->ldt, d->ldo})
        if (ld != 0 && (ld < d->D || ld > kMaxD)) return "a leading dimension";
    return nullptr;
}

Shape shape_of(const oz_embedding_desc* d) {
    return Shape{d->T, d->vocab, d->ldt ? d->ldt : d->D, d->ldo ? d->ldo : d->D, d->padding, (int)d->D, d->type, d->grad_type,
                 d->id_bits == 64, d->accumulate, d->scale};
}

bool misaligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) != 0; }

// Whether rows are whole 16-byte pieces from 16-byte boundaries on.
bool wide_rows(const Shape& s, const void* a, const void* b) {
    return s.D % 8 == 0 && s.ldt % 8 == 0 && s.ldo % 8 == 0 && !(((uintptr_t)a | (uintptr_t)b) & 15);
}

// Sizes of the gradient's workspace: two lists of keys and places, the digits' counts, the cut sums.
struct Work {
    long long tiles, runs;
    int R;
    size_t list, counts, parts, bytes;
};
Work work_of(const oz_embedding_desc* d) {
    Work w;
    const auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    w.tiles = (d->T + TILE - 1) / TILE;
    w.R = 32;
    w.runs = (d->T + w.R - 1) / w.R;
    w.list = up(4 * d->T);
    w.counts = up(4 * DIGITS * w.tiles);
    w.parts = up(8 * (size_t)d->D * w.runs);
    w.bytes = 4 * w.list + w.counts + w.parts;
    return w;
}

}  // namespace

extern "C" {

int oz_embedding(oz_dev* dev, const oz_embedding_desc* d, const void* table, const void* ids, void* out, uint32_t* flags) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_embedding: %s", e);
    if (d->T > 0 && (!table || !ids || !out)) return oz::fail(dev, OZ_ERR_ARG, "oz_embedding: null operand");
    if (misaligned(table, size_of(d->type)) || misaligned(out, size_of(d->type)) || misaligned(ids, d->id_bits / 8) || misaligned(flags, 4))
        return oz::fail(dev, OZ_ERR_ARG, "oz_embedding: operands at addresses that their types do not allow");
    const Shape s = shape_of(d);
    const unsigned slices = oz::ceil_div(s.D, 512);
    const long long groups = (s.T * slices + 3) / 4;
    if (groups > kMaxGroups) return oz::fail(dev, OZ_ERR_ARG, "oz_embedding: %lld tokens of %d values are too many", s.T, s.D);
    if (int st = oz::use(dev)) return st;
    if (!s.T) return OZ_OK;
    if (wide_rows(s, table, out))
        hipLaunchKernelGGL(embedding_kernel<true>, dim3((unsigned)groups), dim3(256), 0, dev->stream, table, ids, out, flags, s, slices);
    else
        hipLaunchKernelGGL(embedding_kernel<false>, dim3((unsigned)groups), dim3(256), 0, dev->stream, table, ids, out, flags, s, slices);
    return oz::launch_check(dev, "embedding_kernel");
}

long long oz_embedding_grad_workspace(oz_dev* dev, const oz_embedding_desc* d) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_embedding_grad: %s", e);
    return (long long)work_of(d).bytes;
}

int oz_embedding_grad(oz_dev* dev, const oz_embedding_desc* d, const void* dOut, const void* ids, void* dTable,
                      uint32_t* flags, void* work, size_t bytes) {
    if (const char* e = refuse(d)) return oz::fail(dev, OZ_ERR_ARG, "oz_embedding_grad: %s", e);
    if (!dTable || (d->T > 0 && (!dOut || !ids))) return oz::fail(dev, OZ_ERR_ARG, "oz_embedding_grad: null operand");
    if (misaligned(dTable, size_of(d->grad_type)) || misaligned(dOut, size_of(d->type)) || misaligned(ids, d->id_bits / 8) || misaligned(flags, 4))
        return oz::fail(dev, OZ_ERR_ARG, "oz_embedding_grad: operands at addresses that their types do not allow");
    const Shape s = shape_of(d);
    const Work w = work_of(d);
    if (w.bytes && (!work || bytes < w.bytes || misaligned(work, 16)))
        return oz::fail(dev, OZ_ERR_ARG, "oz_embedding_grad: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, w.bytes);
    const unsigned slices = oz::ceil_div(s.D, 512);
    const long long groups = (w.runs * slices + 3) / 4;
    if (groups > kMaxGroups) return oz::fail(dev, OZ_ERR_ARG, "oz_embedding_grad: %lld tokens of %d values are too many", s.T, s.D);
    if (int st = oz::use(dev)) return st;
    hipStream_t q = dev->stream;
    if (!s.accumulate) {
        const unsigned blocks = (unsigned)std::min<long long>((s.vocab * s.D + 255) / 256, 8192);
        hipLaunchKernelGGL(zero_rows_kernel, dim3(blocks), dim3(256), 0, q, dTable, s);
    }
    if (s.T) {
        char* p = static_cast<char*>(work);
        uint32_t* keys[2] = {(uint32_t*)p, (uint32_t*)(p + w.list)};
        uint32_t* order[2] = {(uint32_t*)(p + 2 * w.list), (uint32_t*)(p + 3 * w.list)};
        uint32_t* counts = (uint32_t*)(p + 4 * w.list);
        float* parts = (float*)(p + 4 * w.list + w.counts);
        int total = 1;  // bits of the keys 0..vocab
        while (s.vocab >> total) total++;
        const int passes = (total + MAX_BITS - 1) / MAX_BITS, bits = (total + passes - 1) / passes;
        const dim3 tiles((unsigned)w.tiles), block(256);
        for (int k = 0; k < passes; k++) {
            uint32_t *ki = keys[(k + 1) & 1], *oi = order[(k + 1) & 1], *ko = keys[k & 1], *oo = order[k & 1];
            if (!k) hipLaunchKernelGGL(count_kernel<true>, tiles, block, 0, q, ids, ki, s, 0, bits, counts, tiles.x, flags);
            else hipLaunchKernelGGL(count_kernel<false>, tiles, block, 0, q, ids, ki, s, k * bits, bits, counts, tiles.x, flags);
            hipLaunchKernelGGL(scan_kernel, dim3(1), dim3(1024), 0, q, counts, w.tiles << bits);
            if (!k) hipLaunchKernelGGL(scatter_kernel<true>, tiles, block, 0, q, ids, ki, oi, s, 0, bits, counts, tiles.x, ko, oo);
            else hipLaunchKernelGGL(scatter_kernel<false>, tiles, block, 0, q, ids, ki, oi, s, k * bits, bits, counts, tiles.x, ko, oo);
        }
        const uint32_t *sk = keys[(passes - 1) & 1], *so = order[(passes - 1) & 1];
        const dim3 grid((unsigned)groups);
        if (wide_rows(s, dOut, dTable)) {
            hipLaunchKernelGGL(sums_kernel<true>, grid, block, 0, q, dOut, sk, so, dTable, parts, s, w.R, slices);
            hipLaunchKernelGGL(join_kernel<true>, grid, block, 0, q, sk, dTable, parts, s, w.R, slices);
        } else {
            hipLaunchKernelGGL(sums_kernel<false>, grid, block, 0, q, dOut, sk, so, dTable, parts, s, w.R, slices);
            hipLaunchKernelGGL(join_kernel<false>, grid, block, 0, q, sk, dTable, parts, s, w.R, slices);
        }
    }
    return oz::launch_check(dev, "embedding gradient");
}

}  // extern "C"
