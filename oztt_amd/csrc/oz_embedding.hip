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

#include <algorithm>

namespace {

using namespace ozt;

constexpr long long kMaxD = 1ll << 22;

// Workgroups of 256 threads: 2^23 along x (a launch takes fewer than 2^32 threads along a dimension), the rest along y. What is too
// much of the last row finds no work.
constexpr int ROW_LOG = 23;
dim3 grid_of(long long groups) {
    const long long x = std::max(1ll, std::min(groups, 1ll << ROW_LOG));
    return dim3((unsigned)x, (unsigned)((groups + x - 1) / x));
}
__device__ __forceinline__ long long wave_number() {
    return 4 * (((long long)blockIdx.y << ROW_LOG) + blockIdx.x) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

struct Shape {
    long long T, vocab, ldt, ldo, padding;
    int D, type, grad_type, wide, accumulate;
    float scale;
};

__device__ __forceinline__ long long token(const void* ids, int wide, long long t) {
    return wide ? static_cast<const long long*>(ids)[t] : static_cast<const int*>(ids)[t];
}

// Eight columns of a lane, c + k, those below D.
struct Columns {
    int c, count;
    __device__ Columns(int c0, int lane, int D) : c(c0 + 8 * lane), count(D - (c0 + 8 * lane)) {}
    __device__ void get(const void* p, int type, long long row, float* x) const {
        if (count >= 8) load8(p, type, row + c, x);
        else if (count > 0) load_some(p, type, row + c, count, x);
    }
    __device__ void put(void* p, int type, long long row, const float* x) const {
        if (count >= 8) store8(p, type, row + c, x);
        else if (count > 0) store_some(p, type, row + c, count, x);
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

// The same columns of rows that are asked for ahead: the bytes stay as they came until they are used, and no lane's request
// depends on a branch, so that several rows are on their way at once (with branches the compiler waits for each row where they
// meet, and 2.2 TB/s are read). A lane with fewer than 8 columns left asks for the row's last 8 and
// takes its own from them. SMALL: rows of fewer than 8 values, one by one.
template <int TYPE, bool SMALL>
struct Ahead {
    static constexpr int WORDS = TYPE == OZ_F32 ? 8 : 4;
    typedef u32x4 Raw[WORDS / 4];
    int c, shift, D;
    __device__ Ahead(const Columns& cols, int D) : D(D) {
        c = SMALL || cols.count >= 8 ? cols.c : D - 8;
        shift = cols.count > 0 ? cols.c - c : 0;
    }
    __device__ void ask(const void* p, long long row, Raw& w) const {
        if constexpr (SMALL) {
            float x[8] = {};
            if (c == 0) load_some(p, TYPE, row, D, x);
            if constexpr (WORDS == 8) __builtin_memcpy(&w, x, 32);
            else narrow8(x, w[0]);
        } else {
            const char* from = static_cast<const char*>(p) + (row + c) * (WORDS / 2);
#pragma unroll
            for (int k = 0; k < WORDS / 4; k++) w[k] = get16<u32x4>(from + 16 * k);
        }
    }
    __device__ void take(const Raw& w, float* x) const {
        if constexpr (WORDS == 8) {
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = __uint_as_float(w[k / 4][k & 3]);
        } else {
            widen8(w[0], TYPE, x);
        }
        for (int n = 0; n < shift; n++)
#pragma unroll
            for (int k = 0; k < 7; k++) x[k] = x[k + 1];
    }
    __device__ static void narrow8(const float* x, u32x4& w) {
        union {
            u32x4 w;
            __bf16 b[8];
            _Float16 h[8];
        } u;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (TYPE == OZ_BF16) u.b[k] = (__bf16)x[k];
            else u.h[k] = (_Float16)x[k];
        }
        w = u.w;
    }
};

// Rows by tokens: a wave takes 512 columns of a row, whose token is a scalar then, or of narrow rows 2^rows_log rows,
// 64 >> rows_log lanes each (19056 rows of 22 values: 9.6 us by a row a wave). The load is one for every lane, whatever its
// columns (8192 rows of 4093 values 19 us, 25 with a branch on the columns left). Two, four or eight pieces a wave are slower
// (8192 rows of 4096: 17.7 us by one, 18.8 by four). Bound by memory: 21.4 us for rows that no cache holds, 4.7 TB/s.
template <int TYPE, bool SMALL, bool NARROW>
__global__ void __launch_bounds__(256) embedding_kernel(const void* __restrict__ table, const void* __restrict__ ids,
                                                        void* __restrict__ out, uint32_t* __restrict__ flags, Shape s, unsigned slices, int rows_log) {
    const long long wave = wave_number();
    const int lane = threadIdx.x & ((64u >> (NARROW ? rows_log : 0)) - 1);
    long long t;
    int c0 = 0;
    if constexpr (NARROW) {
        t = (wave << rows_log) + ((threadIdx.x & 63) >> (6 - rows_log));
    } else {
        t = wave / slices;
        c0 = (int)(wave - t * slices) * 512;
    }
    if (t >= s.T) return;
    const long long v = token(ids, s.wide, t);
    const bool known = v >= 0 && v < s.vocab;
    if (!known && flags && c0 == 0 && lane == 0) atomicOr(flags, 1u);
    const Columns cols(c0, lane, s.D);
    const Ahead<TYPE, SMALL> rows(cols, s.D);
    typename Ahead<TYPE, SMALL>::Raw w;
    float x[8];
    rows.ask(table, known ? v * s.ldt : 0, w);
    rows.take(w, x);
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = known ? x[k] * s.scale : 0.0f;
    cols.put(out, TYPE, t * s.ldo, x);
}

template <int TYPE>
auto lookup_of(int D, int rows_log) {
    return D < 8 ? embedding_kernel<TYPE, true, true> : rows_log ? embedding_kernel<TYPE, false, true> : embedding_kernel<TYPE, false, false>;
}

// Zeros for part `part` of `parts` of the table's rows, by workgroups `first` to gridDim.x - 1 of a launch, which stride over
// it in 16-byte pieces.
struct Zeros {
    void* table;
    int part, parts;
    unsigned first;
};
__device__ __forceinline__ void zero_rows(const Zeros& z, const Shape& s) {
    const int size = size_of(s.grad_type);
    const long long row_bytes = (long long)s.D * size, first_row = s.vocab * z.part / z.parts, rows = s.vocab * (z.part + 1) / z.parts - first_row;
    char* base = static_cast<char*>(z.table) + first_row * s.ldt * size;
    const long long me = (long long)(blockIdx.x - z.first) * blockDim.x + threadIdx.x, stride = (long long)(gridDim.x - z.first) * blockDim.x;
    const u32x4 none = {0, 0, 0, 0};
    if (s.ldt == s.D) {
        const long long bytes = rows * row_bytes;
        // past the caches, which the sums' rows need (32768 x 2048 into 65536 rows: 179 us against 167)
        const bool even = !((uintptr_t)base & 15);
        for (long long i = me; i < bytes / 16; i += stride) {
            if (even) __builtin_nontemporal_store(none, reinterpret_cast<u32x4*>(base + 16 * i));
            else put16(base + 16 * i, none);
        }
        for (long long i = bytes / 16 * 16 + 2 * me; i < bytes; i += 2 * stride) *reinterpret_cast<uint16_t*>(base + i) = 0;
    } else {
        const long long across = (row_bytes + 15) / 16;
        for (long long i = me; i < rows * across; i += stride) {
            const long long row = i / across, at = 16 * (i - row * across);
            char* to = base + row * s.ldt * size + at;
            if (at + 16 <= row_bytes) put16(to, none);
            else
                for (long long k = at; k < row_bytes; k += 2) *reinterpret_cast<uint16_t*>(to + k - at) = 0;
        }
    }
}
__global__ void __launch_bounds__(256) zero_rows_kernel(Zeros z, Shape s) { zero_rows(z, s); }

// ---- sort ---------------------------------------------------------------------------------------------
// Least digit first, DIGITS values a digit; keys are the tokens, those without a gradient as `vocab`, behind all others. A tile
// is 1024 ITEMS consecutive entries, a sixteenth for each of 16 waves. Per digit a launch counts the tiles' digits and one moves
// the entries; where a tile's entries of a digit begin each workgroup sums up by itself from the counts of all tiles, up to
// SUMMED tiles, and a third launch does for more. The launches also write the table's zeros, by workgroups of their own:
// what the sort takes is hidden behind them where the table is large.
constexpr int MAX_BITS = 9, DIGITS = 1 << MAX_BITS, SORT_THREADS = 1024, SORT_WAVES = 16, SUMMED = 256;

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

// counts[tile][digit]
template <bool FIRST, int ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) count_kernel(const void* __restrict__ ids, const uint32_t* __restrict__ keys, Shape s, int shift,
                                                             int bits, uint32_t* __restrict__ counts, uint32_t* __restrict__ flags, Zeros z) {
    if (blockIdx.x >= z.first) {
        zero_rows(z, s);
        return;
    }
    __shared__ uint32_t n[DIGITS];
    if (threadIdx.x < DIGITS) n[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const long long t = ((long long)blockIdx.x * ITEMS + i) * SORT_THREADS + threadIdx.x;
        if (t < s.T) atomicAdd(&n[((FIRST ? key_of(ids, s, t, flags) : keys[t]) >> shift) & ((1 << bits) - 1)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 1 << bits) counts[((size_t)blockIdx.x << bits) + threadIdx.x] = n[threadIdx.x];
}

// The counts of many tiles to where each tile's entries of a digit begin, by one workgroup, a digit a thread.
__global__ void __launch_bounds__(DIGITS) scan_kernel(uint32_t* __restrict__ counts, int bits, long long tiles) {
    __shared__ uint32_t total[DIGITS];
    const int d = threadIdx.x;
    uint32_t sum = 0;
    if (d < 1 << bits) {
#pragma unroll 8
        for (long long t = 0; t < tiles; t++) sum += counts[(t << bits) + d];
    }
    total[d] = d < 1 << bits ? sum : 0;
    __syncthreads();
    if (d >= 1 << bits) return;
    uint32_t at = 0;
    for (int k = 0; k < d; k++) at += total[k];
    for (long long t = 0; t < tiles; t += 8) {
        uint32_t n[8];
#pragma unroll
        for (int k = 0; k < 8; k++) n[k] = t + k < tiles ? counts[((t + k) << bits) + d] : 0;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (t + k < tiles) {
                counts[((t + k) << bits) + d] = at;
                at += n[k];
            }
    }
}

// Every entry of a tile to its place: its rank among its wave's entries of its digit, 64 entries at a time in order; behind the
// entries of smaller digits, of earlier tiles and of earlier waves. SCANNED: `counts` are scan_kernel's.
template <bool FIRST, int ITEMS, bool SCANNED>
__global__ void __launch_bounds__(SORT_THREADS) scatter_kernel(const void* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                               const uint32_t* __restrict__ order, Shape s, int shift, int bits,
                                                               const uint32_t* __restrict__ counts, unsigned tiles,
                                                               uint32_t* __restrict__ keys_out, uint32_t* __restrict__ order_out, Zeros z) {
    if (blockIdx.x >= z.first) {
        zero_rows(z, s);
        return;
    }
    __shared__ volatile uint16_t seen[SORT_WAVES][DIGITS];  // written by one lane of the owning wave, read by its others
    __shared__ uint32_t start[SORT_WAVES][DIGITS], totals[SORT_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << bits;
    for (int d = threadIdx.x; d < SORT_WAVES * DIGITS; d += SORT_THREADS) seen[d / DIGITS][d % DIGITS] = 0;
    const long long first = ((long long)blockIdx.x * SORT_WAVES + wave) * ITEMS * 64 + lane;
    uint32_t key[ITEMS], who[ITEMS], rank[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const long long t = first + 64 * i;
        key[i] = t < s.T ? (FIRST ? key_of(ids, s, t, nullptr) : keys[t]) : 0;
        who[i] = t < s.T ? (FIRST ? (uint32_t)t : order[t]) : 0;
    }
    // this tile's part of the counts, while those loads are on their way
    uint32_t before = 0, all = 0;
    if (threadIdx.x < digits) {
        if (SCANNED) {
            before = counts[(size_t)blockIdx.x * digits + threadIdx.x];
        } else {
#pragma unroll 8
            for (unsigned t = 0; t < tiles; t++) {
                const uint32_t n = counts[(size_t)t * digits + threadIdx.x];
                before += t < blockIdx.x ? n : 0;
                all += n;
            }
        }
    }
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const bool in = first + 64 * i < s.T;
        const uint32_t d = (key[i] >> shift) & (digits - 1);
        const uint64_t same = same_digit(d, bits, __ballot(in));
        rank[i] = 0;
        if (in) {
            const uint32_t n = seen[wave][d];
            __builtin_amdgcn_wave_barrier();
            if (!(same & below)) seen[wave][d] = (uint16_t)(n + __popcll(same));
            rank[i] = n + __popcll(same & below);
        }
    }
    if (!SCANNED) {
        uint32_t upto = all;
        for (int k = 1; k < 64; k *= 2) {
            const uint32_t y = __shfl_up(upto, k);
            if (lane >= k) upto += y;
        }
        if (lane == 63) totals[wave] = upto;
        __syncthreads();
        before += upto - all;
        for (int w = 0; w < wave; w++) before += totals[w];
    } else {
        __syncthreads();
    }
    if (threadIdx.x < digits)
        for (int w = 0; w < SORT_WAVES; w++) {
            start[w][threadIdx.x] = before;
            before += seen[w][threadIdx.x];
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; i++)
        if (first + 64 * i < s.T) {
            const uint32_t place = start[wave][(key[i] >> shift) & (digits - 1)] + rank[i];
            // ids that another stream still writes give other digits here than when they were counted
            if (place < (uint32_t)s.T) {
                keys_out[place] = key[i];
                order_out[place] = who[i];
            }
        }
}

// All digits of at most 1024 tokens by one workgroup: the same with one tile, whose entries change places in LDS (the
// gradient of 512 tokens 20.0 us, 27.4 by two launches a digit).
__global__ void __launch_bounds__(SORT_THREADS) sort_tile_kernel(const void* __restrict__ ids, Shape s, int passes, int bits,
                                                                 uint32_t* __restrict__ keys_out, uint32_t* __restrict__ order_out,
                                                                 uint32_t* __restrict__ flags, Zeros z) {
    if (blockIdx.x >= z.first) {
        zero_rows(z, s);
        return;
    }
    __shared__ volatile uint16_t seen[SORT_WAVES][DIGITS];
    __shared__ uint32_t start[SORT_WAVES][DIGITS], totals[SORT_WAVES], keys[SORT_THREADS], places[SORT_THREADS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << bits, me = threadIdx.x;
    const bool in = me < s.T;
    const uint64_t below = (1ull << lane) - 1;
    uint32_t key = in ? key_of(ids, s, me, flags) : 0, who = me;
    for (int p = 0; p < passes; p++) {
        for (int d = me; d < SORT_WAVES * DIGITS; d += SORT_THREADS) seen[d / DIGITS][d % DIGITS] = 0;
        __syncthreads();
        const uint32_t digit = (key >> (p * bits)) & (digits - 1);
        const uint64_t same = same_digit(digit, bits, __ballot(in));
        const uint32_t rank = __popcll(same & below);
        if (in && !rank) seen[wave][digit] = (uint16_t)__popcll(same);
        __syncthreads();
        uint32_t all = 0;
        if (me < digits)
            for (int w = 0; w < SORT_WAVES; w++) all += seen[w][me];
        uint32_t upto = all;
        for (int k = 1; k < 64; k *= 2) {
            const uint32_t y = __shfl_up(upto, k);
            if (lane >= k) upto += y;
        }
        if (lane == 63) totals[wave] = upto;
        __syncthreads();
        if (me < digits) {
            uint32_t at = upto - all;
            for (int w = 0; w < wave; w++) at += totals[w];
            for (int w = 0; w < SORT_WAVES; w++) {
                start[w][me] = at;
                at += seen[w][me];
            }
        }
        __syncthreads();
        if (in) {
            const uint32_t place = start[wave][digit] + rank;
            keys[place] = key;
            places[place] = who;
        }
        __syncthreads();
        if (in) {
            key = keys[me];
            who = places[me];
        }
        __syncthreads();
    }
    if (in) {
        keys_out[me] = key;
        order_out[me] = who;
    }
}

// ---- sums ---------------------------------------------------------------------------------------------
// A wave sums run r of R <= 64 sorted entries, 512 columns, the next 8 rows on their way while 8 are added. Sums of tokens that the run's beginning
// cuts go to parts[2 r], of those that its end cuts to parts[2 r + 1] (a token that fills the run: parts[2 r]).
template <int TYPE, bool SMALL>
__global__ void __launch_bounds__(256) sums_kernel(const void* __restrict__ dOut, const uint32_t* __restrict__ keys,
                                                   const uint32_t* __restrict__ order, void* __restrict__ table,
                                                   float* __restrict__ parts, Shape s, int R, unsigned slices) {
    const int lane = threadIdx.x & 63;
    const long long item = wave_number(), r = item / slices;
    const long long begin = r * R, end = begin + R < s.T ? begin + R : s.T;
    if (begin >= s.T) return;
    const Columns cols((int)(item - r * slices) * 512, lane, s.D);
    const int n = (int)(end - begin);
    const uint32_t none = (uint32_t)s.vocab;
    // entry `lane` of the run, its successor's key, and whether the run's first token began before
    const uint32_t mine = lane < n ? keys[begin + lane] : none;
    const uint32_t place = lane < n ? min(order[begin + lane], (uint32_t)s.T - 1) : 0;  // as the sort's places are checked
    const uint32_t after = end < s.T ? keys[end] : none, before = begin > 0 ? keys[begin - 1] : none;
    bool cut = before == (uint32_t)__builtin_amdgcn_readfirstlane(mine);
    float sum[8] = {};
    typedef Ahead<TYPE, SMALL> A;
    const A rows(cols, s.D);
    typename A::Raw w[2][8];
    auto ask = [&](int i0, typename A::Raw (&to)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + j < n ? i0 + j : n - 1;
            rows.ask(dOut, (long long)(uint32_t)__builtin_amdgcn_readlane(place, i) * s.ldo, to[j]);
        }
    };
    // false: the tokens without a gradient are reached, the last ones
    auto add = [&](int i0, const typename A::Raw (&from)[8]) -> bool {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + j;
            if (i >= n) break;
            const uint32_t key = __builtin_amdgcn_readlane(mine, i);
            if (key >= none) return false;
            float x[8];
            rows.take(from[j], x);
#pragma unroll
            for (int k = 0; k < 8; k++) sum[k] += x[k];
            const uint32_t next = i + 1 < n ? (uint32_t)__builtin_amdgcn_readlane(mine, i + 1) : after;
            if (next == key && i + 1 < n) continue;
            if (cut) cols.put(parts, OZ_F32, 2 * r * s.D, sum);
            else if (next == key) cols.put(parts, OZ_F32, (2 * r + 1) * s.D, sum);
            else cols.finish(table, s, key, sum);
            cut = false;
#pragma unroll
            for (int k = 0; k < 8; k++) sum[k] = 0.0f;
        }
        return true;
    };
    ask(0, w[0]);
    for (int i0 = 0; i0 < n; i0 += 16) {
        if (i0 + 8 < n) ask(i0 + 8, w[1]);
        if (!add(i0, w[0])) return;
        if (i0 + 8 >= n) return;
        if (i0 + 16 < n) ask(i0 + 16, w[0]);
        if (!add(i0 + 8, w[1])) return;
    }
}

// Joins the sums of a token that run r's end cuts and that begins in run r, in the runs' order, 8 asked for at a time.
template <bool SMALL>
__global__ void __launch_bounds__(256) join_kernel(const uint32_t* __restrict__ keys, void* __restrict__ table,
                                                   const float* __restrict__ parts, Shape s, int R, unsigned slices) {
    const int lane = threadIdx.x & 63;
    const long long item = wave_number(), r = item / slices;
    const long long begin = r * R, end = begin + R;
    if (end >= s.T) return;
    const uint32_t key = keys[end - 1];
    if (key >= (uint32_t)s.vocab || keys[end] != key || (begin > 0 && keys[begin] == key && keys[begin - 1] == key)) return;
    const Columns cols((int)(item - r * slices) * 512, lane, s.D);
    float sum[8] = {};
    cols.get(parts, OZ_F32, (2 * r + 1) * s.D, sum);
    typedef Ahead<OZ_F32, SMALL> A;
    const A rows(cols, s.D);
    for (long long q = r + 1;; q += 64) {
        // how many of the next 64 runs begin with the token
        const bool on = (q + lane) * R < s.T && keys[(q + lane) * R] == key;
        const uint64_t off = ~__ballot(on);
        const int m = off ? __ffsll((unsigned long long)off) - 1 : 64;
        for (int i0 = 0; i0 < m; i0 += 8) {
            typename A::Raw w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) rows.ask(parts, 2 * (q + (i0 + j < m ? i0 + j : m - 1)) * s.D, w[j]);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i0 + j < m) {
                    float x[8];
                    rows.take(w[j], x);
#pragma unroll
                    for (int k = 0; k < 8; k++) sum[k] += x[k];
                }
        }
        if (m < 64) break;
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

// Sizes of the gradient's workspace: two lists of keys and places, the digits' counts, the cut sums.
struct Work {
    int items, R;
    long long tiles, runs;
    size_t list, counts, parts, bytes;
};
Work work_of(const oz_embedding_desc* d) {
    Work w;
    const auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    w.items = d->T <= 64 * SORT_THREADS ? 1 : 4;  // 64 tiles' counts cost a workgroup 2 us
    w.tiles = (d->T + w.items * SORT_THREADS - 1) / (w.items * SORT_THREADS);
    // runs of 32 entries, shorter where those would leave most of the chip idle: 512 tokens of 500 values 28 us by 8, 47 by 32;
    // 8192 of 1024 68 by 16, 73 by 32; 18651 of 134 50 by 32, 108 by 8 (more cut sums to join)
    const long long waves = d->T * ((d->D + 511) / 512);
    w.R = waves <= 1 << 11 ? 8 : waves <= 1 << 14 ? 16 : 32;
    w.runs = (d->T + w.R - 1) / w.R;
    w.list = up(4 * d->T);
    w.counts = up(4 * DIGITS * w.tiles);
    w.parts = up(8 * (size_t)d->D * w.runs);
    w.bytes = 4 * w.list + w.counts + w.parts;
    return w;
}

// The sorted lists of keys and places (0, 1: which of the two), in 2 launches a digit, 3 of more than SUMMED tiles, 1 of one; `zeros`
// workgroups of each write the table's zeros.
template <int ITEMS>
int sort(oz_dev* dev, const void* ids, void* table, const Shape& s, const Work& w, uint32_t* const* keys, uint32_t* const* order,
         uint32_t* counts, uint32_t* flags, unsigned zeros) {
    int total = 1;  // bits of the keys 0..vocab
    while (s.vocab >> total) total++;
    const int passes = (total + MAX_BITS - 1) / MAX_BITS, bits = (total + passes - 1) / passes;
    const unsigned tiles = (unsigned)w.tiles;
    const dim3 grid(tiles + zeros), block(SORT_THREADS);
    constexpr bool MANY = ITEMS > 1;
    const bool scan = MANY && w.tiles > SUMMED;
    if (!MANY && tiles == 1) {
        hipLaunchKernelGGL(sort_tile_kernel, grid, block, 0, dev->stream, ids, s, passes, bits, keys[0], order[0], flags, Zeros{table, 0, 1, 1});
        return 0;
    }
    for (int k = 0; k < passes; k++) {
        uint32_t *ki = keys[(k + 1) & 1], *oi = order[(k + 1) & 1], *ko = keys[k & 1], *oo = order[k & 1];
        const Zeros z0{table, 2 * k, 2 * passes, tiles}, z1{table, 2 * k + 1, 2 * passes, tiles};
        const auto count = k ? count_kernel<false, ITEMS> : count_kernel<true, ITEMS>;
        hipLaunchKernelGGL(count, grid, block, 0, dev->stream, ids, ki, s, k * bits, bits, counts, k ? nullptr : flags, z0);
        if (scan) hipLaunchKernelGGL(scan_kernel, dim3(1), dim3(DIGITS), 0, dev->stream, counts, bits, w.tiles);
        const auto scatter = k ? (scan ? scatter_kernel<false, ITEMS, MANY> : scatter_kernel<false, ITEMS, false>)
                               : (scan ? scatter_kernel<true, ITEMS, MANY> : scatter_kernel<true, ITEMS, false>);
        hipLaunchKernelGGL(scatter, grid, block, 0, dev->stream, ids, ki, oi, s, k * bits, bits, counts, tiles, ko, oo, z1);
    }
    return (passes - 1) & 1;
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
    int rows_log = 0;
    while (rows_log < 6 && s.D <= 256 >> rows_log) rows_log++;
    const long long per = 4ll << rows_log, groups = (s.T * slices + per - 1) / per;
    if (int st = oz::use(dev)) return st;
    if (!s.T) return OZ_OK;
    const auto kernel = s.type == OZ_F32   ? lookup_of<OZ_F32>(s.D, rows_log)
                        : s.type == OZ_F16 ? lookup_of<OZ_F16>(s.D, rows_log)
                                           : lookup_of<OZ_BF16>(s.D, rows_log);
    hipLaunchKernelGGL(kernel, grid_of(groups), dim3(256), 0, dev->stream, table, ids, out, flags, s, slices, rows_log);
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
    if (int st = oz::use(dev)) return st;
    hipStream_t q = dev->stream;
    // workgroups that write zeros, in each launch: at most 8 a CU, 16 pieces of 16 bytes a thread or more
    const long long pieces = s.vocab * ((long long)s.D * size_of(s.grad_type) / 16 + 1);
    const unsigned zeros = s.accumulate ? 0 : (unsigned)std::max(1ll, std::min<long long>(pieces / (16 * SORT_THREADS), 8 * dev->cus));
    if (!s.T) {
        if (zeros) hipLaunchKernelGGL(zero_rows_kernel, dim3(4 * zeros), dim3(256), 0, q, Zeros{dTable, 0, 1, 0}, s);
        return oz::launch_check(dev, "zero_rows_kernel");
    }
    char* p = static_cast<char*>(work);
    uint32_t* keys[2] = {(uint32_t*)p, (uint32_t*)(p + w.list)};
    uint32_t* order[2] = {(uint32_t*)(p + 2 * w.list), (uint32_t*)(p + 3 * w.list)};
    uint32_t* counts = (uint32_t*)(p + 4 * w.list);
    float* parts = (float*)(p + 4 * w.list + w.counts);
    const int sorted = w.items == 1 ? sort<1>(dev, ids, dTable, s, w, keys, order, counts, flags, zeros)
                                    : sort<4>(dev, ids, dTable, s, w, keys, order, counts, flags, zeros);
    if (int st = oz::launch_check(dev, "sort")) return st;
    const dim3 block(256);
    const bool small = s.D < 8;
    const auto sums = s.type == OZ_F32 ? (small ? sums_kernel<OZ_F32, true> : sums_kernel<OZ_F32, false>)
                      : s.type == OZ_F16 ? (small ? sums_kernel<OZ_F16, true> : sums_kernel<OZ_F16, false>)
                                         : (small ? sums_kernel<OZ_BF16, true> : sums_kernel<OZ_BF16, false>);
    hipLaunchKernelGGL(sums, grid_of(groups), block, 0, q, dOut, keys[sorted], order[sorted], dTable, parts, s, w.R, slices);
    if (w.runs > 1)  // otherwise nothing is cut
        hipLaunchKernelGGL(small ? join_kernel<true> : join_kernel<false>, grid_of(groups), block, 0, q, keys[sorted], dTable, parts, s, w.R, slices);
    return oz::launch_check(dev, "embedding gradient");
}

}  // extern "C"
