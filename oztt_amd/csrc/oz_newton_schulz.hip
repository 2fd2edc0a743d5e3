// The Newton-Schulz iteration (oz_newton_schulz.hpp): its launches, and the products of the first parts alone.
#include "oz_internal.hpp"
#include "oz_newton_schulz_tiles.hpp"

#include <algorithm>

extern template void ozn::launch_products<true>(hipStream_t, Phase, int, const Shapes&, const Ends&, const Pass&);
template void ozn::launch_products<false>(hipStream_t, Phase, int, const Shapes&, const Ends&, const Pass&);

namespace {

using namespace ozn;

long long up(int n, int tile) { return (n + tile - 1) / tile; }

// Tiles of a matrix.
long long tiles_of(const Shape& s, Phase phase, int tile) {
    const long long t = up(side_of(s), tile);
    return phase == UPDATE ? up(s.R, tile) * up(s.C, tile) : t * (t + 1) / 2;
}
int stages_of(const Shape& s, Phase phase) { return (phase == GRAM ? std::max(s.R, s.C) : side_of(s)) / 64 * (s.three ? 3 : 1); }

// Estimated us of a phase in tiles of one size: what the workgroups of all shapes take together, dealt out over the CUs, and, as shapes
// end at different times, half of a workgroup's time more; whole rounds where there is one shape.
float estimate(const Shapes& m, Phase phase, ozl::Tile tile, int cus) {
    const ozl::Shape& t = ozl::shape_of(tile);
    const long long slots = (long long)cus * t.per_cu;
    float all = 0.0f, longest = 0.0f, rounds = 0.0f;
    for (int k = 0; k < m.n; k++) {
        const long long n = tiles_of(m.s[k], phase, t.q) * m.s[k].count;
        const float us = t.fixed + (float)stages_of(m.s[k], phase) * (n > cus ? t.full : t.alone);
        all += us * (float)n / (float)slots;
        longest = std::max(longest, us);
        const long long rest = n % slots;
        rounds = (float)(n / slots) * us + (rest ? t.fixed + (float)stages_of(m.s[k], phase) * (rest > cus ? t.full : t.alone) : 0.0f);
    }
    return m.n == 1 ? rounds : std::max(longest, all + 0.5f * longest);
}

// Places of a phase, or false where there are too many.
bool places(const Shapes& m, Phase phase, int tile, Places* p) {
    long long at = 0;
    for (int k = 0; k < m.n; k++) {
        const long long per = tiles_of(m.s[k], phase, tile);
        if (per >> 22 || (at + per * m.s[k].count) >> 22) return false;
        p->first[k] = (int)at;
        p->per[k] = (int)per;
        at += per * m.s[k].count;
    }
    p->first[m.n] = (int)at;
    return true;
}

int iterate_alike(oz_dev* dev, const Shapes& m, const Ends& ends, const Factors& f, int steps) {
    if (!m.n) return OZ_OK;
    Pass pass[3] = {};
    int tile[3];
    Shapes order[3];
    for (const Phase phase : {GRAM, SQUARE, UPDATE}) {
        order[phase] = m;
        std::stable_sort(order[phase].s, order[phase].s + m.n, [&](const Shape& a, const Shape& b) { return stages_of(a, phase) > stages_of(b, phase); });
        float best = 0.0f;
        for (const ozl::Tile t : {ozl::T256, ozl::T128, ozl::T64}) {
            const float us = estimate(m, phase, t, dev->cus);
            if (best == 0.0f || us < best) best = us, tile[phase] = ozl::shape_of(t).q;
        }
        pass[phase].f = f;
        if (!places(order[phase], phase, tile[phase], &pass[phase].places)) return oz::fail(dev, OZ_ERR_ARG, "too many values in matrices");
    }
    for (int k = 0; k < steps; k++)
        for (const Phase phase : {GRAM, SQUARE, UPDATE}) {
            Pass& p = pass[phase];
            p.from = k & 1;
            p.last = k + 1 == steps;
            if (m.s[0].three) launch_products<true>(dev->stream, phase, tile[phase], order[phase], ends, p);
            else launch_products<false>(dev->stream, phase, tile[phase], order[phase], ends, p);
            if (int st = oz::launch_check(dev, "newton_schulz_kernel")) return st;
        }
    return OZ_OK;
}

}  // namespace

int ozn::iterate(oz_dev* dev, const Shapes& m, const Ends& ends, const Factors& f, int steps) {
    Shapes part[2] = {};
    for (int k = 0; k < m.n; k++) {
        Shapes& p = part[m.s[k].three];
        p.s[p.n++] = m.s[k];
    }
    for (const Shapes& p : part)
        if (int st = iterate_alike(dev, p, ends, f, steps)) return st;
    return OZ_OK;
}
