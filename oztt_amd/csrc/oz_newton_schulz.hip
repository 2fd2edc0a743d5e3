// The Newton-Schulz iteration (oz_newton_schulz.hpp): its launches, and the products of the first parts alone.
#include "oz_internal.hpp"
#include "oz_newton_schulz_tiles.hpp"

#include <algorithm>
#include <cmath>

extern template void ozn::launch_products<true>(hipStream_t, Phase, int, const Shapes&, const Ends&, const Pass&);
template void ozn::launch_products<false>(hipStream_t, Phase, int, const Shapes&, const Ends&, const Pass&);

namespace {

using namespace ozn;

// Tiles of one size: outputs on a side, workgroups that a CU holds, us for a stage of 64 values of c with one of them there and with all,
// us besides for A and B and for X. Fitted to launches on 256 CUs: 8192^2's 512 and 1024 tiles of 256 x 256 (402, 398 and 863 us) and 2048 of
// 128 x 128 (484), 9216 of 32 stages for four large blocks (695), 3 to 198 tiles of 64 x 64 of 6 to 72 stages (6.0 to 24.4); of both
// parts 3 to 198 of 64 x 64 of 2 to 24 stages (5.2 to 16.6) and 540 of 8 and 24 (27.6), 216 of 128 x 128 of 11 (22.2) and 512 of 8 (42).
struct Cost {
    int tile, per_cu;
    float alone, full, square, update;
};
constexpr Cost kOne[] = {{256, 1, 1.42f, 1.42f, 19.0f, 34.0f}, {128, 2, 0.57f, 0.86f, 10.0f, 10.0f}, {64, 2, 0.26f, 0.34f, 4.7f, 5.2f}};
constexpr Cost kBoth[] = {{128, 1, 1.0f, 1.0f, 13.5f, 12.0f}, {64, 2, 0.455f, 0.8f, 4.8f, 5.2f}};

long long up(int n, int tile) { return (n + tile - 1) / tile; }

// Tiles of a matrix.
long long tiles_of(const Shape& s, Phase phase, int tile) {
    const long long t = up(side_of(s), tile);
    return phase == UPDATE ? up(s.R, tile) * up(s.C, tile) : t * (t + 1) / 2;
}
int stages_of(const Shape& s, Phase phase) { return (phase == GRAM ? std::max(s.R, s.C) : side_of(s)) / 64; }

// The tiles of a sequence that a launch has: of shape k, n[k] from begin[k] on.
struct Stretch {
    long long begin[kShapes], n[kShapes];
    long long all(const Shapes& m) const {
        long long a = 0;
        for (int k = 0; k < m.n; k++) a += n[k];
        return a;
    }
};

// Estimated us of a launch: whole rounds of workgroups over the CUs and the last, partly filled one where all tiles are alike; else what they
// take together, dealt out over the CUs, and, as they end at different times, half of the longest one's more.
float estimate(const Shapes& m, Phase phase, const Cost& c, int cus, const Stretch& t) {
    const long long slots = (long long)cus * c.per_cu, tiles = t.all(m);
    float all = 0.0f, longest = 0.0f, same = -1.0f;
    bool alike = true;
    for (int k = 0; k < m.n; k++) {
        if (!t.n[k]) continue;
        const float us = (phase == UPDATE ? c.update : c.square) + (float)stages_of(m.s[k], phase) * (tiles > cus ? c.full : c.alone);
        all += us * (float)t.n[k] / (float)slots;
        longest = std::max(longest, us);
        if (same >= 0.0f && same != us) alike = false;
        same = us;
    }
    if (alike) return (float)((tiles + slots - 1) / slots) * longest;
    return std::max(longest, all + 0.5f * longest);
}

// A phase in tiles of one size, and what a last, partly filled round of them would have in smaller ones by a launch of its own: 8192^2's A in
// 512 tiles of 256 x 256 and the other 16 of 528 as 256 of 64 x 64 takes 434 us for 563. The launch costs 3 us.
// Against every tile alone at 42 other sizes the choice is the fastest or within 2% of the whole call at 210 of 216 phases; of X in 128 x 128 tiles it cuts a last
// round off that had better stayed (6000 x 2000 9%, 1700 x 6800 8%, 3300^2 7%). There are no ranges of c: a side of 64 or less has one workgroup a matrix for A, however
// long the other one is (64 x 8192 280 us in all, 64 x 65536 1800).
struct Choice {
    int tile, rest_tile;
    Stretch main, rest;
};
template <int N>
Choice choose(const Shapes& m, Phase phase, int cus, const Cost (&costs)[N]) {
    Choice best{};
    float least = 0.0f;
    for (const Cost& c : costs) {
        Choice all{};
        all.tile = all.rest_tile = c.tile;
        for (int k = 0; k < m.n; k++) all.main.n[k] = tiles_of(m.s[k], phase, c.tile) * m.s[k].count;
        float us = estimate(m, phase, c, cus, all.main);
        if (least == 0.0f || us < least) least = us, best = all;
        const long long slots = (long long)cus * c.per_cu, over = all.main.all(m) % slots;
        if (!over || over == all.main.all(m)) continue;
        Choice cut = all;
        long long left = over;
        for (int k = m.n - 1; k >= 0 && left; k--) {
            const long long n = std::min(left, cut.main.n[k]);
            cut.main.n[k] -= n;
            cut.rest.n[k] = n;
            cut.rest.begin[k] = cut.main.n[k];
            left -= n;
        }
        us = estimate(m, phase, c, cus, cut.main) + 3.0f;
        for (const Cost& d : costs) {
            if (d.tile >= c.tile) continue;
            Stretch r = cut.rest;
            for (int k = 0; k < m.n; k++) r.n[k] *= (c.tile / d.tile) * (c.tile / d.tile);
            const float more = estimate(m, phase, d, cus, r);
            if (us + more < least) least = us + more, best = cut, best.rest_tile = d.tile;
        }
    }
    return best;
}

// A launch's places, or false where there are too many.
bool places(const Shapes& m, Phase phase, int parent, int tile, const Stretch& t, Pass* p) {
    long long at = 0;
    p->parent = parent;
    for (int k = 0; k < m.n; k++) {
        const long long per = tiles_of(m.s[k], phase, parent);
        p->places.first[k] = (int)at;
        p->places.per[k] = (int)per;
        p->begin[k] = (int)t.begin[k];
        at += t.n[k] * (parent / tile) * (parent / tile);
        if (per >> 24 || at >> 24 || (t.begin[k] + t.n[k]) >> 24) return false;  // 2^32 threads along a dimension
    }
    p->places.first[m.n] = (int)at;
    return true;
}

}  // namespace

// Singular values begin within 0 to 1 and go through s <- s (a + b s^2 + c s^4). A's values are at most their largest square, B's the
// largest |b q + c q^2| of the squares q.
ozn::Factors ozn::factors_of(double a, double b, double c, int steps) {
    double range = 1.0, all = 1.0;
    for (int k = 1; k < steps && all < kMaxSingular; k++) {
        double most = 0.0;
        const auto look = [&](double q) {
            if (q >= 0.0 && q <= range * range) most = std::max(most, std::sqrt(q) * std::fabs(a + b * q + c * q * q));
        };
        look(range * range);
        const double root = std::sqrt(9.0 * b * b - 20.0 * a * c);  // where a + 3 b q + 5 c q^2 is 0; NaN: nowhere
        look((-3.0 * b + root) / (10.0 * c));
        look((-3.0 * b - root) / (10.0 * c));
        look(-a / (3.0 * b));
        range = std::min(most, kMaxSingular);
        all = std::max(all, range);
    }
    const double q = all * all, top = -b / (2.0 * c);
    double most = std::fabs(b * q + c * q * q);
    if (top > 0.0 && top < q) most = std::max(most, std::fabs(b * top + c * top * top));
    const auto scale = [](double x) { return std::exp2(std::floor(std::log2(std::min(std::max(kLargest / x, 1.0), 16384.0)))); };
    const double of_a = scale(q), of_b = scale(most);
    return {(float)a, (float)(b * of_b / of_a), (float)(c * of_b / (of_a * of_a)), (float)(1.0 / of_b), (float)(of_a / kScale / kScale)};
}

int ozn::prepare(oz_dev* dev, const Shapes& m, const Factors& f, Iteration* it) {
    Shapes part[2] = {};
    for (int k = 0; k < m.n; k++) {
        Shapes& p = part[m.s[k].three];
        p.s[p.n++] = m.s[k];
    }
    for (int three = 0; three < 2; three++) {
        Launches& l = it->of[three];
        l = Launches{};
        for (const Phase phase : {GRAM, SQUARE, UPDATE}) {
            Shapes& order = l.order[phase];
            order = part[three];
            if (!order.n) continue;
            std::stable_sort(order.s, order.s + order.n, [&](const Shape& a, const Shape& b) { return stages_of(a, phase) > stages_of(b, phase); });
            const Choice c = three ? choose(order, phase, dev->cus, kBoth) : choose(order, phase, dev->cus, kOne);
            l.tile[phase][0] = c.tile, l.tile[phase][1] = c.rest_tile;
            if (!places(order, phase, c.tile, c.tile, c.main, &l.pass[phase][0]) || !places(order, phase, c.tile, c.rest_tile, c.rest, &l.pass[phase][1]))
                return oz::fail(dev, OZ_ERR_ARG, "too many values in matrices");
            for (Pass& p : l.pass[phase]) p.f = f;
        }
    }
    return OZ_OK;
}

int ozn::iterate(oz_dev* dev, Iteration* it, const Ends& ends, int steps) {
    for (int three = 0; three < 2; three++) {
        Launches& l = it->of[three];
        for (int k = 0; k < steps; k++)
            for (const Phase phase : {GRAM, SQUARE, UPDATE})
                for (int part = 0; part < 2; part++) {
                    const Shapes& order = l.order[phase];
                    Pass& p = l.pass[phase][part];
                    if (!order.n || !p.places.first[order.n]) continue;
                    p.from = k & 1;
                    p.last = k + 1 == steps;
                    if (three) launch_products<true>(dev->stream, phase, l.tile[phase][part], order, ends, p);
                    else launch_products<false>(dev->stream, phase, l.tile[phase][part], order, ends, p);
                    if (int st = oz::launch_check(dev, "newton_schulz_kernel")) return st;
                }
    }
    return OZ_OK;
}

// The tile of a phase's products over `count` matrices of one size, and in *rest that of a last round's own launch or 0, for tests.
extern "C" int oz_rule_newton_schulz(int cus, int phase, int rows, int cols, int count, int three, int* rest) {
    Shapes m{};
    m.n = 1;
    Shape& s = m.s[0];
    s.rows = rows, s.cols = cols, s.count = count, s.three = three;
    s.R = (int)up(rows, kPad) * kPad, s.C = (int)up(cols, kPad) * kPad;
    const Choice c = three ? choose(m, (Phase)phase, cus, kBoth) : choose(m, (Phase)phase, cus, kOne);
    if (rest) *rest = c.rest.n[0] ? c.rest_tile : 0;
    return c.tile;
}

// The scales of A and B for the iteration's factors, for tests.
extern "C" void oz_rule_newton_schulz_scales(double a, double b, double c, int steps, double* of_a, double* of_b) {
    const Factors f = factors_of(a, b, c, steps);
    *of_a = (double)f.gram * kScale * kScale;
    *of_b = 1.0 / f.update;
}
