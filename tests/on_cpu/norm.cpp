// The norm's and dropout's kernels on the CPU, each array ending where nothing is mapped:
// against the definition in 64 bits.  Built for TYPE, F32 or BF16.  Arguments: rows, width; or, with `bad` behind them:
// what scales say of rows that are not finite, and of their neighbours.
//
// Tolerances, u = 2^-24: a thread's sum and a team's take at most 200 + width / 64 roundings and the other
// steps of a value a dozen, so (240 + width / 64) u of the absolute values that it is a sum of, the weight's
// gradient (240 + width / 64 + rows) u; rows are rounded by half a step of their type, e4m3 by 2^-4 and, below
// its normal numbers, 2^-10.
#include "norm_rows.hpp"

#include <memory>
#include <string>

using namespace fg::norm;
using on_cpu::Guarded;

static int failed = 0;
static std::string what;
static void check(double got, double want, double bound, const char* name, size_t at) {
    if (std::fabs(got - want) <= bound) return;
    if (++failed < 10) printf("%s: %s[%zu] is %g, not %g (+- %g)\n", what.c_str(), name, at, got, want, bound);
}

template <class T>
struct Case {
    using raw = typename T::raw;
    static constexpr double half = sizeof(raw) == 4 ? 0 : 0x1p-8, u = 0x1p-24;
    static constexpr uint32_t E = 16 / sizeof(raw);
    const uint32_t rows, width;
    Guarded<float> weight{width};
    uint64_t state = 99;

    double random() {  // about normal
        double v = 0;
        for (int k = 0; k < 4; ++k) v += (double)(fg::splitmix64_at(7, state++) >> 11) * 0x1p-53 - 0.5;
        return 1.7 * v;
    }
    // Rows `pad` elements more than their width apart.
    struct Rows {
        std::unique_ptr<Guarded<raw>> a;
        fg_ssm_view view;
        double at(uint64_t r, uint32_t c) const { return T::up((*a)[r * view.row + c]); }
    };
    Rows make(uint32_t pad, bool filled) {
        Rows r;
        r.a.reset(new Guarded<raw>((size_t)(rows - 1) * (width + pad) + width));
        r.view = {r.a->data(), 0, width + pad};
        for (uint32_t i = 0; filled && i < rows; ++i)
            for (uint32_t c = 0; c < width; ++c) (*r.a)[(size_t)i * (width + pad) + c] = T::down((float)random());
        return r;
    }

    template <int C, int TEAM, bool EVEN>
    void launch(const fg_norm_kargs& g, bool back) {
        constexpr uint32_t teams = FG_NORM_THREADS(TEAM) / TEAM;
        // fewer workgroups than rows: every team has a next one to load
        const uint32_t blocks = std::max<uint32_t>(1, ((uint32_t)g.rows + teams - 1) / teams / 2);
        parts = blocks * teams;
        for (bool last : {false, true})
            on_cpu::launch(blocks, FG_NORM_THREADS(TEAM), last, [&] {
                if (back) fg::norm::Rows<T, C, TEAM, EVEN>::backward(g);
                else fg::norm::Rows<T, C, TEAM, EVEN>::forward(g);
            });
    }
    template <int C, int TEAM>
    void launch(const fg_norm_kargs& g, bool back) {
        if (width % E) launch<C, TEAM, false>(g, back);
        else launch<C, TEAM, true>(g, back);
    }
    // The host's choice (norm_ops.cpp).
    void launch(const fg_norm_kargs& g, bool back) {
        const uint32_t chunks = (width + E - 1) / E;
        const uint32_t team = chunks <= 128 ? 64 : chunks <= 256 ? 256 : chunks <= 512 ? 512 : 1024;
        const uint32_t c = team * 2 < chunks ? 0 : team < chunks ? 2 : 1;
        if (team == 64 && c == 1) launch<1, 64>(g, back);
        else if (team == 64) launch<2, 64>(g, back);
        else if (team == 256) launch<1, 256>(g, back);
        else if (team == 512) launch<1, 512>(g, back);
        else if (c == 1) launch<1, 1024>(g, back);
        else if (c == 2) launch<2, 1024>(g, back);
        else launch<0, 1024>(g, back);
    }
    uint32_t parts = 0;

    Case(uint32_t n, uint32_t w) : rows(n), width(w) {
        for (uint32_t c = 0; c < width; ++c) weight[c] = 1 + 0.3f * (float)random();
    }
    fg_norm_kargs args() const {
        fg_norm_kargs g{};
        g.rows = rows;
        g.width = width;
        g.groups = 1;
        g.eps = 1e-5f;
        g.over_width = (float)(1.0 / width);
        return g;
    }
    double rstd(const std::vector<double>& v) const {
        double s = 0;
        for (double x : v) s += x * x;
        return 1 / std::sqrt(s / width + 1e-5);
    }

    // group: 0, 32 ..: scales of so many elements, a row's; -1: no scales.
    void forward(int group, uint32_t pad) {
        Rows x = make(pad, true), residual = make(pad + 1, true), sum = make(pad, false), out = make(pad, false);
        fg_norm_kargs g = args();
        g.x = x.view, g.residual = residual.view, g.sum = sum.view;
        g.weight = weight.data();
        g.groups = group > 0 ? (width + group - 1) / group : 1;
        g.group_lanes = group > 0 ? group / E : 0;
        Guarded<float> scales(group < 0 ? 0 : (size_t)rows * g.groups);
        Guarded<uint8_t> eight(group < 0 ? 0 : (size_t)rows * width);
        g.out = out.view;
        if (group >= 0) {
            g.scales = scales.data();
            g.out = {eight.data(), 0, width};
        }
        launch(g, false);
        const double f = (240 + width / 64) * u;
        std::vector<double> v(width);
        for (uint32_t r = 0; r < rows; ++r) {
            for (uint32_t c = 0; c < width; ++c) v[c] = x.at(r, c) + residual.at(r, c);
            const double s = rstd(v);
            for (uint32_t c = 0; c < width; ++c) {
                check(sum.at(r, c), v[c], (half + 4 * u) * std::fabs(v[c]), "sum", r * width + c);
                const double y = v[c] * s * weight[c];
                if (group < 0) {
                    check(out.at(r, c), y, (half + f) * std::fabs(y), "out", r * width + c);
                    continue;
                }
                const uint32_t k = group ? c / group : 0, a = group ? k * group : 0;
                const uint32_t b = group ? min(width, a + group) : width;
                double most = 0;
                for (uint32_t i = a; i < b; ++i) most = std::max(most, std::fabs(v[i] * s * weight[i]));
                check(scales[(size_t)r * g.groups + k], most / 448, 2 * f * most / 448, "scale", r * g.groups + k);
                const double q = y / most * 448;
                check(on_cpu::e4m3(eight[(size_t)r * width + c]), q, std::fabs(q) * (0x1p-4 + 4 * f) + 0x1p-10, "out8",
                      r * width + c);
            }
        }
    }

    // Rows 1 to 4 of 6: an infinity; one where the weight is 0; a NaN; finite values whose squares pass the range.
    void not_finite(int group) {
        Rows x = make(0, true);
        weight[width / 2] = 0;
        const uint32_t at[] = {width - 1, width / 2, 0};
        const float v[] = {INFINITY, -INFINITY, NAN};
        for (int k = 0; k < 3; ++k) (*x.a)[(1 + k) * width + at[k]] = T::down(v[k]);
        for (uint32_t c = 0; c < width; ++c) (*x.a)[4 * width + c] = T::down(1e25f);
        fg_norm_kargs g = args();
        g.x = x.view;
        g.weight = weight.data();
        g.groups = group > 0 ? (width + group - 1) / group : 1;
        g.group_lanes = group > 0 ? group / E : 0;
        Guarded<float> scales((size_t)rows * g.groups);
        Guarded<uint8_t> eight((size_t)rows * width);
        g.scales = scales.data();
        g.out = {eight.data(), 0, width};
        launch(g, false);
        for (uint32_t r = 0; r < rows; ++r)
            for (uint32_t k = 0; k < g.groups; ++k) {
                const float s = scales[(size_t)r * g.groups + k];
                if (std::isnan(s) != (r > 0 && r < 5) || s < 0) check(s, r > 0 && r < 5 ? NAN : 1, -1, "scale", r * g.groups + k);
            }
    }

    void backward(uint32_t pad) {
        Rows sum = make(pad, true), dy = make(pad + 1, true), ds = make(pad, true), dx = make(pad, false),
             dr = make(pad, false);
        fg_norm_kargs g = args();
        g.x = sum.view, g.out = dy.view, g.residual = ds.view, g.dx = dx.view, g.dresidual = dr.view;
        g.weight = weight.data();
        launch(g, true);  // without the weight's gradient, and how many parts it has
        Guarded<float> part((size_t)parts * width), dw(width);
        g.part = part.data();
        launch(g, true);
        on_cpu::launch((width + 63) / 64, 1024, false, [&] { reduce(part.data(), dw.data(), width, parts); });
        const double f = (240 + width / 64) * u;
        std::vector<double> v(width), want(width), by(width);
        for (uint32_t r = 0; r < rows; ++r) {
            double along = 0, size = 0;
            for (uint32_t c = 0; c < width; ++c) {
                v[c] = sum.at(r, c);
                const double t = dy.at(r, c) * weight[c] * v[c] / width;
                along += t, size += std::fabs(t);
            }
            const double s = rstd(v);
            for (uint32_t c = 0; c < width; ++c) {
                const double n = dy.at(r, c) * weight[c], d = s * (n - v[c] * s * s * along) + ds.at(r, c);
                const double bound = f * (s * (std::fabs(n) + std::fabs(v[c]) * s * s * size) + std::fabs(ds.at(r, c)));
                check(dr.at(r, c), d, bound + half * (std::fabs(d) + bound), "dresidual", r * width + c);
                check(dx.at(r, c), d, bound + half * (std::fabs(d) + bound), "dx", r * width + c);
                want[c] += dy.at(r, c) * v[c] * s;
                by[c] += std::fabs(dy.at(r, c) * v[c] * s);
            }
        }
        for (uint32_t c = 0; c < width; ++c) check(dw[c], want[c], (f + rows * u) * by[c] + 1e-37, "dweight", c);
    }

    void dropped(uint32_t n) {
        Guarded<raw> x(n), out(n);
        for (uint32_t i = 0; i < n; ++i) x[i] = T::down((float)random());
        fg_dropout_kargs g{};
        g.x = x.data(), g.out = out.data(), g.n = n;
        g.seed = 5, g.drop = 1u << 30, g.keep = 1 / 0.75f;
        on_cpu::launch(2, 256, false, [&] { dropout<T>(g); });
        for (uint32_t i = 0; i < n; ++i) {
            const bool keep = (uint32_t)(fg::splitmix64_at(5, i / 2) >> 32 * (i % 2)) >= g.drop;
            const double want = keep ? T::up(x[i]) / 0.75 : 0;
            check(T::up(out[i]), want, (half + 4 * u) * std::fabs(want), "dropped", i);
        }
    }
};

template <class T>
static void all(uint32_t rows, uint32_t width) {
    Case<T> c(rows, width);
    for (uint32_t pad : {0, 3}) {
        for (int group : {-1, 0, 32, 128}) {
            what = "forward, group " + std::to_string(group) + ", pad " + std::to_string(pad);
            fflush(stdout);
            c.forward(group, pad);
        }
        what = "backward, pad " + std::to_string(pad);
        c.backward(pad);
    }
    what = "dropout";
    c.dropped(rows * width);
}

template <class T>
static void bad(uint32_t rows, uint32_t width) {
    Case<T> c(rows, width);
    for (int group : {0, 32, 64, 128}) {
        what = "group " + std::to_string(group);
        c.not_finite(group);
    }
}

int main(int argc, char** argv) {
    if (argc < 3) return 2;
    const uint32_t rows = atoi(argv[1]), width = atoi(argv[2]);
    if (argc > 3) bad<fg::ssm::TYPE>(rows, width);
    else all<fg::ssm::TYPE>(rows, width);
    printf("%d values off\n", failed);
    return failed != 0;
}
