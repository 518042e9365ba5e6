// The recurrence's kernels on the CPU, each array ending where nothing is mapped.
// Built for TYPE, F32 or BF16.  Arguments: channels, tokens (packed: of all sequences), and
//   dense SEQUENCES     against the definition in 64 bits, forward and backward
//   inplace SEQUENCES   the last states over the first ones, whichever wave goes first, and nothing reads
//                       the first ones once their sequences' first tiles have ended
//   step ROWS           the one-token kernel, gates and parameters infinite among them, against sequences of
//                       one token (TOKENS is 1)
//   places FIRST        where workgroups of CHANNELS blocks and TOKENS chains go, from the FIRST-th launch on
//   packed OFFSET ...   as dense; offsets that fall: for where accesses go alone
//
// Tolerances as for the GPU's results: of a state (240 + 4 tokens) u of the sum of its terms' absolute
// values, u = 2^-24, of gradients twice that, rows rounded by half a step of their type.
#include "rec_scan.hpp"

#include <memory>
#include <string>

using namespace fg::rec;
using on_cpu::Guarded;

static int failed = 0;
static void check(double got, double want, double bound, const char* name, size_t at) {
    if (std::fabs(got - want) <= bound || got == want) return;
    if (++failed < 10) printf("%s[%zu] is %g, not %g (+- %g)\n", name, at, got, want, bound);
}

static uint64_t state_of_numbers = 1;
static double random_number() {  // about normal
    double v = 0;
    for (int k = 0; k < 4; ++k) {
        uint64_t z = state_of_numbers += 0x9E3779B97F4A7C15ull;
        z = (z ^ z >> 30) * 0xBF58476D1CE4E5B9ull;
        z = (z ^ z >> 27) * 0x94D049BB133111EBull;
        v += (double)((z ^ z >> 31) >> 11) * 0x1p-53 - 0.5;
    }
    return 1.7 * v;
}

template <class T>
struct Call {
    using raw = typename T::raw;
    static constexpr double half = sizeof(raw) == 4 ? 0 : 0x1p-8, u = 0x1p-24;
    const bool packed;
    const uint32_t seqs, channels;
    const uint64_t tokens, chains, rows, blocks, checks;
    Guarded<raw> x, ga, gx, out, dy, dx, dga, dgx;
    Guarded<float> decay, ba, bx, initial, final, gfinal, ginitial, check_points, gdecay, gba, gbx;
    Guarded<int32_t> offsets;

    // tokens: of a chain
    Call(bool p, uint32_t s, uint32_t ch, uint64_t t, const std::vector<int32_t>& at)
        : packed(p), seqs(s), channels(ch), tokens(t), chains(p ? 1 : s), rows(chains * t), blocks((ch + CHANNELS - 1) / CHANNELS),
          checks((t + FG_REC_CHECK - 1) / FG_REC_CHECK), x(rows * ch), ga(rows * ch), gx(rows * ch), out(rows * ch),
          dy(rows * ch), dx(rows * ch), dga(rows * ch), dgx(rows * ch), decay(ch), ba(ch), bx(ch), initial(s * ch),
          final(s * ch), gfinal(s * ch), ginitial(s * ch), check_points(ch * (chains * checks + (p ? s : 0))), gdecay(ch),
          gba(ch), gbx(ch), offsets(p ? s + 1 : 0) {
        for (size_t i = 0; i < rows * ch; ++i)
            x[i] = number(), ga[i] = number(), gx[i] = number(), dy[i] = number();
        for (uint32_t c = 0; c < ch; ++c) {
            decay[c] = (float)(-9 + 10.0 * c / ch), ba[c] = 0.5f * (float)random_number(), bx[c] = 0.5f * (float)random_number();
        }
        for (uint32_t i = 0; i < s * ch; ++i) initial[i] = (float)random_number(), gfinal[i] = (float)random_number();
        for (size_t i = 0; i < at.size(); ++i) offsets[i] = at[i];
    }
    static raw number() { return T::down((float)random_number()); }

    // What the host passes (rec_ops.cpp).
    fg_rec_kargs args(uint64_t wave_tokens, uint64_t most_waves, uint32_t& waves) {
        fg_rec_kargs g{};
        const auto view = [&](Guarded<raw>& a) { return fg_ssm_view{a.data(), (int64_t)(tokens * channels), channels}; };
        g.x = view(x), g.ga = view(ga), g.gx = view(gx), g.out = view(out);
        g.dx = view(dx), g.dga = view(dga), g.dgx = view(dgx);
        g.decay = decay.data(), g.bias_a = ba.data(), g.bias_x = bx.data();
        g.offsets = packed ? offsets.data() : nullptr;
        g.check = check_points.data();
        g.tokens = tokens;
        g.checks = checks;
        g.seqs = seqs, g.chains = (uint32_t)chains, g.channels = channels, g.blocks = (uint32_t)blocks;
        g.rate = 8.0f;
        waves = (uint32_t)std::min<uint64_t>(most_waves, std::max<uint64_t>(1, (tokens + wave_tokens - 1) / wave_tokens));
        g.tiles = (uint32_t)std::max<uint64_t>(1, (tokens + wave_tokens * waves - 1) / (wave_tokens * waves));
        g.parts = chains * g.tiles;
        fg_rec_set_divisors(&g);
        return g;
    }

    float* final_to = final.data();
    bool gone = false;  // NaN for the first states behind the first tiles
    template <bool WIDE, bool PACKED>
    void forward(bool last) {
        uint32_t waves;
        fg_rec_kargs g = args(FG_REC_ROWS * FG_REC_SEGMENT(sizeof(raw)), FG_REC_WAVES, waves);
        Guarded<char> words(FG_REC_CHAIN_BYTES(blocks * chains, g.tiles));
        memset(words.data(), 0, words.size());
        if (g.tiles > 1) g.chain = (unsigned long long*)words.data();
        g.initial = initial.data(), g.final = final_to;
        on_cpu::launch((uint32_t)(blocks * chains * g.tiles), 64 * waves, last, [&] { Rec<T, WIDE, PACKED, false>::forward(g); },
                       [&](uint32_t workgroup) {
                           if (gone && workgroup == blocks * chains)
                               for (uint32_t i = 0; i < seqs * channels; ++i) initial[i] = NAN;
                       });
    }
    template <bool WIDE, bool PACKED>
    void backward(bool last) {
        uint32_t waves;
        fg_rec_kargs g = args(FG_REC_ROWS * FG_REC_BACK_SEGMENT, FG_REC_BACK_WAVES, waves);
        Guarded<char> words(FG_REC_CHAIN_BYTES(blocks * chains, g.tiles));
        memset(words.data(), 0, words.size());
        if (g.tiles > 1) g.chain = (unsigned long long*)words.data();
        Guarded<float> part(3ull * channels * g.parts);
        g.out = {dy.data(), (int64_t)(tokens * channels), channels};
        g.gfinal = gfinal.data(), g.ginitial = ginitial.data();
        g.part = part.data();
        g.gdecay = gdecay.data(), g.gbias_a = gba.data(), g.gbias_x = gbx.data();
        on_cpu::launch((uint32_t)(blocks * chains * g.tiles), 64 * waves, last, [&] { Rec<T, WIDE, PACKED, false>::backward(g); });
        on_cpu::launch((3 * channels + 63) / 64, 1024, last, [&] { reduce(g); });
    }
    void run(bool back, bool last) {
        const bool wide = channels % FG_REC_LANE_CHANNELS == 0;
        if (packed && wide) back ? backward<true, true>(last) : forward<true, true>(last);
        else if (packed) back ? backward<false, true>(last) : forward<false, true>(last);
        else if (wide) back ? backward<true, false>(last) : forward<true, false>(last);
        else back ? backward<false, false>(last) : forward<false, false>(last);
    }

    // Sequence s: its first row and its number of rows.
    std::pair<uint64_t, uint64_t> span(uint32_t s) {
        if (!packed) return {s * tokens, tokens};
        const int64_t a = min(max(offsets[s], 0), (int64_t)tokens), b = min(max(offsets[s + 1], 0), (int64_t)tokens);
        return {a, b - a};
    }
    static double softplus64(double v) { return v > 30 ? v : std::log1p(std::exp(v)); }

    // The results of run(false), and with `back` of run(true), against the definition.
    void compare(bool back) {
        std::vector<bool> in(rows, false);
        std::vector<double> want[3], by[3];
        for (int k = 0; k < 3; ++k) want[k].assign(channels, 0), by[k].assign(channels, 0);
        uint64_t longest = 0;
        for (uint32_t s = 0; s < seqs; ++s) longest = std::max(longest, span(s).second);
        const double f = (240 + 4 * longest) * u;
        for (uint32_t s = 0; s < seqs; ++s) {
            const auto [first, n] = span(s);
            for (uint64_t t = 0; t < n; ++t) in[first + t] = true;
            for (uint32_t c = 0; c < channels; ++c) {
                const double k = -8 * softplus64(decay[c]);
                std::vector<double> r(n), i(n), a(n), m(n), h(n + 1), size(n + 1);
                h[0] = initial[s * channels + c], size[0] = std::fabs(h[0]);
                double top = size[0];
                for (uint64_t t = 0; t < n; ++t) {
                    const size_t at = (first + t) * channels + c;
                    r[t] = 1 / (1 + std::exp(-(T::up(ga[at]) + (double)ba[c])));
                    i[t] = 1 / (1 + std::exp(-(T::up(gx[at]) + (double)bx[c])));
                    a[t] = std::exp(k * r[t]), m[t] = std::sqrt(-std::expm1(2 * k * r[t]));
                    h[t + 1] = a[t] * h[t] + m[t] * i[t] * T::up(x[at]);
                    size[t + 1] = a[t] * size[t] + std::fabs(m[t] * i[t] * T::up(x[at]));
                    top = std::max(top, size[t + 1]);
                }
                for (uint64_t t = 0; t < n; ++t) {
                    const double bound = f * top;
                    check(T::up(out[(first + t) * channels + c]), h[t + 1], bound + half * (std::fabs(h[t + 1]) + bound), "out",
                          (first + t) * channels + c);
                }
                check(final[s * channels + c], h[n], f * top, "final", s * channels + c);
                if (!back) continue;
                double d = gfinal[s * channels + c], by_d = std::fabs(d), tops[4] = {};
                std::vector<double> g[3];
                for (auto& v : g) v.resize(n);
                for (uint64_t t = n; t-- > 0;) {
                    const size_t at = (first + t) * channels + c;
                    const double xt = T::up(x[at]), dh = T::up(dy[at]) + d, by_h = std::fabs(T::up(dy[at])) + by_d;
                    const double over = a[t] * a[t] / m[t], log = dh * (a[t] * h[t] - i[t] * xt * over);
                    const double by_log = by_h * (a[t] * std::fabs(h[t]) + std::fabs(i[t] * xt) * over);
                    const double slope = -8 / (1 + std::exp(-(double)decay[c]));
                    g[0][t] = dh * m[t] * i[t], g[1][t] = log * k * r[t] * (1 - r[t]);
                    g[2][t] = dh * m[t] * xt * i[t] * (1 - i[t]);
                    const double sizes[3] = {by_h * m[t] * i[t], by_log * std::fabs(k) * r[t],
                                             by_h * m[t] * std::fabs(xt) * i[t]};
                    for (int q = 0; q < 3; ++q) tops[q] = std::max(tops[q], sizes[q]);
                    want[0][c] += log * r[t] * slope, by[0][c] += by_log * r[t] * std::fabs(slope);
                    for (int q = 1; q < 3; ++q) want[q][c] += g[q][t], by[q][c] += sizes[q];
                    d = a[t] * dh, by_d = a[t] * by_h;
                    tops[3] = std::max(tops[3], by_d);
                }
                Guarded<raw>* got[3] = {&dx, &dga, &dgx};
                const char* names[3] = {"dx", "dgate_a", "dgate_x"};
                for (int q = 0; q < 3; ++q)
                    for (uint64_t t = 0; t < n; ++t) {
                        const double bound = 2 * f * tops[q];
                        check(T::up((*got[q])[(first + t) * channels + c]), g[q][t],
                              bound + half * (std::fabs(g[q][t]) + bound) + 1e-37, names[q], (first + t) * channels + c);
                    }
                check(ginitial[s * channels + c], d, 2 * f * std::max(tops[3], by_d), "dinitial", s * channels + c);
            }
        }
        // rows of no sequence: bytes of 0xff, as they were
        for (uint64_t t = 0; t < rows; ++t)
            for (uint32_t c = 0; c < channels && !in[t]; ++c)
                for (Guarded<raw>* a : {&out, back ? &dx : &out, back ? &dga : &out, back ? &dgx : &out}) {
                    const raw v = (*a)[t * channels + c];
                    if (on_cpu::bits(v) != (sizeof(raw) == 4 ? 0xffffffffull : 0xffffull)) check(1, 0, 0, "row of no sequence", t);
                }
        Guarded<float>* sums[3] = {&gdecay, &gba, &gbx};
        const char* names[3] = {"ddecay", "dbias_a", "dbias_x"};
        for (int q = 0; back && q < 3; ++q)
            for (uint32_t c = 0; c < channels; ++c) check((*sums[q])[c], want[q][c], 2 * f * by[q][c] + 1e-37, names[q], c);
    }
};

template <class T>
static void in_place(uint32_t channels, uint64_t tokens, uint32_t seqs) {
    for (bool last : {false, true}) {
        state_of_numbers = 1;
        Call<T> apart(false, seqs, channels, tokens, {});
        state_of_numbers = 1;
        Call<T> one(false, seqs, channels, tokens, {});
        state_of_numbers = 1;
        Call<T> other(false, seqs, channels, tokens, {});
        one.final_to = one.initial.data();
        other.gone = true;
        for (Call<T>* c : {&apart, &one, &other}) c->run(false, last);
        for (size_t i = 0; i < seqs * tokens * channels; ++i) {
            check(T::up(one.out[i]), T::up(apart.out[i]), 0, "out, in place", i);
            check(T::up(other.out[i]), T::up(apart.out[i]), 0, "out, first states gone", i);
        }
        for (uint32_t i = 0; i < seqs * channels; ++i) {
            check(one.initial[i], apart.final[i], 0, "final, in place", i);
            check(other.final[i], apart.final[i], 0, "final, first states gone", i);
        }
    }
}

template <class T, int W>
static void one_token(uint32_t channels, uint32_t rows) {
    Call<T> c(false, rows, channels, 1, {});
    const float far[] = {INFINITY, -INFINITY, 0.5f};
    const auto pick = [&] { return far[(int)(1e6 * std::fabs(random_number())) % 3]; };
    for (uint32_t k = 0; k < channels; ++k) c.decay[k] = pick(), c.ba[k] = pick(), c.bx[k] = pick();
    for (uint32_t i = 0; i < rows * channels; ++i) c.ga[i] = T::down(pick()), c.gx[i] = T::down(pick());
    c.run(false, false);
    // the rows' states in slots from the last one on; the first row has none, nor has the last one
    const uint32_t slots = rows + 1;
    Guarded<float> state(slots * channels), next(slots * channels);
    Guarded<int32_t> slot(rows);
    Guarded<typename T::raw> out(rows * channels);
    for (uint32_t r = 0; r < rows; ++r) {
        slot[r] = r == 0 ? -1 : r + 1 == rows && rows > 1 ? (int32_t)slots : (int32_t)(slots - 1 - r);
        for (uint32_t k = 0; k < channels && slot[r] >= 0 && slot[r] < (int32_t)slots; ++k)
            state[slot[r] * channels + k] = c.initial[r * channels + k];
    }
    fg_rec_step_kargs g{};
    const auto view = [&](Guarded<typename T::raw>& a) { return fg_ssm_view{a.data(), channels, 0}; };
    g.x = view(c.x), g.ga = view(c.ga), g.gx = view(c.gx), g.out = view(out);
    g.decay = c.decay.data(), g.bias_a = c.ba.data(), g.bias_x = c.bx.data();
    g.state = state.data(), g.state_out = next.data(), g.slots = slot.data();
    g.state_rows = slots, g.rows = rows, g.channels = channels, g.rate = 8.0f;
    const uint32_t waves = (channels / W + 63) / 64 * rows;
    on_cpu::launch((waves + 3) / 4, 256, false, [&] { step<T, W>(g); });
    for (uint32_t r = 0; r < rows; ++r)
        for (uint32_t k = 0; k < channels; ++k) {
            const size_t i = r * channels + k;
            const bool some = slot[r] >= 0 && slot[r] < (int32_t)slots;
            const float want = some ? T::up(c.out[i]) : 0, got = T::up(out[i]);
            if (!(std::isnan(want) && std::isnan(got))) check(got, want, 1e-6 * std::fabs(want) + Call<T>::half * std::fabs(want), "out", i);
            if (!some) continue;
            const float to = next[slot[r] * channels + k], end = c.final[i];
            if (!(std::isnan(to) && std::isnan(end))) check(to, end, 1e-6 * std::fabs(end), "state", i);
            // a closed gate leaves the state whatever the parameters are
            if (std::isinf(T::up(c.ga[i])) && T::up(c.ga[i]) < 0) check(to, c.initial[i], 0, "state behind a closed gate", i);
        }
}

// Launches of every number of tiles: each channel block of each chain has its tiles once, in the order of
// its tickets, with words of its own and a tag that the launch before did not have and new memory does not.
static void places(uint32_t blocks, uint32_t chains, uint64_t first) {
    for (uint32_t tiles : {1, 2, 3, 4, 5, 7, 33, 128}) {
        fg_rec_kargs g{};
        g.blocks = blocks, g.chains = chains, g.tiles = tiles;
        fg_rec_set_divisors(&g);
        const uint64_t across = (uint64_t)blocks * chains, bytes = FG_REC_CHAIN_BYTES(across, tiles);
        Guarded<char> memory(bytes);
        for (uint64_t k = 0; k < across; ++k) *(unsigned long long*)(memory.data() + 64 * k) = first * tiles;
        if (tiles > 1) g.chain = (unsigned long long*)memory.data();
        uint32_t before = 0;
        for (uint64_t launch = first; launch < first + 4; ++launch) {
            std::vector<uint32_t> drawn(across, 0);
            std::vector<bool> taken(across * tiles, false);
            uint32_t tag = 0;
            on_cpu::launch((uint32_t)(across * tiles), 1, false, [&] {
                const Place p = place_of(g);
                if (p.block >= blocks || p.chain >= chains || p.tile >= tiles) return check(1, 0, 0, "beyond", blockIdx.x);
                check(p.tile, drawn[p.chain * blocks + p.block]++, 0, "tile", blockIdx.x);
                if (tiles == 1) return;
                if (tag == 0) tag = p.tag;
                if (p.tag != tag || p.tag == before || p.tag == 0) check(1, 0, 0, "tag", blockIdx.x);
                const uint64_t at = words(g, p, p.tile) - memory.data(), each = 8 * FG_REC_WORDS * CHANNELS;
                if (at < 64 * across || at + each > bytes || (at - 64 * across) % each || taken[(at - 64 * across) / each])
                    return check(1, 0, 0, "words", blockIdx.x);
                taken[(at - 64 * across) / each] = true;
            });
            for (uint64_t k = 0; k < across; ++k) check(drawn[k], tiles, 0, "tiles", k);
            before = tag;
        }
    }
}

template <class T>
static void all(uint32_t channels, uint64_t tokens, const std::string& kind, const std::vector<int32_t>& more) {
    const bool packed = kind == "packed", falls = packed && !std::is_sorted(more.begin(), more.end());
    const uint32_t seqs = packed ? (uint32_t)more.size() - 1 : (uint32_t)more.at(0);
    if (kind == "places") return places(channels, (uint32_t)tokens, (uint64_t)(uint32_t)more.at(0));
    if (kind == "step") return channels % 4 ? one_token<T, 1>(channels, seqs) : one_token<T, 4>(channels, seqs);
    if (kind == "inplace") return in_place<T>(channels, tokens, seqs);
    for (bool last : {false, true}) {
        Call<T> c(packed, seqs, channels, tokens, packed ? more : std::vector<int32_t>{});
        c.run(false, last);
        c.run(true, last);
        if (!falls) c.compare(true);
    }
}

int main(int argc, char** argv) {
    if (argc < 5) return 2;
    std::vector<int32_t> more;
    for (int k = 4; k < argc; ++k) more.push_back(atoi(argv[k]));
    all<fg::ssm::TYPE>(atoi(argv[1]), atoi(argv[2]), argv[3], more);
    printf("%d values off\n", failed);
    return failed != 0;
}
