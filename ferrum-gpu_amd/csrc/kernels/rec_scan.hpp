// rec_scan.hpp -- the gated linear recurrence of each channel over sequences
// (forward and backward) and for single tokens:
//
//   r = sigmoid(ga + bias_a), i = sigmoid(gx + bias_x)
//   a = exp(-rate softplus(decay) r), m = sqrt(1 - a^2)
//   h_t = a h_{t-1} + m i x,  out = h_t
//
// A workgroup has 64 channels.  A lane takes two neighbouring channels through a segment of
// S tokens, the two rows of 32 lanes of a wave two segments that follow one another, its
// waves the segments behind those: a tile.  A lane works out a and b = m i x of its tokens
// once and keeps them in registers; what a segment does to the state that enters it is
// h -> p h + q, with p the product of its a and q its own state from 0.  These pairs
// pass from row to row by lane exchanges and from wave to wave through LDS, and each lane runs
// over its tokens again from the state that then enters them.
//
// From tile to tile of a chain they pass through memory, in one launch.  A word of 8
// bytes holds a float and the launch's tag, so that what is read with the tag is
// whole and of this launch, and no order of memory has to be kept.  Every tile writes
// its pair; a tile composes those of the tiles before it in its group of
// FG_REC_GROUP and the state that leaves the group before, which that group's last
// tile writes: from left to right, so that a result does not depend on who was
// first.  A chain's workgroups take its tiles by a ticket, first tiles first: who waits
// does so for workgroups that hold earlier tickets of the chain, and of those that
// hold one the earliest waits for nobody, so every wait ends.  The tickets count on from
// launch to launch, and their number gives the tag: nothing has to be cleared
// between launches, also when a graph replays them.  (A ticket for all chains, taken
// 512 times at the start, kept the last workgroup waiting for 8 us.)
//
// Packed sequences are one chain of rows: a sequence's first token takes its
// initial state in place of the one before it.
//
// Measured (bfloat16, us; a copy of as many bytes would take): 4 x 2048 tokens x 4096
// channels forward 62 (40), 1 x 8192 x 2048 38 (20), 4 x 1024 x 2048 forward 20 (10), backward
// 39 (17) and 5 for the parameters' sums.  Forward is bound by its arithmetic and by memory
// about alike: 35 us of vector instructions (35 of an element: 6 exponentials, reciprocals and
// roots, which count twice) and 40 of rows, of which workgroups that start at a time do the
// one after the other; without arithmetic it would take 59, without the chain 4 less.
// Backward holds five factors of each token, so a SIMD has three waves of it, four of forward.
// Other shapes, 4 x 2048 x 4096: four channels of a lane 92 (each wave's share of the
// parameters, exchanges and addresses falls on half as many tokens), 128 channels of a
// workgroup 71, four waves of one 72, six 83 (two SIMDs of four get twice the waves), one
// workgroup through a sequence's tiles one by one 81, and 254 for 1 x 8192 x 2048.  Backward, training
// step 4 x 1024 x 2048: six waves 85, eight of half as many tokens 67, two 64, 62 so.
#pragma once

#include "rec_args.h"
#include "ssm_common.hpp"

namespace fg {
namespace rec {

using namespace ssm;

constexpr int CHANNELS = FG_REC_CHANNELS;

__device__ __forceinline__ float gate(float g, float scaled_bias) {
    return __builtin_amdgcn_rcpf(1.0f + exp2_(fmaf(-kLog2e, g, scaled_bias)));
}

// a = 2^(k r) and 1 - a^2, k = -rate softplus(decay) / ln 2.  Where a^2 is close to 1
// the difference would lose what a was rounded by, so from 2^(2 k r) > 0.84 on it is
// the series of -expm1(2 k r ln 2), whose first term left out is 2e-7 of it.
struct Share {
    float a, m2;
};
__device__ __forceinline__ Share share(float k, float r) {
    const float y = k * r, a = exp2_(y);
    constexpr float l = 2 * kLn2, c1 = -l, c2 = c1 * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5;
    const float near1 = y * fmaf(y, fmaf(y, fmaf(y, fmaf(y, c5, c4), c3), c2), c1);
    return {a, y > -0.125f ? near1 : fmaf(-a, a, 1.0f)};
}

// What a run of tokens does to the state that enters it: h -> p h + q.  Packed
// sequences: p < 0 where a sequence begins in the run (backward: ends), which the state
// does not pass whatever it is.  A product that has become too small stays above
// 0, so that an infinite state stays infinite as it does token by token.
constexpr float kLeast = 1.401298464e-45f;
template <bool PACKED>
__device__ __forceinline__ float enter(float p, float q, float h) {
    const float v = fmaf(p, h, q);
    return PACKED && p < 0.0f ? q : v;
}
template <bool PACKED>
__device__ __forceinline__ float through(float p1, float p2) {
    const float v = fmaxf(p1 * p2, kLeast);
    return PACKED && fminf(p1, p2) < 0.0f ? -1.0f : v;
}

// A workgroup's tile, counted from the end that its chain begins at, and its launch's tag.
struct Place {
    uint32_t block, chain, tile, tag;
};
// n / d and the rest, of over = (2^32 - 1) / d, which gives the quotient or one less.
__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t d, uint32_t over, uint32_t& rest) {
    uint32_t q = __umulhi(n, over);
    rest = n - q * d;
    if (rest >= d) {
        rest -= d;
        ++q;
    }
    return q;
}
__device__ __forceinline__ Place place_of(const fg_rec_kargs& g) {
    const uint32_t across = g.blocks * g.chains;
    Place p;
    uint32_t rest;
    p.tile = quotient(blockIdx.x, across, g.over_across, rest);
    // Workgroups go to the eight XCDs in turn: neighbouring channels, whose rows share lines where they
    // are not aligned to them, to the same one (training step 4 x 1024 x 2048 66.2 -> 64.8 us, packed
    // 7001 x 1500 42.6 -> 42.0).
    if (across % 8 == 0) rest = rest % 8 * (across / 8) + rest / 8;
    p.chain = quotient(rest, g.blocks, g.over_blocks, p.block);
    p.tag = 0;
    if (g.chain) {
        __shared__ unsigned long long ticket;
        if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(g.chain + 8ull * rest, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const uint64_t mine = (uint64_t)uniform((int64_t)ticket);
        uint64_t launch = __umul64hi(mine, g.over_tiles);  // mine / tiles, or one less
        uint64_t tile = mine - launch * g.tiles;
        if (tile >= g.tiles) {
            tile -= g.tiles;
            ++launch;
        }
        p.tile = (uint32_t)tile;
        p.tag = (uint32_t)launch << 1 | 1;  // never 0, which memory starts with
    }
    return p;
}

// A tile's words; the same for all lanes.
__device__ __forceinline__ char* words(const fg_rec_kargs& g, const Place& p, uint32_t tile) {
    const uint64_t across = (uint64_t)g.blocks * g.chains, place = tile * across + (uint64_t)p.chain * g.blocks + p.block;
    return (char*)g.chain + uniform((int64_t)(64 * across + place * (8 * FG_REC_WORDS * CHANNELS)));
}
// Word `which` of a thread's channel.
__device__ __forceinline__ void tell(char* at, int which, uint32_t ch, uint32_t tag, float v) {
    unsigned long long* to = (unsigned long long*)(at + 8 * CHANNELS * which + 8 * ch);
    __hip_atomic_store(to, (unsigned long long)tag << 32 | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long ask(const char* at, int which, uint32_t ch) {
    const unsigned long long* from = (const unsigned long long*)(at + 8 * CHANNELS * which + 8 * ch);
    return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// For the first wave, a thread for each channel: tells the tile's pair p, q and returns
// the state that enters the tile, `first` for a chain's first one.  ONE: only the chain's
// first tile is given it, and tells what it makes of it as its q, so that whatever another
// tile stores hangs on the first states having been read.
template <bool PACKED, bool ONE>
__device__ __forceinline__ float entering(const fg_rec_kargs& g, const Place& at, float p, float q, float first) {
    const uint32_t ch = threadIdx.x, in_group = at.tile % FG_REC_GROUP;
    const bool last = at.tile + 1 == g.tiles;
    char* mine = words(g, at, at.tile);
    if (ONE && at.tile == 0) q = enter<PACKED>(p, q, first);
    if (!last) {
        tell(mine, 0, ch, at.tag, p);
        tell(mine, 1, ch, at.tag, q);
    }
    unsigned long long w[2 * FG_REC_GROUP];
    float state = first;
    // Waits end, as above; the count bounds them all the same, with NaN for what has not come.
    for (uint32_t tries = 0;; ++tries) {
        bool all = true;
        each<FG_REC_GROUP - 1>([&](auto k) {
            if (k < in_group) {
                const char* from = words(g, at, at.tile - in_group + k);
                w[2 * k] = ask(from, 0, ch);
                w[2 * k + 1] = ask(from, 1, ch);
            }
        });
        if (at.tile >= FG_REC_GROUP) w[2 * FG_REC_GROUP - 1] = ask(words(g, at, at.tile - in_group - 1), 2, ch);
        each<FG_REC_GROUP - 1>([&](auto k) {
            if (k < in_group) all = all && w[2 * k] >> 32 == at.tag && w[2 * k + 1] >> 32 == at.tag;
        });
        if (at.tile >= FG_REC_GROUP) all = all && w[2 * FG_REC_GROUP - 1] >> 32 == at.tag;
        if (__all(all)) break;
        if (tries == 1u << 22) {
            each<2 * FG_REC_GROUP>([&](auto k) { w[k] = 0x7fc00000; });
            q = __uint_as_float(0x7fc00000);
            break;
        }
        __builtin_amdgcn_s_sleep(1);
    }
    if (at.tile >= FG_REC_GROUP) state = __uint_as_float((uint32_t)w[2 * FG_REC_GROUP - 1]);
    each<FG_REC_GROUP - 1>([&](auto k) {
        if (k < in_group)
            state = enter<PACKED>(__uint_as_float((uint32_t)w[2 * k]), __uint_as_float((uint32_t)w[2 * k + 1]), state);
    });
    if (!last && in_group == FG_REC_GROUP - 1) tell(mine, 2, ch, at.tag, enter<PACKED>(p, q, state));
    return state;
}

// An infinite x as the largest number of its sign; NaN stays.
__device__ __forceinline__ float finite(float x) {
    constexpr float most = 3.402823466e38f;
    return __builtin_elementwise_minimum(__builtin_elementwise_maximum(x, -most), most);
}

// A channel's k and its biases as gate() takes them, finite, so that a closed gate leaves the
// state whatever the parameters are, in sequences and for single tokens.
__device__ __forceinline__ float full(float rate, float decay) { return finite(-kLog2e * rate * softplus(decay).value); }
__device__ __forceinline__ float scaled(float bias) { return finite(-kLog2e * bias); }

template <class T, bool WIDE, bool PACKED, bool STREAM>
struct Rec {
    using raw = typename T::raw;
    static constexpr int V = FG_REC_LANE_CHANNELS, ROWS = FG_REC_ROWS, ROW = 64 / ROWS;  // ROW: lanes that share a token
    static_assert(ROW * V == CHANNELS && ROWS == 2, "one exchange between the rows of lanes");
    struct __attribute__((aligned(V * 4))) Floats {
        float v[V];
    };
    struct __attribute__((aligned(V * sizeof(raw)))) Pack {
        raw v[V];
    };
    // A lane's place in the wave's tokens, and its channels.
    struct Lane {
        uint32_t lane, row, ch;  // ch: within the workgroup's 64
        uint32_t left;           // channels from ch on
        uint32_t off;            // bytes from the workgroup's first channel to what the lane loads: lanes without
                                 // channels load the first ones
    };
    static __device__ __forceinline__ Lane lane_of(const fg_rec_kargs& g, uint32_t block) {
        Lane l;
        l.lane = threadIdx.x & 63;
        l.row = l.lane / ROW;
        l.ch = l.lane % ROW * V;
        const uint32_t all = g.channels - block * CHANNELS;
        l.left = l.ch < all ? all - l.ch : 0;
        l.off = l.left ? l.ch * (uint32_t)sizeof(raw) : 0;
        return l;
    }

    // Floats of the lane's channels, of the workgroup's; 0 beyond them.
    static __device__ __forceinline__ void params(float (&x)[V], const float* p, const Lane& l) {
        if constexpr (WIDE) {
            Floats f{};
            if (p && l.left) f = *(const Floats*)(p + l.ch);
            each<V>([&](auto c) { x[c] = f.v[c]; });
        } else {
            each<V>([&](auto c) { x[c] = p && c < l.left ? p[l.ch + c] : 0.0f; });
        }
    }
    static __device__ __forceinline__ void put(float* p, const Lane& l, const float (&x)[V]) {
        if constexpr (WIDE) {
            Floats f;
            each<V>([&](auto c) { f.v[c] = x[c]; });
            if (l.left) *(Floats*)(p + l.ch) = f;
        } else {
            each<V>([&](auto c) {
                if (c < l.left) p[l.ch + c] = x[c];
            });
        }
    }

    // Rows of a wave's tokens.  p: its first token's row at the workgroup's first
    // channel (uniform); off: token `at` of the wave, at the lane's channels.
    static __device__ __forceinline__ const char* base(const fg_ssm_view& v, uint32_t chain, int64_t t, uint32_t block) {
        return (const char*)v.p +
               uniform(((int64_t)chain * v.seq + t * v.row + (int64_t)block * CHANNELS) * (int64_t)sizeof(raw));
    }
    // The next row's address, by the scalar unit and when it is needed: all rows'
    // addresses ahead would not fit its registers.
    template <class P>
    static __device__ __forceinline__ P further(P p, int64_t step) {
        p += step;
        asm volatile("" : "+s"(p));
        return p;
    }
    static __device__ __forceinline__ Pack fetch(const char* p, uint32_t off, const Lane& l) {
        if constexpr (WIDE) {
            using Word = std::conditional_t<sizeof(Pack) == 4, uint32_t, uint64_t>;
            const Word* from = (const Word*)(p + off);
            return __builtin_bit_cast(Pack, STREAM ? __builtin_nontemporal_load(from) : *from);
        } else {
            Pack k;  // channels beyond the last one load it again
            each<V>([&](auto c) {
                const uint32_t at = c < l.left ? c : l.left ? l.left - 1 : 0;
                k.v[c] = *(const raw*)(p + off + at * sizeof(raw));
            });
            return k;
        }
    }
    static __device__ __forceinline__ void store(char* p, uint32_t off, const Lane& l, const float (&x)[V]) {
        if constexpr (WIDE) {
            Pack k;
            each<V>([&](auto c) { k.v[c] = T::down(x[c]); });
            using Word = std::conditional_t<sizeof(Pack) == 4, uint32_t, uint64_t>;
            Word* to = (Word*)(p + off);
            if (l.left) {
                if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(Word, k), to);
                else *to = __builtin_bit_cast(Word, k);
            }
        } else {
            each<V>([&](auto c) {
                if (c < l.left) *(raw*)(p + off + c * sizeof(raw)) = T::down(x[c]);
            });
        }
    }

    // Which of a segment's S tokens are a sequence's, and where packed ones begin and end.
    struct Marks {
        uint32_t in = 0, first = 0, last = 0;
    };
    static __device__ __forceinline__ int64_t offset(const fg_rec_kargs& g, uint32_t s) {
        const int64_t v = g.offsets[s], all = (int64_t)g.tokens;
        return v < 0 ? 0 : v > all ? all : v;
    }
    // The same for a whole wave, by scalar loads: they wait for no rows that are on their way.
    static __device__ __forceinline__ int64_t offset_of_wave(const fg_rec_kargs& g, uint32_t s) {
        using Scalars = const __attribute__((address_space(4))) int32_t*;
        const int64_t v = ((Scalars)(uint64_t)g.offsets)[uniform(s)], all = (int64_t)g.tokens;
        return v < 0 ? 0 : v > all ? all : v;
    }
    // Of the packed sequences, the first that ends behind row t.  One there is, unless the
    // offsets fall: the last one then, so that no access leaves the states' arrays.
    static __device__ __forceinline__ uint32_t sequence(const fg_rec_kargs& g, int64_t t) {
        uint32_t lo = 0, hi = g.seqs - 1;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (offset(g, mid + 1) <= t) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    }
    // The same for a whole wave, a 64th of the sequences for each lane at a time.  The first
    // look goes out ahead of the rows, so that it is not waited for behind them.
    struct Probe {
        uint32_t step;
        bool before;  // the lane's part of the sequences ends at t or before it
    };
    static __device__ __forceinline__ Probe probe(const fg_rec_kargs& g, int64_t t, uint32_t lo, uint32_t n, uint32_t lane) {
        const uint32_t step = (n + 63) / 64, part = (lane + 1) * step;
        return {step, part <= n && offset(g, lo + part) <= t};
    }
    static __device__ __forceinline__ uint32_t sequence_of_wave(const fg_rec_kargs& g, int64_t t, Probe p, uint32_t lane) {
        uint32_t lo = 0, n = g.seqs;
        while (n > 0) {
            const uint32_t parts = uniform((uint32_t)__popcll(__ballot(p.before)));
            lo += parts * p.step;
            n = min(n - parts * p.step, p.step - 1);
            if (n) p = probe(g, t, lo, n, lane);
        }
        return lo;
    }
    // Of the wave's ROWS S tokens from t0 on, those of the lane's segment.
    template <int S>
    static __device__ __forceinline__ Marks marks(const fg_rec_kargs& g, int64_t t0, const Lane& l, const Probe& look) {
        static_assert(ROWS * S <= 32, "a bit for each");
        constexpr uint32_t ALL = (1u << S) - 1;
        if constexpr (!PACKED) {
            const int64_t left = (int64_t)g.tokens - t0 - l.row * S;
            return {left >= S ? ALL : left > 0 ? (1u << (uint32_t)left) - 1 : 0, 0, 0};
        }
        const int64_t end = min(t0 + ROWS * S, (int64_t)g.tokens);
        uint32_t in = 0, first = 0, last = 0;
        for (uint32_t s = t0 < end ? sequence_of_wave(g, t0, look, l.lane) : g.seqs; s < g.seqs; ++s) {
            const int64_t a = offset_of_wave(g, s), b = offset_of_wave(g, s + 1);
            if (a >= end) break;
            if (b <= a || b <= t0) continue;  // one without tokens
            const uint32_t lo = (uint32_t)(max(a, t0) - t0), hi = (uint32_t)(min(b, end) - t0);
            in |= (uint32_t)((1ull << hi) - (1ull << lo));
            if (a >= t0) first |= 1u << lo;
            if (b <= end) last |= 1u << (hi - 1);
            if (b >= end) break;
        }
        const uint32_t shift = l.row * S;
        return {in >> shift & ALL, first >> shift & ALL, last >> shift & ALL};
    }

    // The pair of the rows before this one (forward) or behind it (backward) in
    // the wave, and in p, q that of them with this row's own.
    template <bool BACK>
    static __device__ __forceinline__ void rows(float (&p)[V], float (&q)[V], float (&ep)[V], float (&eq)[V],
                                                const Lane& l) {
        const bool behind = l.row == (BACK ? 0 : 1);
        each<V>([&](auto c) {
            const float p1 = __shfl_xor(p[c], ROW), q1 = __shfl_xor(q[c], ROW);
            ep[c] = behind ? p1 : 1.0f;
            eq[c] = behind ? q1 : 0.0f;
            if (behind) {
                q[c] = enter<PACKED>(p[c], q[c], q1);
                p[c] = through<PACKED>(p1, p[c]);
            }
        });
    }

    // The waves' pairs, [wave][p, q][channel].
    struct Totals {
        float v[FG_REC_WAVES][2][CHANNELS];
    };
    template <bool BACK>
    static __device__ __forceinline__ void publish(Totals& t, uint32_t wave, const Lane& l, const float (&p)[V],
                                                   const float (&q)[V]) {
        if (l.row == (BACK ? 0 : ROWS - 1)) each<V>([&](auto c) { t.v[wave][0][l.ch + c] = p[c], t.v[wave][1][l.ch + c] = q[c]; });
    }
    // From the state that enters the tile to the one that enters the wave.
    template <bool BACK>
    static __device__ __forceinline__ void pass(const Totals& t, uint32_t wave, uint32_t waves, const Lane& l,
                                                float (&h)[V]) {
        const uint32_t before = BACK ? waves - 1 - wave : wave;
        for (uint32_t k = 0; k < before; ++k) {
            const uint32_t w = BACK ? waves - 1 - k : k;
            const Floats p = *(const Floats*)&t.v[w][0][l.ch], q = *(const Floats*)&t.v[w][1][l.ch];
            each<V>([&](auto c) { h[c] = enter<PACKED>(p.v[c], q.v[c], h[c]); });
        }
    }

    // Forward, the last states may lie over the first ones.  Of a packed sequence the first one is part of
    // what its last one hangs on.  A dense chain's is read by its first tile alone (entering()): its first
    // wave's threads load it, 0 where p is null, ...
    static __device__ __forceinline__ float first_state(const fg_rec_kargs& g, const Place& at, const float* p) {
        const uint32_t ch = threadIdx.x;
        if (PACKED || !p || at.tile != 0) return 0.0f;
        return ch < CHANNELS && at.block * CHANNELS + ch < g.channels ? p[ch] : 0.0f;
    }
    // ... and leave it in LDS ahead of the barrier that enter_tile() stands behind, so that it has been read
    // whichever wave then stores the last one first.
    static __device__ __forceinline__ void keep_first(float* lds, float first) {
        if (!PACKED && threadIdx.x < CHANNELS) lds[threadIdx.x] = first;
    }

    // The state that enters the tile, at the lane's channels.  The chain's first one: forward, where
    // keep_first() left it; backward `first`, [channels of the workgroup] or null, which nothing is stored over.
    template <bool BACK>
    static __device__ __forceinline__ void enter_tile(const fg_rec_kargs& g, const Place& at, const Totals& t, float* lds,
                                                      const float* first, uint32_t waves, const Lane& l, float (&h)[V]) {
        constexpr bool KEPT = !PACKED && !BACK;
        if (!KEPT && g.tiles == 1) {
            params(h, first, l);
            return;
        }
        const uint32_t ch = threadIdx.x;
        if (g.tiles > 1 && ch < CHANNELS) {
            float p = 1.0f, q = 0.0f;
            for (uint32_t k = 0; k < waves; ++k) {
                const uint32_t w = BACK ? waves - 1 - k : k;
                const float p2 = t.v[w][0][ch], q2 = t.v[w][1][ch];
                q = enter<PACKED>(p2, q2, q);
                p = through<PACKED>(p, p2);
            }
            const bool some = !KEPT && first && at.block * CHANNELS + ch < g.channels;
            lds[ch] = entering<PACKED, KEPT>(g, at, p, q, KEPT ? lds[ch] : some ? first[ch] : 0.0f);
        }
        if (g.tiles > 1) __syncthreads();
        const Floats v = *(const Floats*)&lds[l.ch];
        each<V>([&](auto c) { h[c] = v.v[c]; });
    }

    // A packed sequence's row of [sequences][channels].
    static __device__ __forceinline__ const float* of(const float* p, const fg_rec_kargs& g, uint32_t s, uint32_t block) {
        return p ? p + (uint64_t)s * g.channels + (uint64_t)block * CHANNELS : nullptr;
    }

    // Packed: the sequences' initial states, behind the checkpoints of the rows.
    static __device__ __forceinline__ const float* inits(const fg_rec_kargs& g) { return g.check + g.checks * g.channels; }

    // Sequences without tokens: their last state is their first one.  Packed, the
    // tiles take turns at them.
    static __device__ __forceinline__ void empty(const fg_rec_kargs& g, const float* from, float* to, uint32_t block,
                                                 uint32_t chain, uint32_t tile) {
        if (!to) return;
        for (uint32_t k = threadIdx.x; k < CHANNELS && block * CHANNELS + k < g.channels; k += blockDim.x) {
            const uint32_t ch = block * CHANNELS + k;
            if constexpr (PACKED) {
                for (uint64_t s = tile; s < g.seqs; s += g.tiles) {
                    const uint64_t at = s * g.channels + ch;
                    if (offset(g, s) >= offset(g, s + 1)) to[at] = from ? from[at] : 0.0f;
                }
            } else if (g.tokens == 0) {
                const uint64_t at = (uint64_t)chain * g.channels + ch;
                to[at] = from ? from[at] : 0.0f;
            }
        }
    }

    struct Params {
        float k[V], ba[V], bx[V];
        __device__ __forceinline__ void load(const fg_rec_kargs& g, uint32_t block, const Lane& l) {
            const uint64_t at = (uint64_t)block * CHANNELS;
            params(k, g.decay + at, l);
            params(ba, g.bias_a ? g.bias_a + at : nullptr, l);
            params(bx, g.bias_x ? g.bias_x + at : nullptr, l);
            each<V>([&](auto c) {
                k[c] = full(g.rate, k[c]);
                ba[c] = scaled(ba[c]);
                bx[c] = scaled(bx[c]);
            });
        }
    };

    // What leaves a state as it is: a gate so far closed that a is 1 and b is 0.
    static __device__ __forceinline__ void nothing(Pack& x, Pack& ga, Pack& gx) {
        x = gx = Pack{};
        each<V>([&](auto c) { ga.v[c] = T::down(-__builtin_inff()); });
    }

    // Of N arrays (x, the gates, the output's gradient) a wave's ROWS S rows, S for each row of
    // lanes, token after token; unless FULL, only `left` of them exist: nothing() for those behind.
    template <int N, bool FULL>
    struct Source {
        const char* p[N];
        uint32_t step[N], off[N], first;
        int64_t left;
        __device__ __forceinline__ Source(const fg_ssm_view (&v)[N], uint32_t chain, int64_t t0, uint32_t block, const Lane& l,
                                          int64_t rows, uint32_t segment)
            : first(l.row * segment), left(rows) {
            each<N>([&](auto k) {
                p[k] = base(v[k], chain, t0, block);
                step[k] = (uint32_t)v[k].row * (uint32_t)sizeof(raw);
                off[k] = fresh(first * step[k] + l.off);
            });
        }
        // Token j's, the tokens before it having been fetched.
        template <int D>
        __device__ __forceinline__ void next(Pack (&to)[N][D], int at, uint32_t j, const Lane& l) {
            if constexpr (FULL) {
                each<N>([&](auto k) { to[k][at] = fetch(p[k], off[k], l); });
            } else {
                nothing(to[0][at], to[1][at], to[2][at]);
                if (N > 3) to[N - 1][at] = Pack{};
                if (first + j < left) each<N>([&](auto k) { to[k][at] = fetch(p[k], off[k], l); });
            }
            each<N>([&](auto k) { p[k] = further(p[k], step[k]); });
        }
    };

    template <bool FULL>
    static __device__ __forceinline__ void forward_tile(const fg_rec_kargs& g, const Place& at, Totals& totals,
                                                        float4 (&entered)[CHANNELS / 4]) {
        constexpr int S = FG_REC_SEGMENT(sizeof(raw));
        constexpr uint32_t ALL = (1u << S) - 1;
        const uint32_t block = at.block, chain = at.chain;
        const uint32_t wave = uniform(threadIdx.x / 64), waves = blockDim.x / 64;
        const Lane l = lane_of(g, block);
        const int64_t t0 = ((int64_t)at.tile * waves + wave) * (ROWS * S), rows_left = (int64_t)g.tokens - t0;
        Probe look{};
        if constexpr (PACKED) look = probe(g, t0, 0, g.seqs, l.lane);
        constexpr int D = FG_REC_AHEAD(S);
        Pack in[3][D];
        Source<3, FULL> source({g.x, g.ga, g.gx}, chain, t0, block, l, rows_left, S);
        each<D>([&](auto j) { source.next(in, j, j, l); });
        const float initial = first_state(g, at, PACKED ? nullptr : of(g.initial, g, chain, block));
        Params w;
        w.load(g, block, l);
        keep_first(&entered[0].x, initial);
        const Marks m = marks<S>(g, t0, l, look);
        // whether a sequence begins or ends in the wave's rows: few waves' do
        const bool edge = PACKED && !__all(m.in == ALL && !m.first && !m.last);
        float a[S][V], b[S][V], p[V], q[V];
        each<V>([&](auto c) { p[c] = 1.0f, q[c] = 0.0f; });
        each<S>([&](auto j) {
            constexpr int d = j % D;
            if constexpr (PACKED) {
                if (edge && !(m.in >> j & 1)) nothing(in[0][d], in[1][d], in[2][d]);
            }
            each<V>([&](auto c) {
                const float r = gate(T::up(in[1][d].v[c]), w.ba[c]), i = gate(T::up(in[2][d].v[c]), w.bx[c]);
                const Share s = share(w.k[c], r);
                a[j][c] = s.a;
                b[j][c] = __builtin_amdgcn_sqrtf(s.m2) * i * T::up(in[0][d].v[c]);
            });
            const bool first = PACKED && edge && (m.first >> j & 1);
            if (first) {
                float init[V];
                const uint32_t s = sequence(g, t0 + l.row * S + j);
                params(init, of(g.initial, g, s, block), l);
                if (g.check) put(const_cast<float*>(of(inits(g), g, s, block)), l, init);
                each<V>([&](auto c) { b[j][c] = fmaf(a[j][c], init[c], b[j][c]); });
            }
            each<V>([&](auto c) {
                q[c] = first ? b[j][c] : fmaf(a[j][c], q[c], b[j][c]);
                p[c] *= a[j][c];
            });
            // rows of half the segment on their way, of all of it no less time (64 us, 65 so) but more registers
            if constexpr (j + D < S) source.next(in, d, j + D, l);
            __builtin_amdgcn_sched_barrier(0);  // tokens mixed would not fit the registers of four waves
        });
        each<V>([&](auto c) { p[c] = PACKED && m.first ? -1.0f : fmaxf(p[c], kLeast); });
        float ep[V], eq[V], h[V];
        rows<false>(p, q, ep, eq, l);
        publish<false>(totals, wave, l, p, q);
        __syncthreads();
        enter_tile<false>(g, at, totals, &entered[0].x, nullptr, waves, l, h);
        pass<false>(totals, wave, waves, l, h);
        if (g.check && t0 % FG_REC_CHECK == 0 && l.row == 0 && rows_left > 0)
            put(g.check + (chain * g.checks + t0 / FG_REC_CHECK) * g.channels + (uint64_t)block * CHANNELS, l, h);
        each<V>([&](auto c) { h[c] = enter<PACKED>(ep[c], eq[c], h[c]); });
        char* po = const_cast<char*>(base(g.out, chain, t0, block));
        const uint32_t step = (uint32_t)g.out.row * (uint32_t)sizeof(raw), off = fresh(l.row * S * step + l.off);
        if (PACKED ? !edge : FULL) {
            each<S>([&](auto j) {
                each<V>([&](auto c) { h[c] = fmaf(a[j][c], h[c], b[j][c]); });
                store(po, off, l, h);
                po = further(po, step);
            });
        } else {
            each<S>([&](auto j) {
                const bool first = PACKED && (m.first >> j & 1);
                each<V>([&](auto c) { h[c] = first ? b[j][c] : fmaf(a[j][c], h[c], b[j][c]); });
                if (m.in >> j & 1) store(po, off, l, h);
                po = further(po, step);
                if constexpr (PACKED) {
                    if (g.final && (m.last >> j & 1))
                        put(const_cast<float*>(of(g.final, g, sequence(g, t0 + l.row * S + j), block)), l, h);
                }
            });
        }
        if constexpr (!PACKED) {  // tokens behind the last one left h as it was
            const int64_t mine = rows_left - l.row * S;
            if (g.final && mine > 0 && mine <= S) put(const_cast<float*>(of(g.final, g, chain, block)), l, h);
        }
        empty(g, g.initial, g.final, block, chain, at.tile);
    }

    // All but a chain's last tile are full; the two are apart from the start, since rows that may
    // not exist would keep others waiting.
    static __device__ __forceinline__ void forward(const fg_rec_kargs& g) {
        __shared__ Totals totals;
        __shared__ float4 entered[CHANNELS / 4];
        const Place at = place_of(g);
        const uint64_t tokens = blockDim.x / 64 * (ROWS * FG_REC_SEGMENT(sizeof(raw)));
        if ((at.tile + 1) * tokens <= g.tokens) forward_tile<true>(g, at, totals, entered);
        else forward_tile<false>(g, at, totals, entered);
    }

    template <bool FULL>
    static __device__ __forceinline__ void backward_tile(const fg_rec_kargs& g, const Place& at, Totals (&both)[2],
                                                         float4 (&entered)[CHANNELS / 4]) {
        constexpr int S = FG_REC_BACK_SEGMENT;
        Totals &ta = both[0], &tb = both[1];
        const uint32_t block = at.block, chain = at.chain, tile = g.tiles - 1 - at.tile;
        const uint32_t wave = uniform(threadIdx.x / 64), waves = blockDim.x / 64;
        const Lane l = lane_of(g, block);
        const uint64_t at0 = (uint64_t)block * CHANNELS;
        const int64_t t0 = ((int64_t)tile * waves + wave) * (ROWS * S), rows_left = (int64_t)g.tokens - t0;
        Probe look{};
        if constexpr (PACKED) look = probe(g, t0, 0, g.seqs, l.lane);
        Pack in[4][S];
        Source<4, FULL> source({g.x, g.ga, g.gx, g.out}, chain, t0, block, l, rows_left, S);
        each<S>([&](auto j) { source.next(in, j, j, l); });
        Params w;
        w.load(g, block, l);
        const Marks m = marks<S>(g, t0, l, look);
        // Of each token what the gradients go by: mi = m i, e = i x a^2 / m, f = x (1 - i).
        float a[S][V], r[S][V], mi[S][V], e[S][V], f[S][V], p[V], q[V], rp[V], rq[V];
        each<V>([&](auto c) { p[c] = 1.0f, q[c] = 0.0f, rq[c] = 0.0f; });
        each<S>([&](auto j) {
            const bool first = PACKED && (m.first >> j & 1);
            if constexpr (PACKED) {
                if (!(m.in >> j & 1)) {
                    nothing(in[0][j], in[1][j], in[2][j]);
                    in[3][j] = Pack{};
                }
            }
            float init[V] = {};
            if (first) params(init, of(inits(g), g, sequence(g, t0 + l.row * S + j), block), l);
            each<V>([&](auto c) {
                const float x = T::up(in[0][j].v[c]), i = gate(T::up(in[2][j].v[c]), w.bx[c]);
                r[j][c] = gate(T::up(in[1][j].v[c]), w.ba[c]);
                const Share s = share(w.k[c], r[j][c]);
                // of a gate so far closed that m^2 is 0, 1 / m is large, not infinite: it meets r, which is 0
                const float over = __builtin_amdgcn_rsqf(fmaxf(s.m2, 1e-37f));
                a[j][c] = s.a;
                mi[j][c] = s.m2 * over * i;
                e[j][c] = i * x * (s.a * s.a * over);
                f[j][c] = fmaf(-x, i, x);
                q[c] = fmaf(a[j][c], first ? init[c] : q[c], mi[j][c] * x);
                p[c] *= a[j][c];
            });
            __builtin_amdgcn_sched_barrier(0);  // tokens mixed would not fit the registers
        });
        each<S>([&](auto k) {
            constexpr int j = S - 1 - k;
            float end[V] = {};
            const bool last = PACKED && (m.last >> j & 1);
            if (last) params(end, of(g.gfinal, g, sequence(g, t0 + l.row * S + j), block), l);
            each<V>([&](auto c) { rq[c] = a[j][c] * (T::up(in[3][j].v[c]) + (last ? end[c] : rq[c])); });
        });
        each<V>([&](auto c) {
            rp[c] = PACKED && m.last ? -1.0f : fmaxf(p[c], kLeast);
            p[c] = PACKED && m.first ? -1.0f : fmaxf(p[c], kLeast);
        });
        float ep[V], eq[V], rep[V], req[V], h[V] = {}, d[V];
        rows<false>(p, q, ep, eq, l);
        rows<true>(rp, rq, rep, req, l);
        publish<false>(ta, wave, l, p, q);
        publish<true>(tb, wave, l, rp, rq);
        const int64_t first_token = (int64_t)tile * waves * (ROWS * S);
        if (first_token < (int64_t)g.tokens)
            params(h, g.check + (chain * g.checks + first_token / FG_REC_CHECK) * g.channels + at0, l);
        __syncthreads();
        pass<false>(ta, wave, waves, l, h);
        enter_tile<true>(g, at, tb, &entered[0].x, PACKED ? nullptr : of(g.gfinal, g, chain, block), waves, l, d);
        pass<true>(tb, wave, waves, l, d);
        each<V>([&](auto c) {
            h[c] = enter<PACKED>(ep[c], eq[c], h[c]);
            d[c] = enter<PACKED>(rep[c], req[c], d[c]);
        });
        // e becomes a h_{t-1} - e
        each<S>([&](auto j) {
            if constexpr (PACKED) {
                if (m.first >> j & 1) params(h, of(inits(g), g, sequence(g, t0 + l.row * S + j), block), l);
            }
            each<V>([&](auto c) {
                const float kept = a[j][c] * h[c];
                e[j][c] = kept - e[j][c];
                h[c] = fmaf(mi[j][c], T::up(in[0][j].v[c]), kept);
            });
        });
        float sums[3][V] = {};
        char* to[3];
        uint32_t step[3], off[3];
        const fg_ssm_view* outs[3] = {&g.dx, &g.dga, &g.dgx};
        each<3>([&](auto k) {
            step[k] = (uint32_t)outs[k]->row * (uint32_t)sizeof(raw);
            to[k] = const_cast<char*>(base(*outs[k], chain, t0 + S - 1, block));
            off[k] = fresh(l.row * S * step[k] + l.off);
        });
        each<S>([&](auto k) {
            constexpr int j = S - 1 - k;
            if constexpr (PACKED) {
                if (m.last >> j & 1) params(d, of(g.gfinal, g, sequence(g, t0 + l.row * S + j), block), l);
            }
            float o[3][V];
            each<V>([&](auto c) {
                const float dh = T::up(in[3][j].v[c]) + d[c], log = dh * e[j][c];
                o[0][c] = dh * mi[j][c];
                o[1][c] = log * (w.k[c] * kLn2) * fmaf(-r[j][c], r[j][c], r[j][c]);
                o[2][c] = o[0][c] * f[j][c];
                sums[0][c] = fmaf(log, r[j][c], sums[0][c]);
                sums[1][c] += o[1][c];
                sums[2][c] += o[2][c];
                d[c] = a[j][c] * dh;
            });
            if (m.in >> j & 1) {
                each<3>([&](auto n) {
                    if (outs[n]->p) store(to[n], off[n], l, o[n]);
                });
            }
            each<3>([&](auto n) { to[n] = further(to[n], -(int64_t)step[n]); });
            if constexpr (PACKED) {
                if (g.ginitial && (m.first >> j & 1))
                    put(const_cast<float*>(of(g.ginitial, g, sequence(g, t0 + l.row * S + j), block)), l, d);
            }
        });
        if (!PACKED && g.ginitial && t0 == 0 && l.row == 0 && rows_left > 0)
            put(const_cast<float*>(of(g.ginitial, g, chain, block)), l, d);
        empty(g, g.gfinal, g.ginitial, block, chain, tile);
        // the parameters' sums: over the rows of a wave, then over the waves
        __syncthreads();
        float* all = &both[0].v[0][0][0];  // [wave][3][channel]
        static_assert(sizeof(both) >= 4 * 3 * FG_REC_WAVES * CHANNELS, "the sums fit");
        each<3>([&](auto k) {
            each<V>([&](auto c) {
                const float v = sums[k][c] + __shfl_xor(sums[k][c], ROW);
                if (l.row == 0) all[(wave * 3 + k) * CHANNELS + l.ch + c] = v;
            });
        });
        __syncthreads();
        for (uint32_t n = threadIdx.x; n < 3 * CHANNELS; n += blockDim.x) {
            const uint32_t k = n / CHANNELS, ch = n % CHANNELS;
            float v = 0.0f;
            for (uint32_t u = 0; u < waves; ++u) v += all[(u * 3 + k) * CHANNELS + ch];
            if (at0 + ch < g.channels) g.part[(((uint64_t)chain * g.tiles + tile) * 3 + k) * g.channels + at0 + ch] = v;
        }
    }

    static __device__ __forceinline__ void backward(const fg_rec_kargs& g) {
        __shared__ Totals both[2];
        __shared__ float4 entered[CHANNELS / 4];
        const Place at = place_of(g);
        const uint64_t tokens = blockDim.x / 64 * (ROWS * FG_REC_BACK_SEGMENT);
        if ((g.tiles - at.tile) * tokens <= g.tokens) backward_tile<true>(g, at, both, entered);
        else backward_tile<false>(g, at, both, entered);
    }
};

// The parameters' gradients from the parts' sums: 64 of them for a workgroup, whose waves
// share the parts.
__device__ __forceinline__ void reduce(const fg_rec_kargs& g) {
    __shared__ float sums[16][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const uint64_t all = 3ull * g.channels, e = (uint64_t)blockIdx.x * 64 + lane;
    const uint64_t each_wave = (g.parts + waves - 1) / waves, a = min(g.parts, wave * each_wave), b = min(g.parts, a + each_wave);
    sums[wave][lane] = e < all ? ordered_sum(g.part + a * all + e, all, b - a) : 0.0f;
    __syncthreads();
    if (wave || e >= all) return;
    const uint32_t k = e / g.channels, ch = e % g.channels;
    float* to = k == 0 ? g.gdecay : k == 1 ? g.gbias_a : g.gbias_x;
    if (!to) return;
    float v = 0.0f;
    for (uint32_t w = 0; w < waves; ++w) v += sums[w][lane];
    to[ch] = k == 0 ? v * -g.rate * softplus(g.decay[ch]).slope : v;
}

// One token of each row, V channels of a thread.
template <class T, int V>
__device__ __forceinline__ void step(const fg_rec_step_kargs& g) {
    using raw = typename T::raw;
    struct __attribute__((aligned(V * sizeof(raw)))) Pack {
        raw v[V];
    };
    struct __attribute__((aligned(V * 4))) Floats {
        float v[V];
    };
    const uint32_t wide = (g.channels / V + 63) / 64;
    const uint32_t wave = uniform(blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64);
    const uint32_t row = wave / wide, ch = (wave % wide * 64 + (threadIdx.x & 63)) * V;
    if (row >= g.rows || ch >= g.channels) return;
    const int64_t slot = g.slots ? (int64_t)g.slots[row] : (int64_t)row;
    const bool some = slot >= 0 && (uint64_t)slot < g.state_rows;
    const auto at = [&](const fg_ssm_view& v) { return (raw*)v.p + ((int64_t)row * v.seq + ch); };
    Pack out;
    if (!some) {
        each<V>([&](auto c) { out.v[c] = T::down(0.0f); });
        *(Pack*)at(g.out) = out;
        return;
    }
    const uint64_t place = (uint64_t)slot * g.channels + ch;
    const Pack x = *(const Pack*)at(g.x), ga = *(const Pack*)at(g.ga), gx = *(const Pack*)at(g.gx);
    Floats h = *(const Floats*)(g.state + place);
    const Floats decay = *(const Floats*)(g.decay + ch);
    Floats ba{}, bx{};
    if (g.bias_a) ba = *(const Floats*)(g.bias_a + ch);
    if (g.bias_x) bx = *(const Floats*)(g.bias_x + ch);
    each<V>([&](auto c) {
        const float r = gate(T::up(ga.v[c]), scaled(ba.v[c])), i = gate(T::up(gx.v[c]), scaled(bx.v[c]));
        const Share s = share(full(g.rate, decay.v[c]), r);
        h.v[c] = fmaf(s.a, h.v[c], __builtin_amdgcn_sqrtf(s.m2) * i * T::up(x.v[c]));
        out.v[c] = T::down(h.v[c]);
    });
    *(Floats*)(g.state_out + place) = h;
    *(Pack*)at(g.out) = out;
}

}  // namespace rec
}  // namespace fg
