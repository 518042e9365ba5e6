// rec_scan.hpp -- the gated linear recurrence of each channel over sequences
// (forward and backward) and for single tokens:
//
//   r = sigmoid(ga + bias_a), i = sigmoid(gx + bias_x)
//   a = exp(-rate softplus(decay) r), m = sqrt(1 - a^2)
//   h_t = a h_{t-1} + m i x,  out = h_t
//
// A workgroup has 64 channels.  A lane takes four neighbouring channels through a
// segment of S tokens, the four rows of 16 lanes of a wave four segments that
// follow one another, its waves the segments behind those: a tile of 4 S waves
// tokens.  A lane works out a and b = m i x of its tokens once and keeps them in
// registers; what a segment does to the state that enters it is h -> p h + q, with
// p the product of its a and q its own state from 0.  These pairs pass from row to
// row by lane exchanges and from wave to wave through LDS, and each lane runs over
// its tokens again from the state that then enters them.
//
// From tile to tile of a chain they pass through memory, in one launch.  A word of 8
// bytes holds a float and the launch's tag, so that what is read with the tag is
// whole and of this launch, and no order of memory has to be kept.  Every tile writes
// its pair; a tile composes those of the tiles before it in its group of
// FG_REC_GROUP and the state that leaves the group before, which that group's last
// tile writes: from left to right, so that a result does not depend on who was
// first.  Workgroups take their tiles by a ticket, first tiles first: who waits does
// so for workgroups that hold earlier tickets, and of those that hold one the
// earliest waits for nobody, so every wait ends.  The tickets count on from launch
// to launch, and their number gives the tag: nothing has to be cleared between
// launches, also when a graph replays them.
//
// Packed sequences are one chain of rows: a sequence's first token takes its
// initial state in place of the one before it.
#pragma once

#include "rec_args.h"
#include "ssm_common.hpp"

namespace fg {
namespace rec {

using namespace ssm;

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
    const float y = k * r, z = y + y;
    const float a = exp2_(y);
    constexpr float c1 = kLn2, c2 = c1 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4, c5 = c4 * kLn2 / 5;
    const float near1 = -z * fmaf(z, fmaf(z, fmaf(z, fmaf(z, c5, c4), c3), c2), c1);
    return {a, z > -0.25f ? near1 : fmaf(-a, a, 1.0f)};
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
__device__ __forceinline__ Place place_of(const fg_rec_kargs& g) {
    const uint32_t across = g.blocks * g.chains;
    uint32_t at = blockIdx.x, tag = 0;
    if (g.chain) {
        __shared__ unsigned long long ticket;
        if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(g.chain, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const uint64_t mine = ticket, places = (uint64_t)across * g.tiles;
        uint64_t launch = __umul64hi(mine, g.over_places);  // mine / places, or one less
        uint64_t rest = mine - launch * places;
        if (rest >= places) {
            rest -= places;
            ++launch;
        }
        at = uniform((uint32_t)rest);
        tag = uniform((uint32_t)(launch % 0xffffffffull) + 1);  // never 0, which memory starts with
    }
    Place p;
    p.tile = at / across;
    const uint32_t rest = at - p.tile * across;
    p.chain = rest / g.blocks;
    p.block = rest - p.chain * g.blocks;
    p.tag = tag;
    return p;
}

__device__ __forceinline__ unsigned long long* words(const fg_rec_kargs& g, const Place& p, uint32_t tile) {
    return g.chain + 8 +
           (((uint64_t)tile * g.chains + p.chain) * g.blocks + p.block) * (FG_REC_WORDS * FG_REC_CHANNELS);
}
__device__ __forceinline__ void tell(unsigned long long* to, uint32_t tag, float v) {
    __hip_atomic_store(to, (unsigned long long)tag << 32 | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long ask(const unsigned long long* from) {
    return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// For the first wave, a lane for each channel: tells the tile's pair p, q and returns
// the state that enters the tile, `first` for a chain's first one.
template <bool PACKED>
__device__ __forceinline__ float entering(const fg_rec_kargs& g, const Place& at, float p, float q, float first) {
    const uint32_t lane = threadIdx.x, in_group = at.tile % FG_REC_GROUP;
    const bool last = at.tile + 1 == g.tiles;
    unsigned long long* mine = words(g, at, at.tile) + lane;
    if (!last) {
        tell(mine, at.tag, p);
        tell(mine + FG_REC_CHANNELS, at.tag, q);
    }
    unsigned long long w[2 * FG_REC_GROUP];
    float state = first;
    // Waits end, as above; the count bounds them all the same, with NaN for what has not come.
    for (uint32_t tries = 0;; ++tries) {
        bool all = true;
        each<FG_REC_GROUP - 1>([&](auto k) {
            if (k < in_group) {
                const unsigned long long* from = words(g, at, at.tile - in_group + k) + lane;
                w[2 * k] = ask(from);
                w[2 * k + 1] = ask(from + FG_REC_CHANNELS);
            }
        });
        if (at.tile >= FG_REC_GROUP) w[2 * FG_REC_GROUP - 1] = ask(words(g, at, at.tile - in_group - 1) + lane + 2 * FG_REC_CHANNELS);
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
    if (!last && in_group == FG_REC_GROUP - 1) tell(mine + 2 * FG_REC_CHANNELS, at.tag, enter<PACKED>(p, q, state));
    return state;
}

template <class T, bool WIDE, bool PACKED>
struct Rec {
    using raw = typename T::raw;
    static constexpr int V = 4;
    struct __attribute__((aligned(V * sizeof(raw)))) Pack {
        raw v[V];
    };

    // A lane's place in the wave's tokens, and its channels.
    struct Lane {
        uint32_t lane, row, ch;  // ch: within the workgroup's 64
        uint32_t left;           // channels from ch on
    };
    static __device__ __forceinline__ Lane lane_of(const fg_rec_kargs& g, uint32_t block) {
        Lane l;
        l.lane = threadIdx.x & 63;
        l.row = l.lane >> 4;
        l.ch = (l.lane & 15) * V;
        const uint32_t all = g.channels - block * FG_REC_CHANNELS;
        l.left = l.ch < all ? all - l.ch : 0;
        return l;
    }

    // Four floats of the workgroup's channels; 0 beyond them.
    static __device__ __forceinline__ void params(float (&x)[V], const float* p, const Lane& l) {
        if constexpr (WIDE) {
            const float4 v = p && l.left ? *(const float4*)(p + l.ch) : make_float4(0, 0, 0, 0);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
            each<V>([&](auto c) { x[c] = p && c < l.left ? p[l.ch + c] : 0.0f; });
        }
    }
    static __device__ __forceinline__ void put(float* p, const Lane& l, const float (&x)[V]) {
        if constexpr (WIDE) {
            if (l.left) *(float4*)(p + l.ch) = make_float4(x[0], x[1], x[2], x[3]);
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
               uniform(((int64_t)chain * v.seq + t * v.row + (int64_t)block * FG_REC_CHANNELS) * (int64_t)sizeof(raw));
    }
    static __device__ __forceinline__ Pack fetch(const char* p, uint32_t off, const Lane& l) {
        if constexpr (WIDE) {
            return *(const Pack*)(p + off);
        } else {
            Pack k;  // channels beyond the last one load it again
            each<V>([&](auto c) {
                const uint32_t at = l.left == 0 ? 0 : c < l.left ? c : l.left - 1;
                k.v[c] = *(const raw*)(p + off + at * sizeof(raw));
            });
            return k;
        }
    }
    static __device__ __forceinline__ void store(char* p, uint32_t off, const Lane& l, const float (&x)[V]) {
        if constexpr (WIDE) {
            Pack k;
            each<V>([&](auto c) { k.v[c] = T::down(x[c]); });
            if (l.left) *(Pack*)(p + off) = k;
        } else {
            each<V>([&](auto c) {
                if (c < l.left) *(raw*)(p + off + c * sizeof(raw)) = T::down(x[c]);
            });
        }
    }

    // Which of a segment's S tokens are a sequence's, and where sequences begin
    // and end; dense: all up to the chain's end.
    template <int S>
    struct Marks {
        uint32_t in = 0, first = 0, last = 0;
        int32_t seq[PACKED ? S : 1];
    };
    static __device__ __forceinline__ int64_t offset(const fg_rec_kargs& g, uint32_t s) {
        const int64_t v = g.offsets[s], all = (int64_t)g.tokens;
        return v < 0 ? 0 : v > all ? all : v;
    }
    template <int S>
    static __device__ __forceinline__ Marks<S> marks(const fg_rec_kargs& g, int64_t t) {
        Marks<S> m;
        const int64_t left = (int64_t)g.tokens - t;
        if constexpr (!PACKED) {
            m.in = left >= S ? (1u << S) - 1 : left > 0 ? (1u << left) - 1 : 0;
        } else {
            uint32_t lo = 0, hi = g.seqs;  // the sequences whose end is at t or before it
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                if (offset(g, mid + 1) <= t) lo = mid + 1;
                else hi = mid;
            }
            uint32_t s = lo;
            int64_t a = s < g.seqs ? offset(g, s) : 0, b = s < g.seqs ? offset(g, s + 1) : 0;
            each<S>([&](auto j) {
                const int64_t at = t + j;
                while (s < g.seqs && b <= at) {
                    ++s;
                    a = b;
                    if (s < g.seqs) b = offset(g, s + 1);
                }
                const bool in = s < g.seqs && a <= at && j < left;
                m.in |= (uint32_t)in << j;
                m.first |= (uint32_t)(in && a == at) << j;
                m.last |= (uint32_t)(in && b == at + 1) << j;
                m.seq[j] = (int32_t)s;
            });
        }
        return m;
    }

    // The pair of the rows before this one (forward) or behind it (backward) in
    // the wave, and in p, q that of them with this row's own.
    template <bool BACK>
    static __device__ __forceinline__ void rows(float (&p)[V], float (&q)[V], float (&ep)[V], float (&eq)[V],
                                                const Lane& l) {
        const uint32_t row = BACK ? 3 - l.row : l.row;
        each<2>([&](auto step) {
            constexpr int far = 16 << step;
            const int from = (int)l.lane + (BACK ? far : -far);
            const bool some = row >= (1u << step);
            each<V>([&](auto c) {
                const float p1 = __shfl(p[c], from & 63), q1 = __shfl(q[c], from & 63);
                if (some) {
                    q[c] = enter<PACKED>(p[c], q[c], q1);
                    p[c] = through<PACKED>(p1, p[c]);
                }
            });
        });
        const int from = (int)l.lane + (BACK ? 16 : -16);
        each<V>([&](auto c) {
            const float p1 = __shfl(p[c], from & 63), q1 = __shfl(q[c], from & 63);
            ep[c] = row ? p1 : 1.0f;
            eq[c] = row ? q1 : 0.0f;
        });
    }

    // The waves' pairs, [wave][p, q][channel].
    struct Totals {
        float v[FG_REC_WAVES][2][FG_REC_CHANNELS];
    };
    template <bool BACK>
    static __device__ __forceinline__ void publish(Totals& t, uint32_t wave, const Lane& l, const float (&p)[V],
                                                   const float (&q)[V]) {
        if (l.row == (BACK ? 0 : 3)) {
            *(float4*)&t.v[wave][0][l.ch] = make_float4(p[0], p[1], p[2], p[3]);
            *(float4*)&t.v[wave][1][l.ch] = make_float4(q[0], q[1], q[2], q[3]);
        }
    }
    // From the state that enters the tile to the one that enters the wave.
    template <bool BACK>
    static __device__ __forceinline__ void pass(const Totals& t, uint32_t wave, uint32_t waves, const Lane& l,
                                                float (&h)[V]) {
        const uint32_t before = BACK ? waves - 1 - wave : wave;
        for (uint32_t k = 0; k < before; ++k) {
            const uint32_t w = BACK ? waves - 1 - k : k;
            const float4 p = *(const float4*)&t.v[w][0][l.ch], q = *(const float4*)&t.v[w][1][l.ch];
            h[0] = enter<PACKED>(p.x, q.x, h[0]);
            h[1] = enter<PACKED>(p.y, q.y, h[1]);
            h[2] = enter<PACKED>(p.z, q.z, h[2]);
            h[3] = enter<PACKED>(p.w, q.w, h[3]);
        }
    }

    // The state that enters the tile, at the lane's channels.  `first`: a chain's
    // first one, [channels of the workgroup] or null.
    template <bool BACK>
    static __device__ __forceinline__ void enter_tile(const fg_rec_kargs& g, const Place& at, const Totals& t, float* lds,
                                                      const float* first, uint32_t wave, uint32_t waves, const Lane& l,
                                                      float (&h)[V]) {
        if (g.tiles == 1) {
            params(h, first, l);
            return;
        }
        if (wave == 0) {
            float p = 1.0f, q = 0.0f;
            for (uint32_t k = 0; k < waves; ++k) {
                const uint32_t w = BACK ? waves - 1 - k : k;
                const float p2 = t.v[w][0][l.lane], q2 = t.v[w][1][l.lane];
                q = enter<PACKED>(p2, q2, q);
                p = through<PACKED>(p, p2);
            }
            const bool some = first && at.block * FG_REC_CHANNELS + l.lane < g.channels;
            lds[l.lane] = entering<PACKED>(g, at, p, q, some ? first[l.lane] : 0.0f);
        }
        __syncthreads();
        const float4 v = *(const float4*)&lds[l.ch];
        h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
    }

    // A packed sequence's row of [sequences][channels].
    static __device__ __forceinline__ const float* of(const float* p, const fg_rec_kargs& g, uint32_t s, uint32_t block) {
        return p ? p + (uint64_t)s * g.channels + (uint64_t)block * FG_REC_CHANNELS : nullptr;
    }

    // Packed: the sequences' initial states, behind the checkpoints of the rows.
    static __device__ __forceinline__ const float* inits(const fg_rec_kargs& g) { return g.check + g.checks * g.channels; }

    // Sequences without tokens: their last state is their first one.  Packed, the
    // tiles take turns at them.
    static __device__ __forceinline__ void empty(const fg_rec_kargs& g, const float* from, float* to, uint32_t block,
                                                 uint32_t chain, uint32_t tile) {
        if (!to || threadIdx.x >= FG_REC_CHANNELS || block * FG_REC_CHANNELS + threadIdx.x >= g.channels) return;
        const uint32_t ch = block * FG_REC_CHANNELS + threadIdx.x;
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

    struct Params {
        float k[V], ba[V], bx[V];
        __device__ __forceinline__ void load(const fg_rec_kargs& g, uint32_t block, const Lane& l) {
            const uint64_t at = (uint64_t)block * FG_REC_CHANNELS;
            params(k, g.decay + at, l);
            params(ba, g.bias_a ? g.bias_a + at : nullptr, l);
            params(bx, g.bias_x ? g.bias_x + at : nullptr, l);
            each<V>([&](auto c) {
                k[c] = -kLog2e * g.rate * softplus(k[c]).value;
                ba[c] *= -kLog2e;
                bx[c] *= -kLog2e;
            });
        }
    };

    static __device__ __forceinline__ void forward(const fg_rec_kargs& g) {
        constexpr int S = FG_REC_SEGMENT(sizeof(raw));
        __shared__ Totals totals;
        __shared__ float4 entered[FG_REC_CHANNELS / 4];
        const Place at = place_of(g);
        const uint32_t block = at.block, chain = at.chain, tile = at.tile;
        const uint32_t wave = uniform(threadIdx.x / 64), waves = blockDim.x / 64;
        const Lane l = lane_of(g, block);
        Params w;
        w.load(g, block, l);
        const uint64_t at0 = (uint64_t)block * FG_REC_CHANNELS;
        {
            const int64_t t0 = ((int64_t)tile * waves + wave) * (4 * S);
            const Marks<S> m = marks<S>(g, t0 + l.row * S);
            float a[S][V], b[S][V], p[V], q[V];
            const char *px = base(g.x, chain, t0, block), *pa = base(g.ga, chain, t0, block),
                       *pg = base(g.gx, chain, t0, block);
            Pack x[S], ga[S], gx[S];
            each<S>([&](auto j) {
                if (t0 + l.row * S + j < (int64_t)g.tokens && l.left) {
                    const uint32_t t = l.row * S + j;
                    x[j] = fetch(px, (uint32_t)((t * g.x.row + l.ch) * sizeof(raw)), l);
                    ga[j] = fetch(pa, (uint32_t)((t * g.ga.row + l.ch) * sizeof(raw)), l);
                    gx[j] = fetch(pg, (uint32_t)((t * g.gx.row + l.ch) * sizeof(raw)), l);
                }
            });
            each<V>([&](auto c) { p[c] = 1.0f, q[c] = 0.0f; });
            each<S>([&](auto j) {
                each<V>([&](auto c) {
                    const float r = gate(T::up(ga[j].v[c]), w.ba[c]), i = gate(T::up(gx[j].v[c]), w.bx[c]);
                    const Share s = share(w.k[c], r);
                    const bool in = m.in >> j & 1;
                    a[j][c] = in ? s.a : 1.0f;
                    b[j][c] = in ? __builtin_amdgcn_sqrtf(s.m2) * i * T::up(x[j].v[c]) : 0.0f;
                });
                if constexpr (PACKED) {
                    if (m.first >> j & 1) {
                        float init[V];
                        params(init, of(g.initial, g, m.seq[j], block), l);
                        if (g.check) put(const_cast<float*>(of(inits(g), g, m.seq[j], block)), l, init);
                        each<V>([&](auto c) { b[j][c] = fmaf(a[j][c], init[c], b[j][c]); });
                    }
                }
                each<V>([&](auto c) {
                    q[c] = PACKED && (m.first >> j & 1) ? b[j][c] : fmaf(a[j][c], q[c], b[j][c]);
                    p[c] *= a[j][c];
                });
            });
            each<V>([&](auto c) { p[c] = PACKED && m.first ? -1.0f : fmaxf(p[c], kLeast); });
            float ep[V], eq[V], h[V];
            rows<false>(p, q, ep, eq, l);
            publish<false>(totals, wave, l, p, q);
            __syncthreads();
            enter_tile<false>(g, at, totals, &entered[0].x, PACKED ? nullptr : of(g.initial, g, chain, block), wave,
                              waves, l, h);
            pass<false>(totals, wave, waves, l, h);
            if (g.check && t0 % FG_REC_CHECK == 0 && l.row == 0 && t0 < (int64_t)g.tokens)
                put(g.check + (chain * g.checks + t0 / FG_REC_CHECK) * g.channels + at0, l, h);
            each<V>([&](auto c) { h[c] = enter<PACKED>(ep[c], eq[c], h[c]); });
            char* po = const_cast<char*>(base(g.out, chain, t0, block));
            each<S>([&](auto j) {
                each<V>([&](auto c) {
                    h[c] = PACKED && (m.first >> j & 1) ? b[j][c] : fmaf(a[j][c], h[c], b[j][c]);
                });
                if (m.in >> j & 1) {
                    store(po, (uint32_t)(((l.row * S + j) * g.out.row + l.ch) * sizeof(raw)), l, h);
                    if constexpr (PACKED) {
                        if (g.final && (m.last >> j & 1)) put(const_cast<float*>(of(g.final, g, m.seq[j], block)), l, h);
                    } else if (g.final && t0 + l.row * S + j + 1 == (int64_t)g.tokens) {
                        put(const_cast<float*>(of(g.final, g, chain, block)), l, h);
                    }
                }
            });
            empty(g, g.initial, g.final, block, chain, tile);
        }
    }

    static __device__ __forceinline__ void backward(const fg_rec_kargs& g) {
        constexpr int S = FG_REC_BACK_SEGMENT;
        __shared__ Totals both[2];
        __shared__ float4 entered[FG_REC_CHANNELS / 4];
        Totals &ta = both[0], &tb = both[1];
        const Place at = place_of(g);
        const uint32_t block = at.block, chain = at.chain, tile = g.tiles - 1 - at.tile;
        const uint32_t wave = uniform(threadIdx.x / 64), waves = blockDim.x / 64;
        const Lane l = lane_of(g, block);
        Params w;
        w.load(g, block, l);
        const uint64_t at0 = (uint64_t)block * FG_REC_CHANNELS;
        float sums[3][V] = {};
        {
            const int64_t t0 = ((int64_t)tile * waves + wave) * (4 * S);
            const Marks<S> m = marks<S>(g, t0 + l.row * S);
            float a[S][V], b[S][V], p[V], q[V], rp[V], rq[V];
            const char *px = base(g.x, chain, t0, block), *pa = base(g.ga, chain, t0, block),
                       *pg = base(g.gx, chain, t0, block), *pd = base(g.out, chain, t0, block);
            Pack x[S], ga[S], gx[S], dy[S];
            each<S>([&](auto j) {
                if (t0 + l.row * S + j < (int64_t)g.tokens && l.left) {
                    const uint32_t t = l.row * S + j;
                    x[j] = fetch(px, (uint32_t)((t * g.x.row + l.ch) * sizeof(raw)), l);
                    ga[j] = fetch(pa, (uint32_t)((t * g.ga.row + l.ch) * sizeof(raw)), l);
                    gx[j] = fetch(pg, (uint32_t)((t * g.gx.row + l.ch) * sizeof(raw)), l);
                    dy[j] = fetch(pd, (uint32_t)((t * g.out.row + l.ch) * sizeof(raw)), l);
                }
            });
            each<V>([&](auto c) { p[c] = 1.0f, q[c] = 0.0f, rq[c] = 0.0f; });
            each<S>([&](auto j) {
                const bool in = m.in >> j & 1, first = PACKED && (m.first >> j & 1);
                float init[V] = {};
                if constexpr (PACKED) {
                    if (first) params(init, of(inits(g), g, m.seq[j], block), l);
                }
                each<V>([&](auto c) {
                    const float r = gate(T::up(ga[j].v[c]), w.ba[c]), i = gate(T::up(gx[j].v[c]), w.bx[c]);
                    const Share s = share(w.k[c], r);
                    a[j][c] = in ? s.a : 1.0f;
                    b[j][c] = in ? __builtin_amdgcn_sqrtf(s.m2) * i * T::up(x[j].v[c]) : 0.0f;
                    q[c] = fmaf(a[j][c], first ? init[c] : q[c], b[j][c]);
                    p[c] *= a[j][c];
                });
            });
            each<S>([&](auto k) {
                constexpr int j = S - 1 - k;
                const bool in = m.in >> j & 1, last = PACKED && (m.last >> j & 1);
                float end[V] = {};
                if constexpr (PACKED) {
                    if (last) params(end, of(g.gfinal, g, m.seq[j], block), l);
                }
                each<V>([&](auto c) {
                    const float d = in ? T::up(dy[j].v[c]) : 0.0f;
                    rq[c] = a[j][c] * (d + (last ? end[c] : rq[c]));
                });
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
            const int64_t first_token = (int64_t)tile * waves * (4 * S);
            if (first_token < (int64_t)g.tokens)
                params(h, g.check + (chain * g.checks + first_token / FG_REC_CHECK) * g.channels + at0, l);
            __syncthreads();
            pass<false>(ta, wave, waves, l, h);
            enter_tile<true>(g, at, tb, &entered[0].x, PACKED ? nullptr : of(g.gfinal, g, chain, block), wave, waves, l,
                             d);
            pass<true>(tb, wave, waves, l, d);
            each<V>([&](auto c) {
                h[c] = enter<PACKED>(ep[c], eq[c], h[c]);
                d[c] = enter<PACKED>(rep[c], req[c], d[c]);
            });
            // b becomes a h_{t-1}
            each<S>([&](auto j) {
                if constexpr (PACKED) {
                    if (m.first >> j & 1) params(h, of(inits(g), g, m.seq[j], block), l);
                }
                each<V>([&](auto c) {
                    const float kept = a[j][c] * h[c];
                    h[c] = fmaf(a[j][c], h[c], b[j][c]);
                    b[j][c] = kept;
                });
            });
            char *qx = const_cast<char*>(base(g.dx, chain, t0, block)), *qa = const_cast<char*>(base(g.dga, chain, t0, block)),
                 *qg = const_cast<char*>(base(g.dgx, chain, t0, block));
            each<S>([&](auto k) {
                constexpr int j = S - 1 - k;
                if constexpr (PACKED) {
                    if (m.last >> j & 1) params(d, of(g.gfinal, g, m.seq[j], block), l);
                }
                if (m.in >> j & 1) {
                    float gx_[V], ga_[V], dx_[V];
                    each<V>([&](auto c) {
                        const float dh = T::up(dy[j].v[c]) + d[c], xv = T::up(x[j].v[c]);
                        const float r = gate(T::up(ga[j].v[c]), w.ba[c]), i = gate(T::up(gx[j].v[c]), w.bx[c]);
                        const Share s = share(w.k[c], r);
                        // 1 / m, of a gate so far closed that m is 0: 0, as what it is multiplied with tends to
                        const float inv = s.m2 > 1.2e-38f ? __builtin_amdgcn_rsqf(s.m2) : 0.0f;
                        const float mi = s.m2 * inv * i;
                        const float log = dh * fmaf(-i * xv, s.a * s.a * inv, b[j][c]);
                        dx_[c] = dh * mi;
                        ga_[c] = log * w.k[c] * kLn2 * r * (1.0f - r);
                        gx_[c] = dx_[c] * xv * (1.0f - i);
                        sums[0][c] = fmaf(log, r, sums[0][c]);
                        sums[1][c] += ga_[c];
                        sums[2][c] += gx_[c];
                        d[c] = s.a * dh;
                    });
                    const uint32_t t = l.row * S + j;
                    if (g.dx.p) store(qx, (uint32_t)((t * g.dx.row + l.ch) * sizeof(raw)), l, dx_);
                    if (g.dga.p) store(qa, (uint32_t)((t * g.dga.row + l.ch) * sizeof(raw)), l, ga_);
                    if (g.dgx.p) store(qg, (uint32_t)((t * g.dgx.row + l.ch) * sizeof(raw)), l, gx_);
                    if constexpr (PACKED) {
                        if (g.ginitial && (m.first >> j & 1)) put(const_cast<float*>(of(g.ginitial, g, m.seq[j], block)), l, d);
                    } else if (g.ginitial && t0 + t == 0) {
                        put(const_cast<float*>(of(g.ginitial, g, chain, block)), l, d);
                    }
                }
            });
            empty(g, g.gfinal, g.ginitial, block, chain, tile);
        }
        // the parameters' sums: over the rows of a wave, then over the waves
        __syncthreads();
        float* to = &both[0].v[0][0][0];  // [wave][3][channel]
        static_assert(sizeof(both) >= 4 * 3 * FG_REC_WAVES * FG_REC_CHANNELS, "the sums fit");
        each<3>([&](auto k) {
            each<V>([&](auto c) {
                float v = sums[k][c];
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                if (l.row == 0) to[(wave * 3 + k) * FG_REC_CHANNELS + l.ch + c] = v;
            });
        });
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < 3 * FG_REC_CHANNELS; e += blockDim.x) {
            const uint32_t k = e / FG_REC_CHANNELS, ch = e % FG_REC_CHANNELS;
            float v = 0.0f;
            for (uint32_t u = 0; u < waves; ++u) v += to[(u * 3 + k) * FG_REC_CHANNELS + ch];
            if (at0 + ch < g.channels) g.part[(((uint64_t)chain * g.tiles + tile) * 3 + k) * g.channels + at0 + ch] = v;
        }
    }
};

// The parameters' gradients from the parts' sums.
__device__ __forceinline__ void reduce(const fg_rec_kargs& g) {
    const uint64_t e = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= 3ull * g.channels) return;
    const uint32_t k = e / g.channels, ch = e % g.channels;
    float* to = k == 0 ? g.gdecay : k == 1 ? g.gbias_a : g.gbias_x;
    if (!to) return;
    const float v = ordered_sum(g.part + e, 3ull * g.channels, g.parts);
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
        const float r = gate(T::up(ga.v[c]), -kLog2e * ba.v[c]), i = gate(T::up(gx.v[c]), -kLog2e * bx.v[c]);
        const Share s = share(-kLog2e * g.rate * softplus(decay.v[c]).value, r);
        h.v[c] = fmaf(s.a, h.v[c], __builtin_amdgcn_sqrtf(s.m2) * i * T::up(x.v[c]));
        out.v[c] = T::down(h.v[c]);
    });
    *(Floats*)(g.state_out + place) = h;
    *(Pack*)at(g.out) = out;
}

}  // namespace rec
}  // namespace fg
