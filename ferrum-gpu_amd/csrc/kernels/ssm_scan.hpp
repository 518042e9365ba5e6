// ssm_scan.hpp -- the selective scan over sequences, forward and backward:
//
//   dt = softplus(delta + bias)              h_t[d,n] = exp(dt A[d,n]) h_{t-1}[d,n] + dt u B_t[n]
//   y  = (sum_n C_t[n] h_t[d,n] + D u) silu(z)
//
// A wave takes 16 channels, lane (q, c) = (lane / 16, lane % 16) the states
// q S ... q S + S - 1 of channel c, and walks along the tokens four at a time:
//   * row q of the wave loads u, delta and z of token 4 i + q and works out its
//     time step, so that no lane does that work twice; dt and dt u go through
//     LDS to the other three rows;
//   * the four tokens' B and C of the row's states lie in the 16 lanes of a
//     register, one state of one token each, and reach the row as the DPP
//     broadcast operand of the instruction that takes them;
//   * the sums over a channel's states end with an exchange between the rows
//     that leaves token 4 i + q in row q, where its u and z are.
// The workgroup is four waves, 64 channels: 128-byte lines of a 16-bit type.
#pragma once

#include "ssm_common.hpp"

namespace fg {
namespace ssm {

// acc[s] += bcast(v[(J S + s) / 16], lane (J S + s) % 16 of the row) * x[s] for
// the S states of token J of four; X_ONE: one x for all.  One statement of
// assembly for up to four: the compiler does not fold the broadcast into a
// multiply-add, and the s_nop keeps the two wait states that a DPP operand
// needs after the instruction that wrote it.
template <int L>
__device__ __forceinline__ void fmac1(float& a, float v, float x) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf"
        : "+v"(a)
        : "v"(v), "v"(x), "n"(L));
}
template <int L>
__device__ __forceinline__ void fmac2(float& a0, float& a1, float v, float x0, float x1) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %2, %3 row_newbcast:%5 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %2, %4 row_newbcast:%6 row_mask:0xf bank_mask:0xf"
        : "+v"(a0), "+v"(a1)
        : "v"(v), "v"(x0), "v"(x1), "n"(L), "n"(L + 1));
}
template <int L>
__device__ __forceinline__ void fmac4(float& a0, float& a1, float& a2, float& a3, float v, float x0, float x1,
                                      float x2, float x3) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %4, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %4, %6 row_newbcast:%10 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %4, %7 row_newbcast:%11 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %3, %4, %8 row_newbcast:%12 row_mask:0xf bank_mask:0xf"
        : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3)
        : "v"(v), "v"(x0), "v"(x1), "v"(x2), "v"(x3), "n"(L), "n"(L + 1), "n"(L + 2), "n"(L + 3));
}
// One accumulator, four products: the same with a chain.
template <int L>
__device__ __forceinline__ void dot2(float& a, float v, float x0, float x1) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %2 row_newbcast:%4 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %3 row_newbcast:%5 row_mask:0xf bank_mask:0xf"
        : "+&v"(a)
        : "v"(v), "v"(x0), "v"(x1), "n"(L), "n"(L + 1));
}
template <int L>
__device__ __forceinline__ void dot4(float& a, float v, float x0, float x1, float x2, float x3) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %2 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %3 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %4 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf"
        : "+&v"(a)
        : "v"(v), "v"(x0), "v"(x1), "v"(x2), "v"(x3), "n"(L), "n"(L + 1), "n"(L + 2), "n"(L + 3));
}

// acc[s] += B[token J][s] * x, s < S.
template <int S, int J>
__device__ __forceinline__ void bcast_fmac(float (&acc)[S], const float* v, float x) {
    if constexpr (S == 1) fmac1<J>(acc[0], v[0], x);
    else if constexpr (S == 2) fmac2<2 * J>(acc[0], acc[1], v[0], x, x);
    else
        each<S / 4>([&](auto k) {
            constexpr int I = J * S + 4 * k;
            fmac4<I % 16>(acc[4 * k], acc[4 * k + 1], acc[4 * k + 2], acc[4 * k + 3], v[I / 16], x, x, x, x);
        });
}
// acc += sum_s B[token J][s] * x[s].
template <int S, int J>
__device__ __forceinline__ void bcast_dot(float& acc, const float* v, const float (&x)[S]) {
    if constexpr (S == 1) fmac1<J>(acc, v[0], x[0]);
    else if constexpr (S == 2) dot2<2 * J>(acc, v[0], x[0], x[1]);
    else
        each<S / 4>([&](auto k) {
            constexpr int I = J * S + 4 * k;
            dot4<I % 16>(acc, v[I / 16], x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
        });
}

// The sum over a row's 16 channels of each of v[0 .. 4 S): halving the values
// with every bit of the lane number, so that lane c ends with the sums of
// values c * (S / 4) + r in v[r] (S >= 4), of value c >> 1 or c >> 2 (S = 2, 1).
template <int N>
__device__ __forceinline__ void channels_sum(float (&v)[N], uint32_t c) {
    const bool b3 = c & 8, b2 = c & 4, b1 = c & 2, b0 = c & 1;
    auto level = [&](auto half, bool upper, auto ctrl) {
        each<half>([&](auto i) {
            const float keep = upper ? v[i + half] : v[i], give = upper ? v[i] : v[i + half];
            v[i] = keep + dpp<ctrl>(give);
        });
    };
    level(Int<N / 2>{}, b3, Int<kRor8>{});
    level(Int<N / 4>{}, b2, Int<kHalfMirror>{});
    if constexpr (N >= 8) level(Int<N / 8>{}, b1, Int<kXor2>{});
    else v[0] += dpp<kXor2>(v[0]);
    if constexpr (N >= 16) level(Int<N / 16>{}, b0, Int<kXor1>{});
    else v[0] += dpp<kXor1>(v[0]);
}

// Where a wave works: its sequence, the tokens of its chunk, its channels.
struct Place {
    int64_t start;              // packed: the sequence's first row
    uint32_t len;               // tokens of the sequence
    uint32_t seq, chunk, group, block;
    uint32_t t0, t1;            // the chunk's tokens
    uint32_t q, c, wave;
    uint32_t ch;                // the lane's channel (the group's last one where it has none)
    uint32_t wblock;            // the wave's number among all waves over channels
    bool valid;
};

__device__ __forceinline__ Place place(const fg_scan_kargs& g) {
    Place p;
    const uint32_t lane = threadIdx.x & 63;
    p.wave = uniform(threadIdx.x >> 6);
    p.q = lane >> 4;
    p.c = lane & 15;
    const uint32_t blocks = g.groups * g.group_blocks;
    const uint32_t cb = blockIdx.x % blocks, rest = blockIdx.x / blocks;
    p.group = cb / g.group_blocks;
    p.block = cb % g.group_blocks;
    p.chunk = rest % g.chunks;
    p.seq = rest / g.chunks;
    p.start = 0;
    p.len = g.length;
    if (g.offsets) {
        // offsets out of order or beyond the rows give shorter sequences, not accesses outside
        int64_t a = g.offsets[p.seq], b = g.offsets[p.seq + 1];
        const int64_t all = (int64_t)g.tokens;
        a = a < 0 ? 0 : a > all ? all : a;
        b = b < a ? a : b > all ? all : b;
        p.start = uniform(a);
        p.len = uniform((uint32_t)(b - a < (int64_t)g.length ? b - a : (int64_t)g.length));
    }
    const uint64_t first = (uint64_t)p.chunk * g.chunk_len;
    p.t0 = first < p.len ? (uint32_t)first : p.len;
    p.t1 = p.len - p.t0 < g.chunk_len ? p.len : p.t0 + g.chunk_len;
    const uint32_t in_group = p.block * FG_SSM_GROUP_CHANNELS + p.wave * FG_SSM_WAVE_CHANNELS + p.c;
    p.valid = in_group < g.group_channels;
    p.ch = p.group * g.group_channels + (p.valid ? in_group : g.group_channels - 1);
    p.wblock = cb * FG_SSM_WAVES + p.wave;
    return p;
}

template <class T, int S, bool PAD>
struct Scan {
    using raw = typename T::raw;
    static constexpr int SEG = FG_SSM_SEGMENT(S), NG = SEG / 4, NB = S >= 4 ? S / 4 : 1;
    static constexpr int ES = sizeof(raw);

    // A view's rows from token t on: a uniform address.
    static __device__ __forceinline__ const char* rows(const fg_ssm_view& v, const Place& p, uint32_t t) {
        return (const char*)v.p + ((int64_t)p.seq * v.seq + (p.start + t) * v.row) * ES;
    }
    static __device__ __forceinline__ float at(const char* base, uint32_t off) {
        return T::up(*(const raw*)(base + off));
    }

    // The lane's constants.
    struct Lane {
        uint32_t tok[NB], st[NB];  // token of four and state whose B and C the lane loads, register k
        bool has[NB];
        bool pad[S];
        float a2[S];               // A log2(e)
        float bias, skip;
    };
    static __device__ __forceinline__ Lane lane(const fg_scan_kargs& g, const Place& p) {
        Lane l;
        each<NB>([&](auto k) {
            const uint32_t i = k * 16 + p.c;
            const uint32_t tok = i / S, n = p.q * S + i % S;
            l.tok[k] = tok < 4 ? tok : 3;
            l.has[k] = n < g.states;
            l.st[k] = n < g.states ? n : g.states - 1;
        });
        each<S>([&](auto s) {
            const uint32_t n = p.q * S + s;
            l.pad[s] = PAD && n >= g.states;
            l.a2[s] = n < g.states ? g.a[(uint64_t)p.ch * g.states + n] * kLog2e : 0.0f;
        });
        l.bias = g.bias ? g.bias[p.ch] : 0.0f;
        l.skip = g.skip ? g.skip[p.ch] : 0.0f;
        return l;
    }

    // A view's rows of a segment: the uniform address of its first row, moved
    // on from segment to segment, and the lane's offsets from it.
    struct Cursor {
        const char* at;
        uint32_t row;  // bytes
        __device__ __forceinline__ void set(const fg_ssm_view& v, const Place& p, uint32_t t, uint32_t column = 0) {
            at = rows(v, p, t) + (uint64_t)column * ES;
            row = (uint32_t)v.row * ES;
        }
        __device__ __forceinline__ const char* group(int i) const { return at + (uint64_t)(4 * i) * row; }
        __device__ __forceinline__ void forth() { at += (uint64_t)SEG * row; }
        __device__ __forceinline__ void back() { at -= (uint64_t)SEG * row; }
    };

    // A segment's rows as they lie in memory.  TAIL: n < SEG of them; beyond
    // the last, the last.
    template <bool TAIL>
    static __device__ __forceinline__ void load_channels(raw (&v)[NG], const Cursor& w, const Place& p, uint32_t n) {
        each<NG>([&](auto i) {
            if constexpr (TAIL) {
                const uint32_t r = 4 * i + p.q;
                v[i] = *(const raw*)(w.at + ((r < n ? r : n - 1) * w.row + p.ch * ES));
            } else {
                v[i] = *(const raw*)(w.group(i) + (p.q * w.row + p.ch * ES));
            }
        });
    }
    template <bool TAIL>
    static __device__ __forceinline__ void load_states(raw (&v)[NG][NB], const Cursor& w, const Lane& l, uint32_t n) {
        each<NG>([&](auto i) {
            each<NB>([&](auto k) {
                if constexpr (TAIL) {
                    const uint32_t r = 4 * i + l.tok[k];
                    v[i][k] = *(const raw*)(w.at + ((r < n ? r : n - 1) * w.row + l.st[k] * ES));
                } else {
                    v[i][k] = *(const raw*)(w.group(i) + (l.tok[k] * w.row + l.st[k] * ES));
                }
            });
        });
    }
    static __device__ __forceinline__ void up_channels(float (&x)[NG], const raw (&v)[NG]) {
        each<NG>([&](auto i) { x[i] = T::up(v[i]); });
    }
    static __device__ __forceinline__ void up_states(float (&x)[NG][NB], const raw (&v)[NG][NB], const Lane& l) {
        each<NG>([&](auto i) {
            each<NB>([&](auto k) { x[i][k] = !PAD || l.has[k] ? T::up(v[i][k]) : 0.0f; });
        });
    }
    template <bool TAIL>
    static __device__ __forceinline__ void store_channels(const Cursor& w, const Place& p, int i, uint32_t n, float v) {
        if (p.valid && (!TAIL || 4 * i + p.q < n))
            *(raw*)(const_cast<char*>(w.group(i)) + (p.q * w.row + p.ch * ES)) = T::down(v);
    }
    static __device__ __forceinline__ uint64_t check_at(const fg_scan_kargs& g, const Place& p, uint32_t t) {
        const uint64_t seg = g.offsets ? (uint64_t)p.start / SEG + p.seq : (uint64_t)p.seq * g.check_segs;
        return ((seg + t / SEG) * (g.groups * g.group_blocks * FG_SSM_WAVES) + p.wblock) * (64 * S) +
               (threadIdx.x & 63) * S;
    }
    static __device__ __forceinline__ uint64_t carry_at(const fg_scan_kargs& g, const Place& p, uint32_t chunk) {
        return (((uint64_t)p.seq * (g.chunks + 1) + chunk) * (g.groups * g.group_blocks * FG_SSM_WAVES) + p.wblock);
    }
    // The lane's states there; place `chunks` holds the initial states.
    static __device__ __forceinline__ float* carry_of(const fg_scan_kargs& g, const Place& p, uint32_t chunk) {
        return g.carry + carry_at(g, p, chunk) * (64 * S) + (threadIdx.x & 63) * S;
    }
    static __device__ __forceinline__ uint64_t state_at(const fg_scan_kargs& g, const Place& p, int s) {
        return ((uint64_t)p.seq * g.channels + p.ch) * g.states + p.q * S + s;
    }
    static __device__ __forceinline__ bool has_state(const fg_scan_kargs& g, const Place& p, int s) {
        return p.q * S + s < g.states;
    }

    // What a row's token takes part with, exchanged between the wave's rows.
    template <int W>
    struct Exchange {
        static constexpr int STRIDE = SEG * W + 4;  // floats of a channel; the 4 keep the channels off each other's banks
        float v[FG_SSM_WAVES][16 * STRIDE];
    };
    static __device__ __forceinline__ void wave_sync() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // Time steps of the segment's rows: dt and its slope.
    static __device__ __forceinline__ void steps(const fg_scan_kargs& g, const Lane& l, const float (&d)[NG],
                                                 float (&dt)[NG], float (&slope)[NG]) {
        each<NG>([&](auto i) { dt[i] = d[i] + l.bias, slope[i] = 1.0f; });
        if (g.softplus) {
            each<NG>([&](auto i) {
                const Softplus s = softplus(dt[i]);
                dt[i] = s.value;
                slope[i] = s.slope;
            });
        }
    }

    // ------------------------------------------------------------ forward

    template <bool LOCAL>
    struct Segment {
        raw u[NG], d[NG], z[NG], b[NG][NB], c[NG][NB];
    };
    // The forward pass's views, at the segment that is loaded next; `out` at
    // the one that is stored next.
    template <bool LOCAL>
    struct Cursors {
        Cursor u, d, z, b, c, out;
        bool gate;
        __device__ __forceinline__ void set(const fg_scan_kargs& g, const Place& p) {
            u.set(g.u, p, p.t0);
            d.set(g.delta, p, p.t0);
            b.set(g.b, p, p.t0, p.group * g.states);
            gate = false;
            if constexpr (!LOCAL) {
                c.set(g.c, p, p.t0, p.group * g.states);
                gate = g.z.p != nullptr;
                z.set(g.z, p, p.t0);
                out.set(g.out, p, p.t0);
            }
        }
        template <bool TAIL>
        __device__ __forceinline__ void load(Segment<LOCAL>& s, const Place& p, const Lane& l, uint32_t n) {
            load_channels<TAIL>(s.d, d, p, n);
            load_channels<TAIL>(s.u, u, p, n);
            load_states<TAIL>(s.b, b, l, n);
            if constexpr (!LOCAL) {
                load_states<TAIL>(s.c, c, l, n);
                if (gate) load_channels<TAIL>(s.z, z, p, n);
                c.forth();
                z.forth();
            }
            d.forth();
            u.forth();
            b.forth();
        }
    };
    template <bool LOCAL>
    struct Values {
        float u[NG], d[NG], z[NG], b[NG][NB], c[NG][NB];
        __device__ __forceinline__ void take(const Segment<LOCAL>& s, const Lane& l) {
            up_channels(d, s.d);
            up_channels(u, s.u);
            up_states(b, s.b, l);
            if constexpr (!LOCAL) {
                up_states(c, s.c, l);
                up_channels(z, s.z);
            }
        }
    };

    template <bool LOCAL, bool TAIL>
    static __device__ __forceinline__ void forward_segment(const fg_scan_kargs& g, const Place& p, const Lane& l,
                                                           float* x, float (&h)[S], float& sum_dt,
                                                           const Values<LOCAL>& v, Cursors<LOCAL>& at, uint32_t t,
                                                           uint32_t n) {
        float dt[NG], slope[NG], out[NG];
        if constexpr (!LOCAL) {
            if (g.check) {  // lanes without a channel too: the backward pass reads them
                float* to = g.check + check_at(g, p, t);
                each<S>([&](auto s) { to[s] = h[s]; });
            }
        }
        steps(g, l, v.d, dt, slope);
        wave_sync();
        each<NG>([&](auto i) {
            const float2 e = {dt[i], dt[i] * v.u[i]};
            *(float2*)(x + (4 * i + p.q) * 2) = e;
            if constexpr (LOCAL) sum_dt += !TAIL || 4 * i + p.q < n ? dt[i] : 0.0f;
        });
        wave_sync();
        each<NG>([&](auto i) {
            float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            float e[8];
            *(float4*)e = *(const float4*)(x + 8 * i);
            *(float4*)(e + 4) = *(const float4*)(x + 8 * i + 4);
            each<4>([&](auto j) {
                if (!TAIL || 4 * i + j < n) {
                    each<S>([&](auto s) {
                        constexpr int I = j * S + s;
                        h[s] = fmaf(exp2_(e[2 * j] * l.a2[s]), h[s], row_bcast<I % 16>(v.b[i][I / 16]) * e[2 * j + 1]);
                        if (PAD && l.pad[s]) h[s] = 0.0f;
                    });
                    if constexpr (!LOCAL) bcast_dot<S, j>(y[j], v.c[i], h);
                }
            });
            if constexpr (!LOCAL) out[i] = fmaf(l.skip, v.u[i], rows_sum(y));
        });
        if constexpr (!LOCAL) {
            if (at.gate) each<NG>([&](auto i) { out[i] *= v.z[i] * sigmoid(v.z[i]); });
            each<NG>([&](auto i) { store_channels<TAIL>(at.out, p, i, n, out[i]); });
            at.out.forth();
        }
    }

    // LOCAL: the states that the chunk's own tokens leave, from none, and the
    // sum of its time steps; else outputs, from the states before the chunk.
    template <bool LOCAL>
    static __device__ __forceinline__ void forward(const fg_scan_kargs& g) {
        using X = Exchange<2>;
        __shared__ __attribute__((aligned(16))) X xs;
        const Place p = place(g);
        if (LOCAL && p.chunk == 0) {
            // the last chunks may write the final states where the initial ones lie
            each<S>([&](auto s) {
                const bool has = g.initial && has_state(g, p, s);
                carry_of(g, p, g.chunks)[s] = has ? g.initial[state_at(g, p, s)] : 0.0f;
            });
        }
        if (LOCAL && p.t1 == p.len) return;                        // no chunk follows
        if (!LOCAL && p.chunk > 0 && p.t0 == p.t1) return;          // no tokens
        const Lane l = lane(g, p);
        float* x = xs.v[p.wave] + p.c * X::STRIDE;
        float h[S];
        each<S>([&](auto s) { h[s] = 0.0f; });
        if constexpr (!LOCAL) {
            each<S>([&](auto s) {
                if (g.chunks > 1) h[s] = carry_of(g, p, g.chunks)[s];
                else if (g.initial && has_state(g, p, s)) h[s] = g.initial[state_at(g, p, s)];
            });
            for (uint32_t k = 0; k < p.chunk; ++k) {
                const float sum = g.carry_dt[carry_at(g, p, k) * 16 + p.c];
                each<S>([&](auto s) {
                    h[s] = fmaf(exp2_(sum * l.a2[s]), h[s], carry_of(g, p, k)[s]);
                    if (PAD && l.pad[s]) h[s] = 0.0f;
                });
            }
        }
        float sum_dt = 0.0f;
        Cursors<LOCAL> at;
        at.set(g, p);
        Segment<LOCAL> next;
        Values<LOCAL> now;
        uint32_t t = p.t0;
        if (t + SEG <= p.t1) at.template load<false>(next, p, l, SEG);
        while (t + SEG <= p.t1) {
            now.take(next, l);
            // the next segment's rows, while this one is worked through
            if (t + 2 * SEG <= p.t1) at.template load<false>(next, p, l, SEG);
            forward_segment<LOCAL, false>(g, p, l, x, h, sum_dt, now, at, t, SEG);
            t += SEG;
        }
        if (t < p.t1) {
            at.template load<true>(next, p, l, p.t1 - t);
            now.take(next, l);
            forward_segment<LOCAL, true>(g, p, l, x, h, sum_dt, now, at, t, p.t1 - t);
        }
        if constexpr (LOCAL) {
            const float v[4] = {sum_dt, sum_dt, sum_dt, sum_dt};
            sum_dt = rows_sum(v);
            if (p.q == 0) g.carry_dt[carry_at(g, p, p.chunk) * 16 + p.c] = sum_dt;
            each<S>([&](auto s) { carry_of(g, p, p.chunk)[s] = h[s]; });
        } else if (g.final && p.valid && p.t1 == p.len) {
            each<S>([&](auto s) {
                if (has_state(g, p, s)) g.final[state_at(g, p, s)] = h[s];
            });
        }
    }

    // ----------------------------------------------------------- backward

    // LOCAL: a_{t0} g_{t0} of the chunk's own tokens, from nothing after it;
    // else the gradients, from what the tokens after the chunk pass back.
    template <bool LOCAL>
    static __device__ __forceinline__ void backward(const fg_scan_kargs& g) {
        using X = Exchange<4>;
        __shared__ __attribute__((aligned(16))) X xs;
        // sums over the wave's channels: [token of the segment][B, C][state]
        constexpr int NS = 4 * S;
        __shared__ float sums[LOCAL ? 1 : FG_SSM_WAVES][SEG * 2 * NS];
        const Place p = place(g);
        if (LOCAL && (p.chunk == 0 || p.t1 == p.t0)) return;  // no chunk before it, or no tokens
        const Lane l = lane(g, p);
        float* x = xs.v[p.wave] + p.c * X::STRIDE;
        float carry[S], ga[S];
        each<S>([&](auto s) { carry[s] = ga[s] = 0.0f; });
        if constexpr (!LOCAL) {
            each<S>([&](auto s) {
                if (g.gfinal && has_state(g, p, s)) carry[s] = g.gfinal[state_at(g, p, s)];
            });
            const uint32_t used = p.len ? (p.len - 1) / g.chunk_len + 1 : 0;
            for (uint32_t k = used; k-- > p.chunk + 1;) {
                const float sum = g.carry_dt[carry_at(g, p, k) * 16 + p.c];
                each<S>([&](auto s) {
                    carry[s] = fmaf(exp2_(sum * l.a2[s]), carry[s], carry_of(g, p, k)[s]);
                    if (PAD && l.pad[s]) carry[s] = 0.0f;
                });
            }
        }
        float sum_dt = 0.0f, gskip = 0.0f, gbias = 0.0f;
        const uint32_t segs = (p.t1 - p.t0 + SEG - 1) / SEG;
        for (uint32_t k = segs; k-- > 0;) {
            const uint32_t t = p.t0 + k * SEG;
            const uint32_t n = p.t1 - t < SEG ? p.t1 - t : SEG;
            float u[NG], d[NG], dt[NG], slope[NG], dy[NG], b[NG][NB], cc[NG][NB], ds[NG], zs[NG];
            raw rv[NG], rs[NG][NB];
            Cursor cur;
            cur.set(g.delta, p, t);
            load_channels<true>(rv, cur, p, n);
            up_channels(d, rv);
            cur.set(g.gout, p, t);
            load_channels<true>(rv, cur, p, n);
            up_channels(dy, rv);
            cur.set(g.c, p, t, p.group * g.states);
            load_states<true>(rs, cur, l, n);
            up_states(cc, rs, l);
            if constexpr (!LOCAL) {
                cur.set(g.u, p, t);
            load_channels<true>(rv, cur, p, n);
                up_channels(u, rv);
                cur.set(g.b, p, t, p.group * g.states);
                load_states<true>(rs, cur, l, n);
                up_states(b, rs, l);
            }
            each<NG>([&](auto i) { ds[i] = dy[i], zs[i] = 0.0f; });
            if (g.z.p) {
                float z[NG];
                cur.set(g.z, p, t);
            load_channels<true>(rv, cur, p, n);
                up_channels(z, rv);
                each<NG>([&](auto i) {
                    const float sg = sigmoid(z[i]);
                    ds[i] = dy[i] * z[i] * sg;
                    zs[i] = dy[i] * sg * fmaf(z[i], 1.0f - sg, 1.0f);
                });
            }
            steps(g, l, d, dt, slope);
            wave_sync();
            each<NG>([&](auto i) {
                const bool in = 4 * i + p.q < n;
                if constexpr (LOCAL) sum_dt += in ? dt[i] : 0.0f;
                float* to = x + (4 * i + p.q) * 4;
                // a lane without a channel adds nothing to the sums over channels
                to[0] = dt[i];
                to[1] = p.valid ? ds[i] : 0.0f;
                if constexpr (!LOCAL) to[2] = p.valid ? dt[i] * u[i] : 0.0f;
            });
            wave_sync();
            if constexpr (LOCAL) {
                each<NG>([&](auto ri) {
                    constexpr int i = NG - 1 - ri;
                    each<4>([&](auto rj) {
                        constexpr int j = 3 - rj;
                        if (4 * i + j < n) {
                            const float dtj = x[(4 * i + j) * 4], dsj = x[(4 * i + j) * 4 + 1];
                            bcast_fmac<S, j>(carry, cc[i], dsj);
                            each<S>([&](auto s) {
                                carry[s] *= exp2_(dtj * l.a2[s]);
                                if (PAD && l.pad[s]) carry[s] = 0.0f;
                            });
                        }
                    });
                });
            } else {
                float h0[S], a[SEG][S], h[SEG][S];
                const float* from = g.check + check_at(g, p, t);
                each<S>([&](auto s) { h0[s] = from[s]; });
                // the segment's states again
                each<NG>([&](auto i) {
                    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    each<4>([&](auto j) {
                        constexpr int m = 4 * i + j;
                        if (m < n) {
                            const float dtj = x[m * 4], dtu = x[m * 4 + 2];
                            each<S>([&](auto s) {
                                constexpr int I = j * S + s;
                                const float before = m ? h[m ? m - 1 : 0][s] : h0[s];
                                a[m][s] = exp2_(dtj * l.a2[s]);
                                h[m][s] = fmaf(a[m][s], before, row_bcast<I % 16>(b[i][I / 16]) * dtu);
                                if (PAD && l.pad[s]) h[m][s] = 0.0f;
                            });
                            bcast_dot<S, j>(y[j], cc[i], h[m]);
                        }
                    });
                    if (g.gz.p) {
                        const float o = fmaf(l.skip, u[i], rows_sum(y));
                        { cur.set(g.gz, p, t); store_channels<true>(cur, p, i, n, zs[i] * o); }
                    }
                });
                // and back
                each<NG>([&](auto ri) {
                    constexpr int i = NG - 1 - ri;
                    float gb[4 * S], gc[4 * S], gu[4] = {0.0f, 0.0f, 0.0f, 0.0f}, gd[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    each<4 * S>([&](auto e) { gb[e] = gc[e] = 0.0f; });
                    each<4>([&](auto rj) {
                        constexpr int j = 3 - rj, m = 4 * i + j;
                        if (m < n) {
                            const float dtj = x[m * 4], dsj = x[m * 4 + 1], dtu = x[m * 4 + 2];
                            bcast_fmac<S, j>(carry, cc[i], dsj);  // g_t
                            bcast_dot<S, j>(gu[j], b[i], carry);
                            each<S>([&](auto s) {
                                gb[j * S + s] = carry[s] * dtu;
                                gc[j * S + s] = dsj * h[m][s];
                                carry[s] *= a[m][s];
                                if (PAD && l.pad[s]) carry[s] = 0.0f;
                                const float held = carry[s] * (m ? h[m ? m - 1 : 0][s] : h0[s]);
                                gd[j] = fmaf(held, l.a2[s], gd[j]);
                                ga[s] = fmaf(held, dtj, ga[s]);
                            });
                        }
                    });
                    const float gbu = rows_sum(gu), gdd = rows_sum(gd);
                    const bool in = p.valid && 4 * i + p.q < n;
                    const float gdelta = fmaf(u[i], gbu, kLn2 * gdd) * slope[i];
                    if (in) {
                        gbias += gdelta;
                        gskip = fmaf(ds[i], u[i], gskip);
                    }
                    if (g.gdelta.p) { cur.set(g.gdelta, p, t); store_channels<true>(cur, p, i, n, gdelta); }
                    if (g.gu.p) { cur.set(g.gu, p, t); store_channels<true>(cur, p, i, n, fmaf(dt[i], gbu, l.skip * ds[i])); }
                    channels_sum(gb, p.c);
                    channels_sum(gc, p.c);
                    constexpr int R = S >= 4 ? S / 4 : 1;
                    each<R>([&](auto r) {
                        const uint32_t e = S >= 4 ? p.c * R + r : p.c >> (S == 2 ? 1 : 2);
                        const uint32_t m = 4 * i + e / S, s = p.q * S + e % S;
                        if (S >= 4 || (p.c & (S == 2 ? 1 : 3)) == 0) {
                            sums[p.wave][(m * 2) * NS + s] = gb[r];
                            sums[p.wave][(m * 2 + 1) * NS + s] = gc[r];
                        }
                    });
                });
                // B's and C's gradients of the workgroup's channels
                __syncthreads();
                for (uint32_t e = threadIdx.x; e < n * 2 * NS; e += 64 * FG_SSM_WAVES) {
                    float v = 0.0f;
                    each<FG_SSM_WAVES>([&](auto w) { v += sums[w][e]; });
                    const uint32_t s = e % NS, m = e / (2 * NS), which = e / NS % 2;
                    if (s < g.states) {
                        const uint64_t tok = (g.offsets ? (uint64_t)p.start : (uint64_t)p.seq * g.length) + t + m;
                        g.part_bc[((((uint64_t)p.block * g.tokens + tok) * g.groups + p.group) * 2 + which) * g.states +
                                  s] = v;
                    }
                }
                __syncthreads();
            }
        }
        if constexpr (LOCAL) {
            const float v[4] = {sum_dt, sum_dt, sum_dt, sum_dt};
            sum_dt = rows_sum(v);
            if (p.q == 0) g.carry_dt[carry_at(g, p, p.chunk) * 16 + p.c] = sum_dt;
            each<S>([&](auto s) { carry_of(g, p, p.chunk)[s] = carry[s]; });
        } else {
            float vb[4] = {gbias, gbias, gbias, gbias}, vs[4] = {gskip, gskip, gskip, gskip};
            gbias = rows_sum(vb);
            gskip = rows_sum(vs);
            if (p.valid) {
                float* to = g.part_p + ((uint64_t)p.seq * g.chunks + p.chunk) * g.channels * (g.states + 2);
                each<S>([&](auto s) {
                    if (has_state(g, p, s)) to[(uint64_t)p.ch * g.states + p.q * S + s] = ga[s];
                });
                if (p.q == 0) to[(uint64_t)g.channels * g.states + p.ch] = gskip;
                if (p.q == 1) to[(uint64_t)g.channels * (g.states + 1) + p.ch] = gbias;
                if (g.ginitial && p.chunk == 0) {
                    each<S>([&](auto s) {
                        if (has_state(g, p, s)) g.ginitial[state_at(g, p, s)] = carry[s];
                    });
                }
            }
        }
    }
};

// B's and C's gradients from the channel blocks' parts, in the order of the blocks.
template <class T>
__device__ __forceinline__ void scan_reduce_bc(const fg_scan_kargs& g) {
    const uint32_t row = g.groups * 2 * g.states;
    const uint64_t n = g.tokens * row;
    const uint64_t e = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= n) return;
    float v = 0.0f;
    for (uint32_t b = 0; b < g.group_blocks; ++b) v += g.part_bc[b * n + e];
    const uint64_t tok = e / row;
    const uint32_t r = (uint32_t)(e % row), s = r % g.states, which = r / g.states % 2, grp = r / (2 * g.states);
    const uint64_t seq = g.offsets ? 0 : tok / g.length, t = g.offsets ? tok : tok % g.length;
    if (g.offsets) {  // rows outside every sequence have no parts
        uint32_t lo = 0, hi = g.seqs;  // the last sequence that starts at or before the row
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (g.offsets[mid] <= (int64_t)tok) lo = mid;
            else hi = mid;
        }
        const int64_t start = g.offsets[lo];
        if ((int64_t)tok < start || (int64_t)tok >= g.offsets[lo + 1] || (int64_t)tok - start >= g.length) return;
    }
    const fg_ssm_view& w = which ? g.gc : g.gb;
    if (w.p) {
        ((typename T::raw*)w.p)[(int64_t)seq * w.seq + (int64_t)t * w.row + grp * g.states + s] = T::down(v);
    }
}

// The parameters' gradients from the chunks' parts, in the order of the chunks.
__device__ __forceinline__ void scan_reduce_p(const fg_scan_kargs& g) {
    const uint64_t n = (uint64_t)g.channels * (g.states + 2);
    const uint64_t e = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= n) return;
    float v = 0.0f;
    for (uint64_t k = 0; k < (uint64_t)g.seqs * g.chunks; ++k) v += g.part_p[k * n + e];
    const uint64_t states = (uint64_t)g.channels * g.states;
    if (e < states) {
        if (g.ga) g.ga[e] = v;
    } else if (e < states + g.channels) {
        if (g.gskip) g.gskip[e - states] = v;
    } else if (g.gbias) {
        g.gbias[e - states - g.channels] = v;
    }
}

// One token of each row, the states in a cache of slots: a lane takes four
// states of a channel, `lanes` neighbouring lanes (a power of two) a channel.
template <class T>
__device__ __forceinline__ void scan_step_body(const fg_scan_step_kargs& g) {
    using raw = typename T::raw;
    const uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const uint32_t part = (uint32_t)(id % g.lanes);
    const uint64_t of = id / g.lanes;
    const bool valid = of < (uint64_t)g.rows * g.channels;
    const uint32_t row = valid ? (uint32_t)(of / g.channels) : 0, ch = valid ? (uint32_t)(of % g.channels) : 0;
    const int64_t slot = g.slots ? g.slots[row] : (int64_t)row;
    const bool live = valid && slot >= 0 && (uint64_t)slot < g.state_rows;  // a row without a slot: zeros out
    float acc = 0.0f, u = 0.0f;
    if (live) {
        auto in = [&](const fg_ssm_view& v, uint32_t i) { return T::up(((const raw*)v.p)[(int64_t)row * v.seq + i]); };
        u = in(g.u, ch);
        const float x = in(g.delta, ch) + (g.bias ? g.bias[ch] : 0.0f);
        const float dt = g.softplus ? softplus(x).value : x;
        const uint32_t grp = ch / g.group_channels;
        const uint64_t at = ((uint64_t)slot * g.channels + ch) * g.states;
        for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t n = part * 4 + k;
            if (n < g.states) {
                float h = exp2_(dt * (g.a[(uint64_t)ch * g.states + n] * kLog2e)) * g.state[at + n];
                h = fmaf(dt * u, in(g.b, grp * g.states + n), h);
                g.state_out[at + n] = h;
                acc = fmaf(in(g.c, grp * g.states + n), h, acc);
            }
        }
    }
    for (uint32_t m = 1; m < g.lanes; m *= 2) acc += __shfl_xor(acc, m);
    if (valid && part == 0) {
        if (live) {
            if (g.skip) acc = fmaf(g.skip[ch], u, acc);
            if (g.z.p) {
                const float z = T::up(((const raw*)g.z.p)[(int64_t)row * g.z.seq + ch]);
                acc *= z * sigmoid(z);
            }
        } else {
            acc = 0.0f;
        }
        ((raw*)g.out.p)[(int64_t)row * g.out.seq + ch] = T::down(acc);
    }
}

}  // namespace ssm
}  // namespace fg
