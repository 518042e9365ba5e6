// ssm_scan.hpp -- the selective scan over sequences, forward and backward:
//
//   dt = softplus(delta + bias)              h_t[d,n] = exp(dt A[d,n]) h_{t-1}[d,n] + dt u B_t[n]
//   y  = (sum_n C_t[n] h_t[d,n] + D u) silu(z)
//
// A wave takes 16 channels and walks along the tokens in segments of 16.  Its
// lanes have two roles, between which LDS carries values:
//   * per token and channel (time steps, gates, outputs): lane l has token l / 4
//     of the segment and four neighbouring channels, 4 (l % 4) ...; rows are
//     loaded and stored eight bytes a lane of a 16-bit type;
//   * per state: lane (q, c) = (l / 16, l % 16) has the states q S ... q S + S - 1
//     of channel c and steps through the tokens.  B and C of those states lie
//     one token a lane in the row's 16 lanes, and reach the row as the DPP
//     broadcast operand of the instruction that takes them; sums over a
//     channel's states end with an exchange between the wave's four rows.
// Nothing is worked out twice, and waves wait for each other only where the
// backward pass adds up over channels.  The workgroup is four waves, 64
// channels: 128-byte lines of a 16-bit type.
#pragma once

#include "ssm_common.hpp"

namespace fg {
namespace ssm {

// acc[i] += bcast(v[i], lane J of the row) * x[i], and acc += sum_i of it, for
// up to four i in one statement of assembly: the compiler does not fold the
// broadcast into a multiply-add.  The s_nop keeps the two wait states that a
// DPP operand needs after the instruction that wrote it.
#define FG_BC "row_newbcast:%"
template <int J>
__device__ __forceinline__ void fmac1(float& a, float v, float x) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %2 " FG_BC "3 row_mask:0xf bank_mask:0xf" : "+v"(a) : "v"(v), "v"(x), "n"(J));
}
template <int J>
__device__ __forceinline__ void fmac2(float& a0, float& a1, float v0, float v1, float x) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %2, %4 " FG_BC "5 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %3, %4 " FG_BC "5 row_mask:0xf bank_mask:0xf"
        : "+&v"(a0), "+&v"(a1)
        : "v"(v0), "v"(v1), "v"(x), "n"(J));
}
template <int J>
__device__ __forceinline__ void fmac4(float& a0, float& a1, float& a2, float& a3, float v0, float v1, float v2,
                                      float v3, float x) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %4, %8 " FG_BC "9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %5, %8 " FG_BC "9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %6, %8 " FG_BC "9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %3, %7, %8 " FG_BC "9 row_mask:0xf bank_mask:0xf"
        : "+&v"(a0), "+&v"(a1), "+&v"(a2), "+&v"(a3)
        : "v"(v0), "v"(v1), "v"(v2), "v"(v3), "v"(x), "n"(J));
}
template <int J>
__device__ __forceinline__ void dot2(float& a, float v0, float v1, float x0, float x1) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %3 " FG_BC "5 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %4 " FG_BC "5 row_mask:0xf bank_mask:0xf"
        : "+&v"(a)
        : "v"(v0), "v"(v1), "v"(x0), "v"(x1), "n"(J));
}
template <int J>
__device__ __forceinline__ void dot4(float& a, float v0, float v1, float v2, float v3, float x0, float x1, float x2,
                                     float x3) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %5 " FG_BC "9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %6 " FG_BC "9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %3, %7 " FG_BC "9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %4, %8 " FG_BC "9 row_mask:0xf bank_mask:0xf"
        : "+&v"(a)
        : "v"(v0), "v"(v1), "v"(v2), "v"(v3), "v"(x0), "v"(x1), "v"(x2), "v"(x3), "n"(J));
}
#undef FG_BC

// acc[s] += (token J's v[s]) * x, s < N.
template <int N, int J>
__device__ __forceinline__ void bcast_fmac(float* acc, const float* v, float x) {
    if constexpr (N == 1) fmac1<J>(acc[0], v[0], x);
    else if constexpr (N == 2) fmac2<J>(acc[0], acc[1], v[0], v[1], x);
    else
        each<N / 4>([&](auto k) {
            constexpr int i = 4 * k;
            fmac4<J>(acc[i], acc[i + 1], acc[i + 2], acc[i + 3], v[i], v[i + 1], v[i + 2], v[i + 3], x);
        });
}
// acc += sum_s (token J's v[s]) * x[s].
template <int N, int J>
__device__ __forceinline__ void bcast_dot(float& acc, const float* v, const float* x) {
    if constexpr (N == 1) fmac1<J>(acc, v[0], x[0]);
    else if constexpr (N == 2) dot2<J>(acc, v[0], v[1], x[0], x[1]);
    else
        each<N / 4>([&](auto k) {
            constexpr int i = 4 * k;
            dot4<J>(acc, v[i], v[i + 1], v[i + 2], v[i + 3], x[i], x[i + 1], x[i + 2], x[i + 3]);
        });
}

// The sum over a row's 16 channels of each of v[0 .. 4 N), N <= 4: halving the
// values with every bit of the lane number, so that lane c ends with the sum
// of value c (N = 4), c >> 1 (2) or c >> 2 (1) in v[0].
template <int N>
__device__ __forceinline__ void channels_sum(float (&v)[4 * N], uint32_t c) {
    const bool b3 = c & 8, b2 = c & 4, b1 = c & 2, b0 = c & 1;
    auto level = [&](auto half, bool upper, auto ctrl) {
        each<half>([&](auto i) {
            const float low = v[i], high = v[i + half];
            v[i] = (upper ? high : low) + dpp<ctrl>(upper ? low : high);
        });
    };
    level(Int<2 * N>{}, b3, Int<kRor8>{});
    level(Int<N>{}, b2, Int<kHalfMirror>{});
    if constexpr (N >= 2) level(Int<N / 2>{}, b1, Int<kXor2>{});
    else v[0] += dpp<kXor2>(v[0]);
    if constexpr (N >= 4) level(Int<1>{}, b0, Int<kXor1>{});
    else v[0] += dpp<kXor1>(v[0]);
}

// Where a wave works: its sequence, the tokens of its chunk, its channels.
struct Place {
    int64_t start;               // packed: the sequence's first row
    uint32_t len;                // tokens of the sequence
    uint32_t seq, chunk, group, block;
    uint32_t t0, t1;             // the chunk's tokens
    uint32_t wave, wblock;       // its number in the workgroup, and among all waves over channels
    // as (q, c): the channel, within the group and among all (the group's last where it has none)
    uint32_t q, c, ch;
    bool valid;
    // as (token, four channels): the first channel, how many of the four there are
    uint32_t tok, ch4;
    int have;
};

__device__ __forceinline__ Place place(const fg_scan_kargs& g) {
    Place p;
    const uint32_t lane = threadIdx.x & 63;
    p.wave = uniform(threadIdx.x >> 6);
    p.q = lane >> 4;
    p.c = lane & 15;
    p.tok = lane >> 2;
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
    const uint32_t base = p.block * FG_SSM_GROUP_CHANNELS + p.wave * FG_SSM_WAVE_CHANNELS;
    const uint32_t one = base + p.c, four = base + 4 * (lane & 3);
    p.valid = one < g.group_channels;
    p.ch = p.group * g.group_channels + (p.valid ? one : g.group_channels - 1);
    p.have = four >= g.group_channels ? 0 : g.group_channels - four < 4 ? (int)(g.group_channels - four) : 4;
    p.ch4 = four;
    p.wblock = cb * FG_SSM_WAVES + p.wave;
    return p;
}

template <class T, int S, bool PAD>
struct Scan {
    using raw = typename T::raw;
    static constexpr int SEG = FG_SSM_SEGMENT;
    static constexpr int ES = sizeof(raw);
    static constexpr int SP = S < 4 ? S : 4, PASSES = S / SP;  // states of a lane at a time (backward)

    // N elements as they lie in memory, in whole registers: 16-bit ones two to
    // a register, so that a wide load needs no work that would wait for it.
    template <int N>
    struct Pack {
        static constexpr int WORDS = (N * ES + 3) / 4;
        uint32_t w[WORDS];
        __device__ __forceinline__ float up(int i) const {
            if constexpr (ES == 4) return __uint_as_float(w[i]);
            else return T::up((raw)(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffff));
        }
        __device__ __forceinline__ void load(const char* at) {
            if constexpr (N * ES >= 4) {
                struct __attribute__((aligned(N * ES > 16 ? 16 : N * ES))) Words {
                    uint32_t w[WORDS];
                };
                const Words x = *(const Words*)at;
                each<WORDS>([&](auto i) { w[i] = x.w[i]; });
            } else {
                w[0] = *(const raw*)at;
            }
        }
        __device__ __forceinline__ void fill(const raw (&x)[N]) {
            if constexpr (ES == 4) each<N>([&](auto i) { w[i] = __builtin_bit_cast(uint32_t, x[i]); });
            else
                each<WORDS>([&](auto i) {
                    w[i] = (uint16_t)__builtin_bit_cast(uint16_t, (uint16_t)x[2 * i]);
                    if constexpr (2 * i + 1 < N) w[i] |= (uint32_t)x[2 * i + 1] << 16;
                });
        }
    };
    using Raw4 = Pack<4>;
    using RawS = Pack<S>;

    // The lane's constants.
    struct Lane {
        bool pad[S];
        float a2[S];               // A log2(e)
        float bias[4], skip[4];
        uint32_t off4[4];          // the four channels' offsets in a row, bytes
        uint32_t offs[S];          // the states' offsets in a row of B and C, bytes
    };
    static __device__ __forceinline__ Lane lane(const fg_scan_kargs& g, const Place& p) {
        Lane l;
        each<S>([&](auto s) {
            const uint32_t n = p.q * S + s, m = n < g.states ? n : g.states - 1;
            l.pad[s] = PAD && n >= g.states;
            l.a2[s] = n < g.states ? g.a[(uint64_t)p.ch * g.states + n] * kLog2e : 0.0f;
            l.offs[s] = (p.group * g.states + m) * ES;
        });
        each<4>([&](auto i) {
            // a channel that is not there: the group's last one (wide loads: its last four)
            uint32_t c = p.ch4 + i;
            if (c >= g.group_channels) c = p.have > 0 || !g.wide ? g.group_channels - 1 : g.group_channels - 4 + i;
            c += p.group * g.group_channels;
            l.off4[i] = c * ES;
            l.bias[i] = g.bias ? g.bias[c] : 0.0f;
            l.skip[i] = g.skip ? g.skip[c] : 0.0f;
        });
        return l;
    }

    // A view's rows of a segment: the uniform address of its first row, moved
    // from segment to segment.
    struct Cursor {
        const char* at;
        uint32_t row;  // bytes
        __device__ __forceinline__ void set(const fg_ssm_view& v, const Place& p, uint32_t t) {
            at = (const char*)v.p + ((int64_t)p.seq * v.seq + (p.start + t) * v.row) * ES;
            row = (uint32_t)v.row * ES;
        }
        __device__ __forceinline__ void move(int32_t segments) { at += (int64_t)segments * SEG * row; }
    };
    // The lane's row of n (beyond the last: the last).
    template <bool TAIL>
    static __device__ __forceinline__ uint32_t row_of(uint32_t r, uint32_t n) {
        return TAIL && r >= n ? n - 1 : r;
    }
    template <bool TAIL>
    static __device__ __forceinline__ void load4(Raw4& v, const Cursor& w, const Place& p, const Lane& l, bool wide,
                                                 uint32_t n) {
        const uint32_t r = row_of<TAIL>(p.tok, n) * w.row;
        if (wide) {
            v.load(w.at + fresh(r + l.off4[0]));
        } else {
            raw x[4];
            each<4>([&](auto i) { x[i] = *(const raw*)(w.at + fresh(r + l.off4[i])); });
            v.fill(x);
        }
    }
    template <bool TAIL>
    static __device__ __forceinline__ void store4(const Cursor& w, const Place& p, const Lane& l, bool wide, uint32_t n,
                                                  const float (&x)[4]) {
        if (TAIL && p.tok >= n) return;
        const uint32_t r = p.tok * w.row;
        char* to = const_cast<char*>(w.at);
        if (wide) {
            struct __attribute__((aligned(4 * ES))) Out {
                raw v[4];
            } v;
            each<4>([&](auto i) { v.v[i] = T::down(x[i]); });
            if (p.have > 0) *(Out*)(to + fresh(r + l.off4[0])) = v;
        } else {
            each<4>([&](auto i) {
                if (i < p.have) *(raw*)(to + fresh(r + l.off4[i])) = T::down(x[i]);
            });
        }
    }
    // B's or C's rows: lane (q, c) has token c's states of row q.
    template <bool TAIL>
    static __device__ __forceinline__ void load_states(RawS& v, const Cursor& w, const Place& p, const Lane& l,
                                                       bool wide, uint32_t n) {
        const uint32_t r = row_of<TAIL>(p.c, n) * w.row;
        if (wide) {
            v.load(w.at + fresh(r + l.offs[0]));
        } else {
            raw x[S];
            each<S>([&](auto s) { x[s] = *(const raw*)(w.at + fresh(r + l.offs[s])); });
            v.fill(x);
        }
    }
    static __device__ __forceinline__ void up4(float (&x)[4], const Raw4& v) {
        each<4>([&](auto i) { x[i] = v.up(i); });
    }
    static __device__ __forceinline__ void up_states(float (&x)[S], const RawS& v, const Lane& l) {
        each<S>([&](auto s) { x[s] = PAD && l.pad[s] ? 0.0f : v.up(s); });
    }

    // States at the start of the segment at token t: place of the wave's 64 S.
    static __device__ __forceinline__ float* check_of(const fg_scan_kargs& g, const Place& p, uint32_t t) {
        const uint64_t seg = g.offsets ? (uint64_t)p.start / SEG + p.seq : (uint64_t)p.seq * g.check_segs;
        return g.check + ((seg + t / SEG) * (g.groups * g.group_blocks * FG_SSM_WAVES) + p.wblock) * (64 * S) +
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
        return !PAD || p.q * S + s < g.states;
    }
    // Orders the wave's own LDS accesses.
    static __device__ __forceinline__ void wave_sync() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // Sum over the segment's tokens of what lane (token, four channels) holds; all lanes get it.
    static __device__ __forceinline__ float tokens_sum(float v) {
        for (int m = 4; m < 64; m *= 2) v += __shfl_xor(v, m);
        return v;
    }

    // No branch on softplus: the segment stays one block, which the compiler interleaves.
    static __device__ __forceinline__ Softplus time_step(const fg_scan_kargs& g, float x) {
        const Softplus s = softplus(x);
        return {g.softplus ? s.value : x, g.softplus ? s.slope : 1.0f};
    }

    // ------------------------------------------------------------ forward

    // LDS of a wave: per channel the tokens' (dt, dt u), twice (a segment is
    // made ready while the one before it is worked through); the outputs.
    static constexpr int XSTRIDE = 2 * SEG + 4;  // keeps the 16 channels on banks of their own
    struct ForwardLds {
        float x[2][16 * XSTRIDE];
        float y[SEG * 16];
    };

    // A segment's time steps, to LDS.
    template <bool LOCAL, bool TAIL>
    static __device__ __forceinline__ void prepare(const fg_scan_kargs& g, const Place& p, const Lane& l, float* x,
                                                   float (&sum_dt)[4], const float (&d)[4], const float (&u)[4],
                                                   uint32_t n, bool count) {
        each<4>([&](auto i) {
            const float dt = time_step(g, d[i] + l.bias[i]).value;
            const float2 e = {dt, dt * u[i]};
            *(float2*)(x + (4 * (threadIdx.x & 3) + i) * XSTRIDE + 2 * p.tok) = e;
            if constexpr (LOCAL) sum_dt[i] += count && (!TAIL || p.tok < n) ? dt : 0.0f;
        });
    }
    template <bool LOCAL, bool TAIL>
    static __device__ __forceinline__ void forward_segment(const Place& p, const Lane& l, const float* x, float* y,
                                                           float (&h)[S], const float (&b)[S], const float (&c)[S],
                                                           uint32_t n) {
        x += p.c * XSTRIDE;
        each<SEG / 4>([&](auto i) {
            float e[8], ys[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            *(float4*)e = *(const float4*)(x + 8 * i);
            *(float4*)(e + 4) = *(const float4*)(x + 8 * i + 4);
            each<4>([&](auto j) {
                if (!TAIL || 4 * i + j < n) {
                    each<S>([&](auto s) {
                        h[s] = fmaf(exp2_(e[2 * j] * l.a2[s]), h[s], row_bcast<4 * i + j>(b[s]) * e[2 * j + 1]);
                        if (PAD && l.pad[s]) h[s] = 0.0f;
                    });
                    if constexpr (!LOCAL) bcast_dot<S, 4 * i + j>(ys[j], c, h);
                }
            });
            if constexpr (!LOCAL) y[(4 * i + p.q) * 16 + p.c] = rows_sum(ys);
        });
    }
    template <bool TAIL>
    static __device__ __forceinline__ void outputs(const fg_scan_kargs& g, const Place& p, const Lane& l,
                                                   const float* y, const Cursor& out, const Raw4& ru, const Raw4& rz,
                                                   bool gated, uint32_t n) {
        float u[4], z[4], o[4];
        up4(u, ru);
        up4(z, rz);
        const float4 v = *(const float4*)(y + p.tok * 16 + 4 * (threadIdx.x & 3));
        const float ys[4] = {v.x, v.y, v.z, v.w};
        each<4>([&](auto i) {
            const float gate = z[i] * sigmoid(z[i]);
            o[i] = fmaf(l.skip[i], u[i], ys[i]) * (gated ? gate : 1.0f);
        });
        store4<TAIL>(out, p, l, g.wide, n, o);
    }

    // LOCAL: the states that the chunk's own tokens leave, from none, and the
    // sum of its time steps; else outputs, from the states before the chunk.
    template <bool LOCAL>
    static __device__ __forceinline__ void forward(const fg_scan_kargs& g) {
        __shared__ __attribute__((aligned(16))) ForwardLds lds[FG_SSM_WAVES];
        const Place p = place(g);
        if (LOCAL && p.chunk == 0) {
            // the last chunks may write the final states where the initial ones lie
            each<S>([&](auto s) {
                const bool has = g.initial && has_state(g, p, s);
                carry_of(g, p, g.chunks)[s] = has ? g.initial[state_at(g, p, s)] : 0.0f;
            });
        }
        if (LOCAL && p.t1 == p.len) return;                 // no chunk follows
        if (!LOCAL && p.chunk > 0 && p.t0 == p.t1) return;  // no tokens
        const Lane l = lane(g, p);
        float(&x)[2][16 * XSTRIDE] = lds[p.wave].x;
        float* y = lds[p.wave].y;
        float h[S], sum_dt[4] = {0.0f, 0.0f, 0.0f, 0.0f};
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
        // Without a gate u's rows stand in for z's, which are then not used.
        const bool gated = g.z.p != nullptr;
        Cursor cu, cd, cz, cu2, cb, cc, co;
        cu.set(g.u, p, p.t0);
        cd.set(g.delta, p, p.t0);
        cb.set(g.b, p, p.t0);
        if constexpr (!LOCAL) {
            cc.set(g.c, p, p.t0);
            cz.set(gated ? g.z : g.u, p, p.t0);
            cu2.set(g.u, p, p.t0);
            co.set(g.out, p, p.t0);
        }
        Raw4 rd, ru, rz, ru2;
        RawS rb, rc;
        float d[4], u[4], b[S], c[S];
        auto checkpoint = [&](uint32_t t) {
            if constexpr (!LOCAL) {
                if (g.check) {  // lanes without a channel too: the backward pass reads them
                    float* to = check_of(g, p, t);
                    each<S>([&](auto s) { to[s] = h[s]; });
                }
            }
        };
        const uint32_t full = (p.t1 - p.t0) / SEG, rest = (p.t1 - p.t0) % SEG;
        if (full > 0) {
            // While segment k is worked through, k + 1 is made ready, the rows
            // of k + 2 are loaded (at the end some once more, to no use), and
            // the outputs of k - 1 are stored.
            load4<false>(rd, cd, p, l, g.wide, SEG);
            load4<false>(ru, cu, p, l, g.wide, SEG);
            load_states<false>(rb, cb, p, l, g.wide, SEG);
            if constexpr (!LOCAL) load_states<false>(rc, cc, p, l, g.wide, SEG);
            up4(d, rd);
            up4(u, ru);
            cd.move(full > 1);
            cu.move(full > 1);
            load4<false>(rd, cd, p, l, g.wide, SEG);
            load4<false>(ru, cu, p, l, g.wide, SEG);
            prepare<LOCAL, false>(g, p, l, x[0], sum_dt, d, u, SEG, true);
            for (uint32_t k = 0; k < full; ++k) {
                up_states(b, rb, l);
                up4(d, rd);
                up4(u, ru);
                cd.move(k + 2 < full);
                cu.move(k + 2 < full);
                cb.move(k + 1 < full);
                if constexpr (!LOCAL) {
                    up_states(c, rc, l);
                    cc.move(k + 1 < full);
                    if (k > 0) {
                        outputs<false>(g, p, l, y, co, ru2, rz, gated, SEG);
                        co.move(1);
                    }
                }
                // one branch around all: loads of several branches would wait for each other
                auto loads = [&](bool wide) {
                    load4<false>(rd, cd, p, l, wide, SEG);
                    load4<false>(ru, cu, p, l, wide, SEG);
                    load_states<false>(rb, cb, p, l, wide, SEG);
                    if constexpr (!LOCAL) {
                        load_states<false>(rc, cc, p, l, wide, SEG);
                        load4<false>(rz, cz, p, l, wide, SEG);
                        load4<false>(ru2, cu2, p, l, wide, SEG);
                    }
                };
                if (g.wide) loads(true);
                else loads(false);
                if constexpr (!LOCAL) {
                    cz.move(1);
                    cu2.move(1);
                }
                checkpoint(p.t0 + k * SEG);
                wave_sync();
                prepare<LOCAL, false>(g, p, l, x[(k + 1) & 1], sum_dt, d, u, SEG, k + 1 < full);
                forward_segment<LOCAL, false>(p, l, x[k & 1], y, h, b, c, SEG);
                wave_sync();
            }
            if constexpr (!LOCAL) {
                outputs<false>(g, p, l, y, co, ru2, rz, gated, SEG);
                co.move(1);
                cc.move(1);
            }
            cd.move(1);
            cu.move(1);
            cb.move(1);
            wave_sync();
        }
        if (rest > 0) {
            checkpoint(p.t0 + full * SEG);
            load4<true>(rd, cd, p, l, g.wide, rest);
            load4<true>(ru, cu, p, l, g.wide, rest);
            load_states<true>(rb, cb, p, l, g.wide, rest);
            if constexpr (!LOCAL) {
                load_states<true>(rc, cc, p, l, g.wide, rest);
                load4<true>(rz, cz, p, l, g.wide, rest);
                up_states(c, rc, l);
            }
            up4(d, rd);
            up4(u, ru);
            up_states(b, rb, l);
            prepare<LOCAL, true>(g, p, l, x[0], sum_dt, d, u, rest, true);
            wave_sync();
            forward_segment<LOCAL, true>(p, l, x[0], y, h, b, c, rest);
            wave_sync();
            if constexpr (!LOCAL) outputs<true>(g, p, l, y, co, ru, rz, gated, rest);
        }
        if constexpr (LOCAL) {
            each<4>([&](auto i) {
                const float sum = tokens_sum(sum_dt[i]);
                if (p.tok == 0) g.carry_dt[carry_at(g, p, p.chunk) * 16 + 4 * (threadIdx.x & 3) + i] = sum;
            });
            each<S>([&](auto s) { carry_of(g, p, p.chunk)[s] = h[s]; });
        } else if (g.final && p.valid && p.t1 == p.len) {
            each<S>([&](auto s) {
                if (has_state(g, p, s)) g.final[state_at(g, p, s)] = h[s];
            });
        }
    }

    // ----------------------------------------------------------- backward

    // LDS of a wave: per channel the tokens' time steps dt, gradients ds of the
    // ungated outputs, and inputs dt u; per token and channel the sums over
    // states (y, g B, g a h A); B's and C's gradients summed over the channels.
    static constexpr int TSTRIDE = SEG + 4;
    struct BackwardLds {
        float dt[16 * TSTRIDE], ds[16 * TSTRIDE], dtu[16 * TSTRIDE];
        float res[3][SEG * 16];
        float4 keep[5][64];  // u, dt, its slope, ds, z's factor of each lane (token, four channels)
        float sums[SEG * 2 * 4 * S];
    };
    struct LocalLds {
        float dt[16 * TSTRIDE], ds[16 * TSTRIDE];
    };

    template <bool LOCAL>
    struct BackRaws {
        Raw4 u, d, dy, z;
        RawS b, c;
        float h0[S];
    };
    template <bool LOCAL>
    struct BackCursors {
        Cursor u, d, dy, z, b, c;
    };
    template <bool LOCAL, bool TAIL>
    static __device__ __forceinline__ void back_load(BackRaws<LOCAL>& r, const BackCursors<LOCAL>& at,
                                                     const fg_scan_kargs& g, const Place& p, const Lane& l, uint32_t t,
                                                     uint32_t n) {
        auto loads = [&](bool wide) {
            load4<TAIL>(r.d, at.d, p, l, wide, n);
            load4<TAIL>(r.dy, at.dy, p, l, wide, n);
            load4<TAIL>(r.z, at.z, p, l, wide, n);
            load_states<TAIL>(r.c, at.c, p, l, wide, n);
            if constexpr (!LOCAL) {
                load4<TAIL>(r.u, at.u, p, l, wide, n);
                load_states<TAIL>(r.b, at.b, p, l, wide, n);
            }
        };
        if (g.wide) loads(true);
        else loads(false);
        if constexpr (!LOCAL) {
            const float* from = check_of(g, p, t);
            each<S>([&](auto s) { r.h0[s] = from[s]; });
        }
    }
    // Time steps and output gradients, to LDS, with what the end of the segment needs.
    template <bool LOCAL, class L>
    static __device__ __forceinline__ void back_prepare(const BackRaws<LOCAL>& r, const fg_scan_kargs& g,
                                                        const Place& p, const Lane& l, L& lds, float (&dt)[4],
                                                        bool gated) {
        float d[4], dy[4], z[4], u[4], slope[4], ds[4], zs[4];
        up4(d, r.d);
        up4(dy, r.dy);
        up4(z, r.z);
        if constexpr (!LOCAL) up4(u, r.u);
        each<4>([&](auto i) {
            const Softplus s = time_step(g, d[i] + l.bias[i]);
            dt[i] = s.value;
            slope[i] = s.slope;
            const float sg = sigmoid(z[i]);
            ds[i] = gated ? dy[i] * (z[i] * sg) : dy[i];
            zs[i] = dy[i] * (sg * fmaf(z[i], 1.0f - sg, 1.0f));
            // a channel that is not there adds nothing to the sums over channels
            const bool here = i < p.have;
            const uint32_t at = (4 * (threadIdx.x & 3) + i) * TSTRIDE + p.tok;
            lds.dt[at] = dt[i];
            lds.ds[at] = here ? ds[i] : 0.0f;
            if constexpr (!LOCAL) lds.dtu[at] = here ? dt[i] * u[i] : 0.0f;
        });
        if constexpr (!LOCAL) {
            const uint32_t lane = threadIdx.x & 63;
            lds.keep[0][lane] = {u[0], u[1], u[2], u[3]};
            lds.keep[1][lane] = {dt[0], dt[1], dt[2], dt[3]};
            lds.keep[2][lane] = {slope[0], slope[1], slope[2], slope[3]};
            lds.keep[3][lane] = {ds[0], ds[1], ds[2], ds[3]};
            lds.keep[4][lane] = {zs[0], zs[1], zs[2], zs[3]};
        }
    }
    template <bool TAIL>
    static __device__ __forceinline__ void back_local(const Place& p, const Lane& l, const LocalLds& lds,
                                                      float (&carry)[S], const float (&c)[S], uint32_t n) {
        each<SEG / 4>([&](auto ri) {
            constexpr int i = SEG / 4 - 1 - ri;
            float dt[4], ds[4];
            *(float4*)dt = *(const float4*)(lds.dt + p.c * TSTRIDE + 4 * i);
            *(float4*)ds = *(const float4*)(lds.ds + p.c * TSTRIDE + 4 * i);
            each<4>([&](auto rj) {
                constexpr int j = 3 - rj;
                if (!TAIL || 4 * i + j < n) {
                    bcast_fmac<S, 4 * i + j>(carry, c, ds[j]);
                    each<S>([&](auto s) {
                        carry[s] *= exp2_(dt[j] * l.a2[s]);
                        if (PAD && l.pad[s]) carry[s] = 0.0f;
                    });
                }
            });
        });
    }
    // The gradients of one segment's tokens, SP states of the lane at a time.
    // `midway` runs where half of the states are no longer needed: it loads
    // the next segment's rows.
    template <bool TAIL, class F>
    static __device__ __forceinline__ void back_segment(const Place& p, const Lane& l, BackwardLds& lds,
                                                        float (&carry)[S], float (&ga)[S], const float (&b)[S],
                                                        const float (&c)[S], const float (&h0)[S], uint32_t n,
                                                        F&& midway) {
        each<PASSES>([&](auto pass) {
            constexpr int P = pass * SP;
            float a[SEG][SP], h[SEG][SP];
            auto result = [&](int which, int i, float v) {
                float* to = lds.res[which] + (4 * i + p.q) * 16 + p.c;
                *to = P ? *to + v : v;
            };
            // the segment's states again
            each<SEG / 4>([&](auto i) {
                float dt[4], dtu[4], y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                *(float4*)dt = *(const float4*)(lds.dt + p.c * TSTRIDE + 4 * i);
                *(float4*)dtu = *(const float4*)(lds.dtu + p.c * TSTRIDE + 4 * i);
                each<4>([&](auto j) {
                    constexpr int m = 4 * i + j;
                    if (!TAIL || m < n) {
                        each<SP>([&](auto s) {
                            const float before = m ? h[m ? m - 1 : 0][s] : h0[P + s];
                            a[m][s] = exp2_(dt[j] * l.a2[P + s]);
                            h[m][s] = fmaf(a[m][s], before, row_bcast<m>(b[P + s]) * dtu[j]);
                            if (PAD && l.pad[P + s]) h[m][s] = 0.0f;
                        });
                        bcast_dot<SP, m>(y[j], c + P, h[m]);
                    }
                });
                result(0, i, rows_sum(y));
            });
            // and back
            each<SEG / 4>([&](auto ri) {
                constexpr int i = SEG / 4 - 1 - ri;
                if constexpr (pass == PASSES - 1 && ri == SEG / 8) midway();
                float dt[4], ds[4], dtu[4];
                *(float4*)dt = *(const float4*)(lds.dt + p.c * TSTRIDE + 4 * i);
                *(float4*)ds = *(const float4*)(lds.ds + p.c * TSTRIDE + 4 * i);
                *(float4*)dtu = *(const float4*)(lds.dtu + p.c * TSTRIDE + 4 * i);
                float gb[4 * SP], gc[4 * SP], gu[4] = {0.0f, 0.0f, 0.0f, 0.0f}, gd[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (TAIL) each<4 * SP>([&](auto e) { gb[e] = gc[e] = 0.0f; });
                each<4>([&](auto rj) {
                    constexpr int j = 3 - rj, m = 4 * i + j;
                    if (!TAIL || m < n) {
                        bcast_fmac<SP, m>(carry + P, c + P, ds[j]);  // g_t
                        bcast_dot<SP, m>(gu[j], b + P, carry + P);
                        each<SP>([&](auto s) {
                            gb[j * SP + s] = carry[P + s] * dtu[j];
                            gc[j * SP + s] = ds[j] * h[m][s];
                            carry[P + s] *= a[m][s];
                            if (PAD && l.pad[P + s]) carry[P + s] = 0.0f;
                            const float held = carry[P + s] * (m ? h[m ? m - 1 : 0][s] : h0[P + s]);
                            gd[j] = fmaf(held, l.a2[P + s], gd[j]);
                            ga[P + s] = fmaf(held, dt[j], ga[P + s]);
                        });
                    }
                });
                result(1, i, rows_sum(gu));
                result(2, i, rows_sum(gd));
                channels_sum<SP>(gb, p.c);
                channels_sum<SP>(gc, p.c);
                const uint32_t e = SP == 4 ? p.c : p.c >> (SP == 2 ? 1 : 2);
                float* to = lds.sums + ((4 * i + e / SP) * 2) * (4 * S) + p.q * S + P + e % SP;
                if (SP == 4 || (p.c & (SP == 2 ? 1 : 3)) == 0) {
                    to[0] = gb[0];
                    to[4 * S] = gc[0];
                }
            });
        });
    }

    // LOCAL: a_{t0} g_{t0} of the chunk's own tokens, from nothing after it;
    // else the gradients, from what the tokens after the chunk pass back.
    template <bool LOCAL>
    static __device__ __forceinline__ void backward(const fg_scan_kargs& g) {
        using Lds = std::conditional_t<LOCAL, LocalLds, BackwardLds>;
        __shared__ __attribute__((aligned(16))) Lds all[FG_SSM_WAVES];
        const Place p = place(g);
        if (LOCAL && (p.chunk == 0 || p.t1 == p.t0)) return;  // no chunk before it, or no tokens
        const Lane l = lane(g, p);
        Lds& lds = all[p.wave];
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
        const bool gated = g.z.p != nullptr;
        float sum_dt[4] = {0.0f, 0.0f, 0.0f, 0.0f}, gskip[4] = {0.0f, 0.0f, 0.0f, 0.0f},
              gbias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const uint32_t full = (p.t1 - p.t0) / SEG, rest = (p.t1 - p.t0) % SEG;
        BackCursors<LOCAL> at;
        Cursor cgu, cgd, cgz;
        const uint32_t last = p.t0 + full * SEG;  // the rest's first token
        at.d.set(g.delta, p, last);
        at.dy.set(g.gout, p, last);
        at.z.set(gated ? g.z : g.gout, p, last);
        at.c.set(g.c, p, last);
        if constexpr (!LOCAL) {
            at.u.set(g.u, p, last);
            at.b.set(g.b, p, last);
            cgu.set(g.gu, p, last);
            cgd.set(g.gdelta, p, last);
            cgz.set(g.gz, p, last);
        }
        auto move = [&](int by) {
            at.d.move(by);
            at.dy.move(by);
            at.z.move(by);
            at.c.move(by);
            if constexpr (!LOCAL) {
                at.u.move(by);
                at.b.move(by);
            }
        };
        BackRaws<LOCAL> r;
        auto segment = [&](auto tail, uint32_t t, uint32_t n, bool more) {
            constexpr bool TAIL = decltype(tail)::value;
            float b[S], c[S], h0[S], dt[4];
            back_prepare<LOCAL>(r, g, p, l, lds, dt, gated);
            up_states(c, r.c, l);
            if constexpr (!LOCAL) {
                up_states(b, r.b, l);
                each<S>([&](auto s) { h0[s] = r.h0[s]; });
            }
            auto midway = [&] {
                if (more) {  // the segment before this one
                    move(-1);
                    back_load<LOCAL, false>(r, at, g, p, l, t - SEG, SEG);
                }
            };
            wave_sync();
            if constexpr (LOCAL) {
                midway();
                each<4>([&](auto i) { sum_dt[i] += !TAIL || p.tok < n ? dt[i] : 0.0f; });
                back_local<TAIL>(p, l, lds, carry, c, n);
                wave_sync();
            } else {
                back_segment<TAIL>(p, l, lds, carry, ga, b, c, h0, n, midway);
                wave_sync();
                const uint32_t lane = threadIdx.x & 63;
                const float* from = lds.res[0] + p.tok * 16 + 4 * (threadIdx.x & 3);
                float y[4], gu[4], gd[4], o[4], u[4], ds[4], v[4];
                *(float4*)u = lds.keep[0][lane];
                *(float4*)ds = lds.keep[3][lane];
                *(float4*)gu = *(const float4*)(from + SEG * 16);
                if (g.gz.p) {
                    *(float4*)y = *(const float4*)from;
                    *(float4*)v = lds.keep[4][lane];
                    each<4>([&](auto i) { o[i] = v[i] * fmaf(l.skip[i], u[i], y[i]); });
                    store4<TAIL>(cgz, p, l, g.wide, n, o);
                    cgz.move(-1);
                }
                if (g.gu.p) {
                    *(float4*)v = lds.keep[1][lane];
                    each<4>([&](auto i) { o[i] = fmaf(v[i], gu[i], l.skip[i] * ds[i]); });
                    store4<TAIL>(cgu, p, l, g.wide, n, o);
                    cgu.move(-1);
                }
                *(float4*)gd = *(const float4*)(from + 2 * SEG * 16);
                *(float4*)v = lds.keep[2][lane];
                each<4>([&](auto i) {
                    o[i] = fmaf(u[i], gu[i], kLn2 * gd[i]) * v[i];
                    const bool in = !TAIL || p.tok < n;
                    gbias[i] += in ? o[i] : 0.0f;
                    gskip[i] += in ? ds[i] * u[i] : 0.0f;
                });
                if (g.gdelta.p) {
                    store4<TAIL>(cgd, p, l, g.wide, n, o);
                    cgd.move(-1);
                }
                // B's and C's gradients of the workgroup's channels
                __syncthreads();
                constexpr int NS = 4 * S;
                for (uint32_t e = threadIdx.x; e < n * 2 * NS; e += 64 * FG_SSM_WAVES) {
                    float sum = 0.0f;
                    each<FG_SSM_WAVES>([&](auto w) { sum += all[w].sums[e]; });
                    const uint32_t s = e % NS, m = e / (2 * NS), which = e / NS % 2;
                    if (!PAD || s < g.states) {
                        const uint64_t tok = (g.offsets ? (uint64_t)p.start : (uint64_t)p.seq * g.length) + t + m;
                        g.part_bc[((((uint64_t)p.block * g.tokens + tok) * g.groups + p.group) * 2 + which) * g.states +
                                  s] = sum;
                    }
                }
                __syncthreads();
            }
        };
        if (rest > 0) {
            back_load<LOCAL, true>(r, at, g, p, l, last, rest);
            segment(std::true_type{}, last, rest, full > 0);
        } else if (full > 0) {
            move(-1);
            cgu.move(-1);
            cgd.move(-1);
            cgz.move(-1);
            back_load<LOCAL, false>(r, at, g, p, l, last - SEG, SEG);
        }
        for (uint32_t k = full; k-- > 0;) segment(std::false_type{}, p.t0 + k * SEG, SEG, k > 0);
        if constexpr (LOCAL) {
            each<4>([&](auto i) {
                const float sum = tokens_sum(sum_dt[i]);
                if (p.tok == 0) g.carry_dt[carry_at(g, p, p.chunk) * 16 + 4 * (threadIdx.x & 3) + i] = sum;
            });
            each<S>([&](auto s) { carry_of(g, p, p.chunk)[s] = carry[s]; });
        } else {
            float* to = g.part_p + ((uint64_t)p.seq * g.chunks + p.chunk) * g.channels * (g.states + 2);
            each<4>([&](auto i) {
                const float s = tokens_sum(gskip[i]), v = tokens_sum(gbias[i]);
                if (i < p.have && p.tok == 0) {
                    const uint64_t ch = p.group * g.group_channels + p.ch4 + i;
                    to[(uint64_t)g.channels * g.states + ch] = s;
                    to[(uint64_t)g.channels * (g.states + 1) + ch] = v;
                }
            });
            if (p.valid) {
                each<S>([&](auto s) {
                    if (has_state(g, p, s)) {
                        to[(uint64_t)p.ch * g.states + p.q * S + s] = ga[s];
                        if (g.ginitial && p.chunk == 0) g.ginitial[state_at(g, p, s)] = carry[s];
                    }
                });
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
