// ssm_scan.hpp -- the selective scan over sequences, forward and backward:
//
//   dt = softplus(delta + bias)              h_t[d,n] = exp(dt A[d,n]) h_{t-1}[d,n] + dt u B_t[n]
//   y  = (sum_n C_t[n] h_t[d,n] + D u) silu(z)
//
// W waves take 16 channels and walk along the tokens in segments of 16.  Their
// lanes have two roles, between which LDS carries values:
//   * per token and channel (time steps, gates, outputs): each of the 64 W
//     lanes has 4 / W neighbouring channels of one token, loaded and stored
//     together;
//   * per state: lane (q, c) = (lane / 16, lane % 16) of wave w has S states of
//     channel c, from (4 w + q) S on, and steps through the tokens.  B and C of
//     those states lie one token a lane in the row's 16 lanes, and reach the
//     row as the DPP broadcast operand of the instruction that takes them.
//     Sums over a channel's states go to LDS after one exchange within the wave.
// Within a pass nothing is worked out twice.  (Where the token axis is cut, the
// pass before it works out the time steps and decays too, and the backward pass
// works the states out again.)  A workgroup has 64 channels, 128-byte lines of a
// 16-bit type, above 16 states 32.
//
// Bound by the issue of VALU instructions: 7.8 for each state of a token
// forward (5 of them the formula's), 22.7 in the gradients' pass, issued in 74
// to 81 % of the cycles (counters of 4 x 1024 tokens x 2048 channels x 16 states
// in bfloat16).  Measured: 4 x 2048 tokens x 4096 channels forward 166 us; 4 x
// 1024 x 2048 forward and backward 233 us; steps of 256 rows x 4096 channels 33
// us, 4.3 TB/s of states.
//
// W is 1 up to 16 states, 2 up to 32, 4 up to 64.  (16 states on two waves were
// tried where every SIMD has a wave without: 4 x 2048 tokens x 4096 channels in
// bfloat16 194 us, when one took 177.  For tensors of fewer waves they are not
// measured.)
#pragma once

#include "ssm_common.hpp"

namespace fg {
namespace ssm {

// Multiply-adds whose first factor is lane J of the row's v, in statements of
// assembly: the compiler does not fold the broadcast into a multiply-add.  The
// s_nop keeps the two wait states that a DPP operand needs after the
// instruction that wrote it; who takes a result into a lane exchange settles it
// first (settle()).
#define FG_FMAC(acc, v, x, j) "v_fmac_f32_dpp %" #acc ", %" #v ", %" #x " row_newbcast:%" #j " row_mask:0xf bank_mask:0xf\n\t"
// acc[s] += v[s] * x, s < N.
template <int N, int J>
__device__ __forceinline__ void bcast_fmac(float (&a)[N], const float (&v)[N], float x) {
    if constexpr (N == 1)
        asm("s_nop 1\n\t" FG_FMAC(0, 1, 2, 3) : "+v"(a[0]) : "v"(v[0]), "v"(x), "n"(J));
    else if constexpr (N == 2)
        asm("s_nop 1\n\t" FG_FMAC(0, 2, 4, 5) FG_FMAC(1, 3, 4, 5)
            : "+&v"(a[0]), "+&v"(a[1])
            : "v"(v[0]), "v"(v[1]), "v"(x), "n"(J));
    else
        asm("s_nop 1\n\t" FG_FMAC(0, 4, 8, 9) FG_FMAC(1, 5, 8, 9) FG_FMAC(2, 6, 8, 9) FG_FMAC(3, 7, 8, 9)
            : "+&v"(a[0]), "+&v"(a[1]), "+&v"(a[2]), "+&v"(a[3])
            : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(x), "n"(J));
}
// acc += sum_s v[s] * x[s].
template <int N, int J>
__device__ __forceinline__ void bcast_dot(float& a, const float (&v)[N], const float (&x)[N]) {
    if constexpr (N == 1)
        asm("s_nop 1\n\t" FG_FMAC(0, 1, 2, 3) : "+&v"(a) : "v"(v[0]), "v"(x[0]), "n"(J));
    else if constexpr (N == 2)
        asm("s_nop 1\n\t" FG_FMAC(0, 1, 3, 5) FG_FMAC(0, 2, 4, 5)
            : "+&v"(a)
            : "v"(v[0]), "v"(v[1]), "v"(x[0]), "v"(x[1]), "n"(J));
    else
        asm("s_nop 1\n\t" FG_FMAC(0, 1, 5, 9) FG_FMAC(0, 2, 6, 9) FG_FMAC(0, 3, 7, 9) FG_FMAC(0, 4, 8, 9)
            : "+&v"(a)
            : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "n"(J));
}
// Two tokens' sums (lanes J and K), their instructions in turn.
template <int N, int J, int K>
__device__ __forceinline__ void bcast_dots(float& a, float& b, const float (&v)[N], const float (&x)[N],
                                           const float (&y)[N]) {
    if constexpr (N == 1)
        asm("s_nop 1\n\t" FG_FMAC(0, 2, 3, 5) FG_FMAC(1, 2, 4, 6)
            : "+&v"(a), "+&v"(b)
            : "v"(v[0]), "v"(x[0]), "v"(y[0]), "n"(J), "n"(K));
    else if constexpr (N == 2)
        asm("s_nop 1\n\t" FG_FMAC(0, 2, 4, 8) FG_FMAC(1, 2, 6, 9) FG_FMAC(0, 3, 5, 8) FG_FMAC(1, 3, 7, 9)
            : "+&v"(a), "+&v"(b)
            : "v"(v[0]), "v"(v[1]), "v"(x[0]), "v"(x[1]), "v"(y[0]), "v"(y[1]), "n"(J), "n"(K));
    else
        asm("s_nop 1\n\t" FG_FMAC(0, 2, 6, 14) FG_FMAC(1, 2, 10, 15) FG_FMAC(0, 3, 7, 14) FG_FMAC(1, 3, 11, 15)
            FG_FMAC(0, 4, 8, 14) FG_FMAC(1, 4, 12, 15) FG_FMAC(0, 5, 9, 14) FG_FMAC(1, 5, 13, 15)
            : "+&v"(a), "+&v"(b)
            : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(y[0]),
              "v"(y[1]), "v"(y[2]), "v"(y[3]), "n"(J), "n"(K));
}
#undef FG_FMAC

// For i < N: low[i] + low[i] of the lane that MOVE names, in the banks of four
// lanes of BANKS high[i] + high[i] of it, to low[i].  In assembly: the compiler
// makes two selections of this and one sum.
#define FG_FOLD(i, move) "v_add_f32_dpp %" #i ", %" #i ", %" #i " " move " row_mask:0xf bank_mask:0xf\n\t"
#define FG_OVER(i, n, move, banks) "v_add_f32_dpp %" #i ", %" #n ", %" #n " " move " row_mask:0xf bank_mask:" banks "\n\t"
#define FG_HALVE(NAME, MOVE, BANKS)                                                                             \
    template <int N>                                                                                            \
    __device__ __forceinline__ void NAME(float* low, const float* high) {                                       \
        if constexpr (N == 8) {                                                                                 \
            NAME<4>(low, high);                                                                                 \
            NAME<4>(low + 4, high + 4);                                                                         \
        } else if constexpr (N == 4) {                                                                          \
            asm("s_nop 1\n\t" FG_FOLD(0, MOVE) FG_FOLD(1, MOVE) FG_FOLD(2, MOVE)  \
                FG_FOLD(3, MOVE) FG_OVER(0, 4, MOVE, BANKS) FG_OVER(1, 5, MOVE, BANKS)                \
                FG_OVER(2, 6, MOVE, BANKS) FG_OVER(3, 7, MOVE, BANKS)                                           \
                : "+&v"(low[0]), "+&v"(low[1]), "+&v"(low[2]), "+&v"(low[3])                                    \
                : "v"(high[0]), "v"(high[1]), "v"(high[2]), "v"(high[3]));                                      \
        } else if constexpr (N == 2) {                                                                          \
            asm("s_nop 1\n\t" FG_FOLD(0, MOVE) FG_FOLD(1, MOVE) FG_OVER(0, 2, MOVE, BANKS)  \
                FG_OVER(1, 3, MOVE, BANKS)                                                                      \
                : "+&v"(low[0]), "+&v"(low[1])                                                                  \
                : "v"(high[0]), "v"(high[1]));                                                                  \
        } else {                                                                                                \
            asm("s_nop 1\n\t" FG_FOLD(0, MOVE) FG_OVER(0, 1, MOVE, BANKS)                             \
                : "+&v"(low[0])                                                                                 \
                : "v"(high[0]));                                                                                \
        }                                                                                                       \
    }
FG_HALVE(halve8, "row_ror:8", "0xc")
FG_HALVE(halve4, "row_half_mirror", "0xa")
#undef FG_HALVE
#undef FG_OVER
#undef FG_FOLD

// The sum over a row's 16 channels of each of v[0 .. 4 N): halving the values
// with every bit of the lane number, so that lane c ends with the sum of value
// c (N = 4), c >> 1 (2) or c >> 2 (1) in v[0].
template <int N>
__device__ __forceinline__ void channels_sum(float (&v)[4 * N], uint32_t c) {
    const bool b1 = c & 2, b0 = c & 1;
    auto level = [&](auto half, bool upper, auto ctrl) {
        each<half>([&](auto i) {
            const float low = v[i], high = v[i + half];
            v[i] = (upper ? high : low) + dpp<ctrl>(upper ? low : high);
        });
    };
    halve8<2 * N>(v, v + 2 * N);
    halve4<N>(v, v + N);
    if constexpr (N >= 2) level(Int<N / 2>{}, b1, Int<kXor2>{});
    else settle(v[0]), v[0] += dpp<kXor2>(v[0]);  // written in assembly (halve4)
    if constexpr (N >= 4) level(Int<1>{}, b0, Int<kXor1>{});
    else v[0] += dpp<kXor1>(v[0]);
}

// A sequence's first row, packed; offsets beyond the rows are taken as the nearest.
__device__ __forceinline__ int64_t scan_row_of(const fg_scan_kargs& g, uint32_t seq) {
    const int64_t a = g.offsets[seq], all = (int64_t)g.tokens;
    return a < 0 ? 0 : a > all ? all : a;
}

// The first place of sequence `seq` among the chunks of all.  Packed: one for
// every chunk's length of rows and one more for each sequence, not for each
// sequence's longest.
__device__ __forceinline__ uint64_t scan_places_before(const fg_scan_kargs& g, uint32_t seq) {
    return g.offsets ? (uint64_t)((uint32_t)scan_row_of(g, seq) / g.chunk_len) + seq : (uint64_t)seq * g.chunks;
}

// WIDE: every row takes vector loads and stores, every channel has 4 S W
// states; else any alignment and stride, and fewer states.
template <class T, int S, int W, bool WIDE>
struct Scan {
    static constexpr bool PAD = !WIDE;
    using raw = typename T::raw;
    static constexpr int SEG = FG_SSM_SEGMENT, ES = sizeof(raw);
    static constexpr int VC = 4 / W;                      // channels of a lane as (token, channels)
    static constexpr int BLOCKS = FG_SSM_BLOCKS(W);       // of 16 channels in a workgroup
    static constexpr int THREADS = 64 * W * BLOCKS;

    // Where a wave works: its sequence, the tokens of its chunk, its channels.
    struct Place {
        int64_t start;               // packed: the sequence's first row
        uint64_t first;              // its first place among the chunks of all
        uint32_t len;                // tokens of the sequence
        uint32_t seq, chunk, group, block;
        uint32_t t0, t1;             // the chunk's tokens
        uint32_t set;                // the 16 channels' number in the workgroup
        uint32_t part;               // the wave's number among the W
        uint32_t sets;               // the 16 channels' number among all
        // as (q, c): channel among all (the group's last where there is none), row among 4 W
        uint32_t q, c, ch, row;
        bool valid;
        // as (token, channels): first channel in the 16 and in the group, how many there are
        uint32_t tok, sub, in_group;
        int have;
    };
    static __device__ __forceinline__ Place place(const fg_scan_kargs& g) {
        Place p;
        const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
        p.set = wave / W;
        p.part = wave % W;
        p.q = lane >> 4;
        p.c = lane & 15;
        p.row = 4 * p.part + p.q;
        const uint32_t e = (p.part * 64 + lane) * VC;
        p.tok = e / 16;
        p.sub = e % 16;
        const uint32_t blocks = g.groups * g.group_blocks;
        // Workgroups go to the 8 XCDs in turn, which spreads packed sequences'
        // unequal parts; in whole lines, neighbours share only B and C.
        const uint32_t cb = blockIdx.x % blocks, rest = blockIdx.x / blocks;
        p.group = cb / g.group_blocks;
        p.block = cb % g.group_blocks;
        p.chunk = rest % g.chunks;
        p.seq = rest / g.chunks;
        p.start = 0;
        p.first = (uint64_t)p.seq * g.chunks;
        p.len = g.length;
        if (g.offsets) {
            // offsets out of order or beyond the rows give shorter sequences, not accesses outside
            const int64_t a = scan_row_of(g, p.seq);
            int64_t b = scan_row_of(g, p.seq + 1);
            b = b < a ? a : b;
            p.start = uniform(a);
            p.first = (uint64_t)((uint32_t)p.start / g.chunk_len) + p.seq;
            p.len = uniform((uint32_t)(b - a < (int64_t)g.length ? b - a : (int64_t)g.length));
        }
        const uint64_t first = (uint64_t)p.chunk * g.chunk_len;
        p.t0 = first < p.len ? (uint32_t)first : p.len;
        p.t1 = p.len - p.t0 < g.chunk_len ? p.len : p.t0 + g.chunk_len;
        const uint32_t base = (p.block * BLOCKS + p.set) * 16;
        p.valid = base + p.c < g.group_channels;
        p.ch = p.group * g.group_channels + (p.valid ? base + p.c : g.group_channels - 1);
        p.in_group = base + p.sub;
        p.have = p.in_group >= g.group_channels ? 0
                 : g.group_channels - p.in_group < VC ? (int)(g.group_channels - p.in_group) : VC;
        p.sets = cb * BLOCKS + p.set;
        return p;
    }

    // N neighbouring elements as they lie in memory, in whole registers.  Wide:
    // one load, 16-bit ones two to a register; else one load and register for
    // each, at offsets of their own.  Nothing waits for a load before up().
    template <int N>
    struct Pack {
        static constexpr int WORDS = WIDE ? (N * ES + 3) / 4 : N;
        uint32_t w[WORDS];
        __device__ __forceinline__ float up(int i) const {
            if constexpr (ES == 4) return __uint_as_float(w[i]);
            else if constexpr (WIDE) return T::up((raw)(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffff));
            else return T::up((raw)w[i]);
        }
        // The first use of what was loaded: conversions that the compiler moves
        // up to the segment before wait for their loads there.
        __device__ __forceinline__ void arrive() {
            each<WORDS>([&](auto i) { asm volatile("" : "+v"(w[i])); });
        }
        __device__ __forceinline__ void load(const char* at, uint32_t row, const uint32_t (&off)[N]) {
            if constexpr (!WIDE) {
                each<N>([&](auto i) {
                    const raw x = *(const raw*)(at + fresh(row + off[i]));
                    if constexpr (ES == 4) w[i] = __builtin_bit_cast(uint32_t, x);
                    else w[i] = x;
                });
            } else if constexpr (N * ES >= 4) {
                struct __attribute__((aligned(N * ES))) Words {
                    uint32_t w[WORDS];
                };
                const Words x = *(const Words*)(at + fresh(row + off[0]));
                each<WORDS>([&](auto i) { w[i] = x.w[i]; });
            } else {
                w[0] = *(const raw*)(at + fresh(row + off[0]));
            }
        }
    };
    using RawC = Pack<VC>;
    using RawS = Pack<S>;
    struct __attribute__((aligned(4 * VC))) FloatC {
        float v[VC];
    };

    // The lane's constants.
    struct Lane {
        bool pad[S];
        float a2[S];               // A log2(e)
        float bias[VC], skip[VC];
        uint32_t offc[VC];         // the channels' offsets in a row, bytes
        uint32_t offs[S];          // the states' offsets in a row of B and C, bytes
    };
    static __device__ __forceinline__ Lane lane(const fg_scan_kargs& g, const Place& p) {
        Lane l;
        each<S>([&](auto s) {
            const uint32_t n = p.row * S + s, m = n < g.states ? n : g.states - 1;
            l.pad[s] = PAD && n >= g.states;
            l.a2[s] = n < g.states ? g.a[(uint64_t)p.ch * g.states + n] * kLog2e : 0.0f;
            l.offs[s] = (p.group * g.states + m) * ES;
        });
        each<VC>([&](auto i) {
            // a channel that is not there: the group's last one (wide loads: its last ones)
            uint32_t c = p.in_group + i;
            if (c >= g.group_channels) c = WIDE ? g.group_channels - VC + i : g.group_channels - 1;
            c += p.group * g.group_channels;
            l.offc[i] = c * ES;
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
    template <bool TAIL, int N>
    static __device__ __forceinline__ void load(Pack<N>& v, const Cursor& w, uint32_t row, const uint32_t (&off)[N],
                                                uint32_t n) {
        v.load(w.at, row_of<TAIL>(row, n) * w.row, off);
    }
    template <bool TAIL>
    static __device__ __forceinline__ void store(const Cursor& w, const Place& p, const Lane& l, uint32_t n,
                                                 const float (&x)[VC]) {
        if (TAIL && p.tok >= n) return;
        const uint32_t r = p.tok * w.row;
        char* to = const_cast<char*>(w.at);
        if constexpr (WIDE) {
            struct __attribute__((aligned(VC * ES))) Out {
                raw v[VC];
            } v;
            each<VC>([&](auto i) { v.v[i] = T::down(x[i]); });
            if (p.have > 0) *(Out*)(to + fresh(r + l.offc[0])) = v;
        } else {
            each<VC>([&](auto i) {
                if (i < p.have) *(raw*)(to + fresh(r + l.offc[i])) = T::down(x[i]);
            });
        }
    }
    static __device__ __forceinline__ void up(float (&x)[VC], RawC& v) {
        v.arrive();
        each<VC>([&](auto i) { x[i] = v.up(i); });
    }
    static __device__ __forceinline__ void up(float (&x)[S], RawS& v, const Lane& l) {
        v.arrive();
        each<S>([&](auto s) { x[s] = PAD && l.pad[s] ? 0.0f : v.up(s); });
    }

    // Places of the wave's 64 S values: the states at the start of the segment
    // at token t, what a chunk adds, and the initial states.
    static __device__ __forceinline__ uint64_t lanes_of(const fg_scan_kargs& g, const Place& p, uint64_t k) {
        return ((k * (g.groups * g.group_blocks * BLOCKS) + p.sets) * W + p.part) * (64 * S) + (threadIdx.x & 63) * S;
    }
    static __device__ __forceinline__ float* check_of(const fg_scan_kargs& g, const Place& p, uint32_t t) {
        const uint64_t seg = g.offsets ? (uint64_t)p.start / SEG + p.seq : (uint64_t)p.seq * g.check_segs;
        return g.check + lanes_of(g, p, seg + t / SEG);
    }
    static __device__ __forceinline__ float* carry_of(const fg_scan_kargs& g, const Place& p, uint32_t chunk) {
        return g.carry + lanes_of(g, p, p.first + chunk);
    }
    static __device__ __forceinline__ float* initial_of(const fg_scan_kargs& g, const Place& p) {
        return g.carry + lanes_of(g, p, g.places + p.seq);
    }
    // The 16 channels' summed time steps of chunk k.
    static __device__ __forceinline__ float* carry_dt_of(const fg_scan_kargs& g, const Place& p, uint32_t chunk) {
        return g.carry_dt + ((p.first + chunk) * (g.groups * g.group_blocks * BLOCKS) + p.sets) * 16;
    }
    static __device__ __forceinline__ uint64_t state_at(const fg_scan_kargs& g, const Place& p, int s) {
        return ((uint64_t)p.seq * g.channels + p.ch) * g.states + p.row * S + s;
    }
    static __device__ __forceinline__ bool has_state(const fg_scan_kargs& g, const Place& p, int s) {
        return !PAD || p.row * S + s < g.states;
    }

    // Takes the states h over n chunks, the i-th of them chunk at(i): four are
    // loaded at a time.  A chunk's factor can pass the range that the states keep
    // token by token (growing ones, of positive A or negative steps).
    template <class At>
    static __device__ __forceinline__ void take_chunks(const fg_scan_kargs& g, const Place& p, const Lane& l,
                                                       float (&h)[S], uint32_t n, At&& at) {
        for (uint32_t k = 0; k < n; k += 4) {
            float sum[4], add[4][S];
            each<4>([&](auto j) {
                const uint32_t i = at(k + j < n ? k + j : n - 1);
                sum[j] = carry_dt_of(g, p, i)[p.c];
                each<S>([&](auto s) { add[j][s] = carry_of(g, p, i)[s]; });
            });
            each<4>([&](auto j) {
                const float half = 0.5f * sum[j];
                if (k + j < n)
                    each<S>([&](auto s) {
                        h[s] = times_exp2_twice(h[s], half * l.a2[s], add[j][s]);
                        if (PAD && l.pad[s]) h[s] = 0.0f;
                    });
            });
        }
    }

    // Orders LDS accesses of the waves that share channels: the wave's own
    // (W = 1), or the workgroup's.  Global loads on their way stay on it.
    template <bool GROUP>
    static __device__ __forceinline__ void sync() {
        if constexpr (GROUP) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }

    // Sums over the states of each (token, channel): 2 W parts, each the sum of
    // two rows of a wave.
    static constexpr int PART = SEG * 16 + 16;  // the 16 keep a wave's rows on banks of their own
    struct Sums {
        float v[2 * W][PART];
        // v[j]: the lane's sum for token 4 i + j
        __device__ __forceinline__ void put(const Place& p, int i, float (&x)[4]) {
            settle(x[0], x[1], x[2], x[3]);  // written in assembly (bcast_dot)
            float* to = v[2 * p.part + (p.q & 1)] + (4 * i + (p.q & 2)) * 16 + p.c;
            to[0] = swap32_add(x[0], x[2]);
            to[16] = swap32_add(x[1], x[3]);
        }
        __device__ __forceinline__ void get(const Place& p, float (&x)[VC]) const {
            FloatC f = *(const FloatC*)(v[0] + p.tok * 16 + p.sub);
            each<VC>([&](auto i) { x[i] = f.v[i]; });
            each<2 * W - 1>([&](auto k) {
                f = *(const FloatC*)(v[k + 1] + p.tok * 16 + p.sub);
                each<VC>([&](auto i) { x[i] += f.v[i]; });
            });
        }
    };
    // Sum over a segment's tokens of what each (token, channels) lane holds, to
    // the lanes of the first token; `room`: LDS, 16 floats for each wave.
    static __device__ __forceinline__ float tokens_sum(const Place& p, float v, float* room) {
        for (int m = 16 / VC; m < 64; m *= 2) v += __shfl_xor(v, m);
        if constexpr (W > 1) {
            const uint32_t lane = threadIdx.x & 63;
            sync<true>();
            if (lane < 16 / VC) room[p.part * 16 + lane] = v;
            sync<true>();
            v = 0.0f;
            each<W>([&](auto w) { v += room[w * 16 + lane % (16 / VC)]; });
            sync<true>();
        }
        return v;
    }

    // No branch on softplus: the segment stays one block, which the compiler interleaves.
    static __device__ __forceinline__ Softplus time_step(const fg_scan_kargs& g, float x) {
        const Softplus s = softplus(x);
        return {g.softplus ? s.value : x, g.softplus ? s.slope : 1.0f};
    }

    // ------------------------------------------------------------ forward

    // LDS of 16 channels, twice, so that one barrier a segment does: a segment
    // is made ready, and the one before it stored, while one is worked through.
    static constexpr int XSTRIDE = 2 * SEG + 4;  // keeps the 16 channels on banks of their own
    template <bool LOCAL>
    struct ForwardLds {
        float x[2][16 * XSTRIDE];  // per channel the tokens' (dt, dt u)
        std::conditional_t<LOCAL, float, Sums> y[2];
    };

    // Segments whose rows are in registers or on the way: what a lane loads is
    // small, and memory answers after one to two microseconds.
    static constexpr int RING = ES == 2 ? 4 : 3;

    // A segment's time steps, to LDS.
    template <bool LOCAL, bool TAIL>
    static __device__ __forceinline__ void prepare(const fg_scan_kargs& g, const Place& p, const Lane& l, float* x,
                                                   float (&sum_dt)[VC], const float (&d)[VC], const float (&u)[VC],
                                                   uint32_t n, bool count) {
        each<VC>([&](auto i) {
            const float dt = time_step(g, d[i] + l.bias[i]).value;
            const float2 e = {dt, dt * u[i]};
            *(float2*)(x + (p.sub + i) * XSTRIDE + 2 * p.tok) = e;
            if constexpr (LOCAL) sum_dt[i] += count && (!TAIL || p.tok < n) ? dt : 0.0f;
        });
    }
    template <int J>
    static __device__ __forceinline__ void advance(const Lane& l, float (&h)[S], const float (&b)[S], float dt,
                                                   float dtu) {
        each<S>([&](auto s) {
            h[s] = fmaf(exp2_(dt * l.a2[s]), h[s], row_bcast<J>(b[s]) * dtu);
            if (PAD && l.pad[s]) h[s] = 0.0f;
        });
    }
    // Four tokens' (dt, dt u), read before what is worked through ahead of
    // them: the compiler moves no LDS read above a write.
    struct Steps {
        float4 a, b;
        __device__ __forceinline__ void read(const Place& p, const float* x, int i) {
            a = *(const float4*)(x + p.c * XSTRIDE + 8 * i);
            b = *(const float4*)(x + p.c * XSTRIDE + 8 * i + 4);
        }
    };
    template <bool LOCAL, bool TAIL, class Y>
    static __device__ __forceinline__ void forward_segment(const Place& p, const Lane& l, const float* x, Steps next,
                                                           Y& y, float (&h)[S], const float (&b)[S],
                                                           const float (&c)[S], uint32_t n) {
        each<SEG / 4>([&](auto i) {
            const float e[8] = {next.a.x, next.a.y, next.a.z, next.a.w, next.b.x, next.b.y, next.b.z, next.b.w};
            float ys[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (i + 1 < SEG / 4) next.read(p, x, i + 1);
            each<2>([&](auto k) {
                constexpr int j = 2 * k, m = 4 * i + j;
                if constexpr (TAIL) {
                    if (m < n) {
                        advance<m>(l, h, b, e[2 * j], e[2 * j + 1]);
                        if constexpr (!LOCAL) bcast_dot<S, m>(ys[j], c, h);
                    }
                    if (m + 1 < n) {
                        advance<m + 1>(l, h, b, e[2 * j + 2], e[2 * j + 3]);
                        if constexpr (!LOCAL) bcast_dot<S, m + 1>(ys[j + 1], c, h);
                    }
                } else {
                    float first[S];
                    advance<m>(l, h, b, e[2 * j], e[2 * j + 1]);
                    each<S>([&](auto s) { first[s] = h[s]; });
                    advance<m + 1>(l, h, b, e[2 * j + 2], e[2 * j + 3]);
                    if constexpr (!LOCAL) bcast_dots<S, m, m + 1>(ys[j], ys[j + 1], c, first, h);
                }
            });
            if constexpr (!LOCAL) y.put(p, i, ys);
        });
    }
    template <bool TAIL>
    static __device__ __forceinline__ void outputs(const fg_scan_kargs& g, const Place& p, const Lane& l,
                                                   const Sums& y, const Cursor& out, RawC& ru, RawC& rz,
                                                   bool gated, uint32_t n) {
        float u[VC], z[VC], o[VC];
        up(u, ru);
        up(z, rz);
        y.get(p, o);
        each<VC>([&](auto i) {
            const float gate = z[i] * sigmoid(z[i]);
            o[i] = fmaf(l.skip[i], u[i], o[i]) * (gated ? gate : 1.0f);
        });
        store<TAIL>(out, p, l, n, o);
    }

    // LOCAL: the states that the chunk's own tokens leave, from none, and the
    // sum of its time steps; else outputs, from the states before the chunk.
    template <bool LOCAL>
    static __device__ __forceinline__ void forward(const fg_scan_kargs& g) {
        __shared__ __attribute__((aligned(16))) ForwardLds<LOCAL> all[BLOCKS];
        constexpr bool SHARED = W > 1;
        const Place p = place(g);
        if (LOCAL && p.chunk == 0) {
            // the last chunks may write the final states where the initial ones lie
            each<S>([&](auto s) {
                const bool has = g.initial && has_state(g, p, s);
                initial_of(g, p)[s] = has ? g.initial[state_at(g, p, s)] : 0.0f;
            });
        }
        if (LOCAL && p.t1 == p.len) return;                 // no chunk follows
        if (!LOCAL && p.chunk > 0 && p.t0 == p.t1) return;  // no tokens
        const Lane l = lane(g, p);
        ForwardLds<LOCAL>& lds = all[p.set];
        float h[S], sum_dt[VC];
        each<VC>([&](auto i) { sum_dt[i] = 0.0f; });
        each<S>([&](auto s) { h[s] = 0.0f; });
        if constexpr (!LOCAL) {
            each<S>([&](auto s) {
                if (g.chunks > 1) h[s] = initial_of(g, p)[s];
                else if (g.initial && has_state(g, p, s)) h[s] = g.initial[state_at(g, p, s)];
            });
            take_chunks(g, p, l, h, p.chunk, [](uint32_t i) { return i; });
        }
        // Without a gate u's rows stand in for z's, which are then not used.
        const bool gated = g.z.p != nullptr;
        struct {
            Cursor u, d, z, b, c;
        } at;
        Cursor out;
        auto set = [&](uint32_t t) {
            at.u.set(g.u, p, t);
            at.d.set(g.delta, p, t);
            at.b.set(g.b, p, t);
            if constexpr (!LOCAL) {
                at.c.set(g.c, p, t);
                at.z.set(gated ? g.z : g.u, p, t);
                out.set(g.out, p, t);
            }
        };
        struct Rows {
            RawC u, d, z;
            RawS b, c;
        } ring[RING];
        auto fetch = [&](Rows& r, auto tail, uint32_t n) {
            constexpr bool TAIL = decltype(tail)::value;
            load<TAIL>(r.d, at.d, p.tok, l.offc, n);
            load<TAIL>(r.u, at.u, p.tok, l.offc, n);
            load<TAIL>(r.b, at.b, p.c, l.offs, n);
            if constexpr (!LOCAL) {
                load<TAIL>(r.c, at.c, p.c, l.offs, n);
                load<TAIL>(r.z, at.z, p.tok, l.offc, n);
            }
        };
        auto forth = [&](int by) {
            at.u.move(by);
            at.d.move(by);
            at.b.move(by);
            if constexpr (!LOCAL) {
                at.c.move(by);
                at.z.move(by);
            }
        };
        float d[VC], u[VC], b[S], c[S];
        auto checkpoint = [&](uint32_t t) {
            if constexpr (!LOCAL) {
                if (g.check) {  // lanes without a channel too: the backward pass reads them
                    float* to = check_of(g, p, t);
                    each<S>([&](auto s) { to[s] = h[s]; });
                }
            }
        };
        const uint32_t full = (p.t1 - p.t0) / SEG, rest = (p.t1 - p.t0) % SEG;
        set(p.t0);
        if (full > 0) {
            // While segment k is worked through, k + 1 is made ready, the rows
            // of k + RING - 1 are loaded (beyond the last the last, to no
            // use), and the outputs of k - 1 are stored.
            each<RING - 1>([&](auto j) {
                fetch(ring[j], std::false_type{}, SEG);
                forth(j + 1 < full);
            });
            up(d, ring[0].d);
            up(u, ring[0].u);
            prepare<LOCAL, false>(g, p, l, lds.x[0], sum_dt, d, u, SEG, true);
            auto store_last = [&](auto j, uint32_t m) {  // segment m, which lies in ring[j]
                if constexpr (!LOCAL) {
                    outputs<false>(g, p, l, lds.y[m & 1], out, ring[j].u, ring[j].z, gated, SEG);
                    out.move(1);
                }
            };
            auto step = [&](auto j, uint32_t m) {
                constexpr int before = (j + RING - 1) % RING;
                sync<SHARED>();
                if (j > 0 || m > 0) store_last(Int<before>{}, m - 1);
                fetch(ring[before], std::false_type{}, SEG);
                forth(m + RING < full);
                up(b, ring[j].b, l);
                if constexpr (!LOCAL) up(c, ring[j].c, l);
                up(d, ring[(j + 1) % RING].d);
                up(u, ring[(j + 1) % RING].u);
                checkpoint(p.t0 + m * SEG);
                Steps first;
                first.read(p, lds.x[m & 1], 0);
                prepare<LOCAL, false>(g, p, l, lds.x[(m + 1) & 1], sum_dt, d, u, SEG, m + 1 < full);
                forward_segment<LOCAL, false>(p, l, lds.x[m & 1], first, lds.y[m & 1], h, b, c, SEG);
            };
            // Whole turns of the ring: a step that could be skipped would cost
            // the others their count of loads on the way.
            uint32_t k = 0;
            for (; k + RING <= full; k += RING) each<RING>([&](auto j) { step(j, k + j); });
            auto finish = [&](auto self, auto j) {
                if (k + j < full) {
                    step(j, k + j);
                    if constexpr (j + 2 < RING) self(self, Int<j + 1>{});
                    else sync<SHARED>(), store_last(j, k + j);
                } else {
                    sync<SHARED>();
                    store_last(Int<(j + RING - 1) % RING>{}, k + j - 1);
                }
            };
            finish(finish, Int<0>{});
            sync<SHARED>();
        }
        if (rest > 0) {
            Rows& r = ring[0];
            set(p.t0 + full * SEG);
            checkpoint(p.t0 + full * SEG);
            fetch(r, std::true_type{}, rest);
            if constexpr (!LOCAL) up(c, r.c, l);
            up(d, r.d);
            up(u, r.u);
            up(b, r.b, l);
            prepare<LOCAL, true>(g, p, l, lds.x[0], sum_dt, d, u, rest, true);
            sync<SHARED>();
            Steps first;
            first.read(p, lds.x[0], 0);
            forward_segment<LOCAL, true>(p, l, lds.x[0], first, lds.y[0], h, b, c, rest);
            sync<SHARED>();
            if constexpr (!LOCAL) outputs<true>(g, p, l, lds.y[0], out, r.u, r.z, gated, rest);
        }
        if constexpr (LOCAL) {
            each<VC>([&](auto i) {
                const float sum = tokens_sum(p, sum_dt[i], lds.x[0]);
                if (p.tok == 0) carry_dt_of(g, p, p.chunk)[p.sub + i] = sum;
            });
            each<S>([&](auto s) { carry_of(g, p, p.chunk)[s] = h[s]; });
        } else if (g.final && p.valid && p.t1 == p.len) {
            each<S>([&](auto s) {
                if (has_state(g, p, s)) g.final[state_at(g, p, s)] = h[s];
            });
        }
    }

    // ----------------------------------------------------------- backward

    // LDS of 16 channels: per channel the tokens' time steps dt, gradients ds
    // of the ungated outputs, and inputs dt u; the sums over states (y, g B,
    // g a h A); what the (token, channels) lanes keep until the end of the
    // segment; B's and C's gradients summed over the 16 channels.
    static constexpr int TSTRIDE = SEG + 4;
    struct BackwardLds {
        float dt[16 * TSTRIDE], ds[16 * TSTRIDE], dtu[16 * TSTRIDE];
        Sums res[3];
        FloatC keep[5][64 * W];  // u, dt, its slope, ds, z's factor
        float bc[SEG * 2 * 4 * S * W];
    };
    struct LocalLds {
        float dt[16 * TSTRIDE], ds[16 * TSTRIDE];
    };
    template <bool LOCAL>
    struct BackRaws {
        RawC u, d, dy, z;
        RawS b, c;
        float h0[S];
    };
    template <bool LOCAL>
    struct BackCursors {
        Cursor u, d, dy, z, b, c;
        __device__ __forceinline__ void move(int by) {
            d.move(by);
            dy.move(by);
            z.move(by);
            c.move(by);
            if constexpr (!LOCAL) {
                u.move(by);
                b.move(by);
            }
        }
    };
    template <bool LOCAL, bool TAIL>
    static __device__ __forceinline__ void back_load(BackRaws<LOCAL>& r, const BackCursors<LOCAL>& at,
                                                     const fg_scan_kargs& g, const Place& p, const Lane& l, uint32_t t,
                                                     uint32_t n) {
        load<TAIL>(r.d, at.d, p.tok, l.offc, n);
        load<TAIL>(r.dy, at.dy, p.tok, l.offc, n);
        load<TAIL>(r.z, at.z, p.tok, l.offc, n);
        load<TAIL>(r.c, at.c, p.c, l.offs, n);
        if constexpr (!LOCAL) {
            load<TAIL>(r.u, at.u, p.tok, l.offc, n);
            load<TAIL>(r.b, at.b, p.c, l.offs, n);
        }
        if constexpr (!LOCAL) {
            const float* from = check_of(g, p, t);
            each<S>([&](auto s) { r.h0[s] = from[s]; });
        }
    }
    // Time steps and output gradients, to LDS, with what the end of the segment needs.
    template <bool LOCAL, class L>
    static __device__ __forceinline__ void back_prepare(BackRaws<LOCAL>& r, const fg_scan_kargs& g,
                                                        const Place& p, const Lane& l, L& lds, float (&dt)[VC],
                                                        bool gated) {
        float d[VC], dy[VC], z[VC], u[VC];
        FloatC k[5];
        up(d, r.d);
        up(dy, r.dy);
        up(z, r.z);
        if constexpr (!LOCAL) up(u, r.u);
        each<VC>([&](auto i) {
            const Softplus s = time_step(g, d[i] + l.bias[i]);
            dt[i] = s.value;
            const float sg = sigmoid(z[i]);
            const float ds = gated ? dy[i] * (z[i] * sg) : dy[i];
            // a channel that is not there adds nothing to the sums over channels
            const bool here = i < p.have;
            const uint32_t at = (p.sub + i) * TSTRIDE + p.tok;
            lds.dt[at] = dt[i];
            lds.ds[at] = here ? ds : 0.0f;
            if constexpr (!LOCAL) {
                lds.dtu[at] = here ? dt[i] * u[i] : 0.0f;
                k[0].v[i] = u[i];
                k[1].v[i] = dt[i];
                k[2].v[i] = s.slope;
                k[3].v[i] = ds;
                k[4].v[i] = dy[i] * (sg * fmaf(z[i], 1.0f - sg, 1.0f));
            }
        });
        if constexpr (!LOCAL) each<5>([&](auto i) { lds.keep[i][p.part * 64 + (threadIdx.x & 63)] = k[i]; });
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
    // The gradients of one segment's tokens.  `midway` runs where half of the
    // states are no longer needed: it loads the next segment's rows.
    template <bool TAIL, class F>
    static __device__ __forceinline__ void back_segment(const Place& p, const Lane& l, BackwardLds& lds,
                                                        float (&carry)[S], float (&ga)[S], const float (&b)[S],
                                                        const float (&c)[S], const float (&h0)[S], uint32_t n,
                                                        F&& midway) {
        float a[SEG][S], h[SEG][S];
        const float *xdt = lds.dt + p.c * TSTRIDE, *xds = lds.ds + p.c * TSTRIDE, *xdtu = lds.dtu + p.c * TSTRIDE;
        // Four tokens' values, read ahead as in forward_segment.
        struct Steps {
            float4 dt, dtu, ds;
        } next;
        next.dt = *(const float4*)xdt;
        next.dtu = *(const float4*)xdtu;
        // the segment's states again
        each<SEG / 4>([&](auto i) {
            const float dt[4] = {next.dt.x, next.dt.y, next.dt.z, next.dt.w};
            const float dtu[4] = {next.dtu.x, next.dtu.y, next.dtu.z, next.dtu.w};
            float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            constexpr int after = i + 1 < SEG / 4 ? i + 1 : SEG / 4 - 1;  // the last is where the way back begins
            next.dt = *(const float4*)(xdt + 4 * after);
            next.dtu = *(const float4*)(xdtu + 4 * after);
            if constexpr (i + 1 == SEG / 4) next.ds = *(const float4*)(xds + 4 * after);
            each<4>([&](auto j) {
                constexpr int m = 4 * i + j;
                if (!TAIL || m < n) {
                    each<S>([&](auto s) {
                        const float before = m ? h[m ? m - 1 : 0][s] : h0[s];
                        a[m][s] = exp2_(dt[j] * l.a2[s]);
                        h[m][s] = fmaf(a[m][s], before, row_bcast<m>(b[s]) * dtu[j]);
                        if (PAD && l.pad[s]) h[m][s] = 0.0f;
                    });
                    if constexpr (TAIL) bcast_dot<S, m>(y[j], c, h[m]);
                    else if constexpr (j % 2 == 1) bcast_dots<S, m - 1, m>(y[j - 1], y[j], c, h[m - 1], h[m]);
                }
            });
            lds.res[0].put(p, i, y);
        });
        // and back
        each<SEG / 4>([&](auto ri) {
            constexpr int i = SEG / 4 - 1 - ri;
            if constexpr (ri == SEG / 8) midway();
            const float dt[4] = {next.dt.x, next.dt.y, next.dt.z, next.dt.w};
            const float dtu[4] = {next.dtu.x, next.dtu.y, next.dtu.z, next.dtu.w};
            const float ds[4] = {next.ds.x, next.ds.y, next.ds.z, next.ds.w};
            if constexpr (i > 0) {
                next.dt = *(const float4*)(xdt + 4 * (i - 1));
                next.dtu = *(const float4*)(xdtu + 4 * (i - 1));
                next.ds = *(const float4*)(xds + 4 * (i - 1));
            }
            float gb[4 * S], gc[4 * S], gu[4] = {0.0f, 0.0f, 0.0f, 0.0f}, gd[4] = {0.0f, 0.0f, 0.0f, 0.0f}, later[S];
            if constexpr (TAIL) each<4 * S>([&](auto e) { gb[e] = gc[e] = 0.0f; });
            each<4>([&](auto rj) {
                constexpr int j = 3 - rj, m = 4 * i + j;
                if (!TAIL || m < n) {
                    bcast_fmac<S, m>(carry, c, ds[j]);  // g_t
                    if constexpr (TAIL) bcast_dot<S, m>(gu[j], b, carry);
                    else if constexpr (j % 2 == 0) bcast_dots<S, m + 1, m>(gu[j + 1], gu[j], b, later, carry);
                    else each<S>([&](auto s) { later[s] = carry[s]; });
                    each<S>([&](auto s) {
                        gb[j * S + s] = carry[s] * dtu[j];
                        gc[j * S + s] = ds[j] * h[m][s];
                        carry[s] *= a[m][s];
                        if (PAD && l.pad[s]) carry[s] = 0.0f;
                        const float held = carry[s] * (m ? h[m ? m - 1 : 0][s] : h0[s]);
                        gd[j] = fmaf(held, l.a2[s], gd[j]);
                        ga[s] = fmaf(held, dt[j], ga[s]);
                    });
                }
            });
            lds.res[1].put(p, i, gu);
            lds.res[2].put(p, i, gd);
            channels_sum<S>(gb, p.c);
            channels_sum<S>(gc, p.c);
            const uint32_t e = S == 4 ? p.c : p.c >> (S == 2 ? 1 : 2);
            float* to = lds.bc + ((4 * i + e / S) * 2) * (4 * S * W) + p.row * S + e % S;
            if (S == 4 || (p.c & (S == 2 ? 1 : 3)) == 0) {
                to[0] = gb[0];
                to[4 * S * W] = gc[0];
            }
        });
    }

    // LOCAL: a_{t0} g_{t0} of the chunk's own tokens, from nothing after it;
    // else the gradients, from what the tokens after the chunk pass back.
    template <bool LOCAL>
    static __device__ __forceinline__ void backward(const fg_scan_kargs& g) {
        using Lds = std::conditional_t<LOCAL, LocalLds, BackwardLds>;
        __shared__ __attribute__((aligned(16))) Lds all[BLOCKS];
        constexpr bool SHARED = !LOCAL || W > 1;
        const Place p = place(g);
        if (LOCAL && (p.chunk == 0 || p.t1 == p.t0)) return;  // no chunk before it, or no tokens
        // packed chunks without tokens may have no place for the parameters' parts
        if (!LOCAL && p.chunk > 0 && p.t1 == p.t0 && p.first + p.chunk >= scan_places_before(g, p.seq + 1)) return;
        const Lane l = lane(g, p);
        Lds& lds = all[p.set];
        float carry[S], ga[S];
        each<S>([&](auto s) { carry[s] = ga[s] = 0.0f; });
        const bool gated = g.z.p != nullptr;
        float sum_dt[VC], gskip[VC], gbias[VC];
        each<VC>([&](auto i) { sum_dt[i] = gskip[i] = gbias[i] = 0.0f; });
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
        BackRaws<LOCAL> r;
        auto segment = [&](auto tail, uint32_t t, uint32_t n, bool more) {
            constexpr bool TAIL = decltype(tail)::value;
            float b[S], c[S], h0[S], dt[VC];
            back_prepare<LOCAL>(r, g, p, l, lds, dt, gated);
            up(c, r.c, l);
            if constexpr (!LOCAL) {
                up(b, r.b, l);
                each<S>([&](auto s) { h0[s] = r.h0[s]; });
            }
            auto midway = [&] {
                if (more) {  // the segment before this one
                    at.move(-1);
                    back_load<LOCAL, false>(r, at, g, p, l, t - SEG, SEG);
                }
            };
            sync<SHARED>();
            if constexpr (LOCAL) {
                midway();
                each<VC>([&](auto i) { sum_dt[i] += !TAIL || p.tok < n ? dt[i] : 0.0f; });
                back_local<TAIL>(p, l, lds, carry, c, n);
                sync<SHARED>();
            } else {
                back_segment<TAIL>(p, l, lds, carry, ga, b, c, h0, n, midway);
                sync<SHARED>();
                const uint32_t lane = p.part * 64 + (threadIdx.x & 63);
                float gu[VC], gd[VC], o[VC];
                const FloatC u = lds.keep[0][lane], ds = lds.keep[3][lane];
                lds.res[1].get(p, gu);
                if (g.gz.p) {
                    const FloatC v = lds.keep[4][lane];
                    lds.res[0].get(p, o);
                    each<VC>([&](auto i) { o[i] = v.v[i] * fmaf(l.skip[i], u.v[i], o[i]); });
                    store<TAIL>(cgz, p, l, n, o);
                    cgz.move(-1);
                }
                if (g.gu.p) {
                    const FloatC v = lds.keep[1][lane];
                    each<VC>([&](auto i) { o[i] = fmaf(v.v[i], gu[i], l.skip[i] * ds.v[i]); });
                    store<TAIL>(cgu, p, l, n, o);
                    cgu.move(-1);
                }
                const FloatC slope = lds.keep[2][lane];
                lds.res[2].get(p, gd);
                each<VC>([&](auto i) {
                    o[i] = fmaf(u.v[i], gu[i], kLn2 * gd[i]) * slope.v[i];
                    const bool in = !TAIL || p.tok < n;
                    gbias[i] += in ? o[i] : 0.0f;
                    gskip[i] += in ? ds.v[i] * u.v[i] : 0.0f;
                });
                if (g.gdelta.p) {
                    store<TAIL>(cgd, p, l, n, o);
                    cgd.move(-1);
                }
                // B's and C's gradients of the workgroup's channels
                constexpr int NS = 4 * S * W;
                for (uint32_t e = threadIdx.x; e < n * 2 * NS; e += THREADS) {
                    float sum = 0.0f;
                    each<BLOCKS>([&](auto w) { sum += all[w].bc[e]; });
                    const uint32_t s = e % NS, m = e / (2 * NS), which = e / NS % 2;
                    if (!PAD || s < g.states) {
                        const uint64_t tok = (g.offsets ? (uint64_t)p.start : (uint64_t)p.seq * g.length) + t + m;
                        g.part_bc[((((uint64_t)p.block * g.tokens + tok) * g.groups + p.group) * 2 + which) * g.states +
                                  s] = sum;
                    }
                }
            }
        };
        if (rest > 0) {
            back_load<LOCAL, true>(r, at, g, p, l, last, rest);
        } else if (full > 0) {
            at.move(-1);
            back_load<LOCAL, false>(r, at, g, p, l, last - SEG, SEG);
            if constexpr (!LOCAL) {
                cgu.move(-1);
                cgd.move(-1);
                cgz.move(-1);
            }
        }
        if constexpr (!LOCAL) {  // what comes from after the chunk, while the first rows are on their way
            each<S>([&](auto s) {
                if (g.gfinal && has_state(g, p, s)) carry[s] = g.gfinal[state_at(g, p, s)];
            });
            const uint32_t used = p.len ? (p.len - 1) / g.chunk_len + 1 : 0;
            if (used > p.chunk + 1)
                take_chunks(g, p, l, carry, used - p.chunk - 1, [&](uint32_t i) { return used - 1 - i; });
        }
        if (rest > 0) segment(std::true_type{}, last, rest, full > 0);
        for (uint32_t k = full; k-- > 0;) segment(std::false_type{}, p.t0 + k * SEG, SEG, k > 0);
        if constexpr (LOCAL) {
            each<VC>([&](auto i) {
                const float sum = tokens_sum(p, sum_dt[i], lds.dt);
                if (p.tok == 0) carry_dt_of(g, p, p.chunk)[p.sub + i] = sum;
            });
            each<S>([&](auto s) { carry_of(g, p, p.chunk)[s] = carry[s]; });
        } else {
            each<VC>([&](auto i) {
                gskip[i] = tokens_sum(p, gskip[i], lds.dt);
                gbias[i] = tokens_sum(p, gbias[i], lds.dt);
            });
            auto put = [&](uint64_t k) {
                float* to = g.part_p + k * g.channels * (g.states + 2);
                each<VC>([&](auto i) {
                    if (i < p.have && p.tok == 0) {
                        const uint64_t ch = p.group * g.group_channels + p.in_group + i;
                        to[(uint64_t)g.channels * g.states + ch] = gskip[i];
                        to[(uint64_t)g.channels * (g.states + 1) + ch] = gbias[i];
                    }
                });
                each<S>([&](auto s) {
                    if (p.valid && has_state(g, p, s)) to[(uint64_t)p.ch * g.states + p.row * S + s] = ga[s];
                });
            };
            const uint64_t place = p.first + p.chunk, end = scan_places_before(g, p.seq + 1);
            if (place < end) put(place);
            if (g.offsets && p.chunk + 1 == g.chunks) {
                // what is left before the next sequence's first place: zeros
                each<VC>([&](auto i) { gskip[i] = gbias[i] = 0.0f; });
                each<S>([&](auto s) { ga[s] = 0.0f; });
                for (uint64_t k = place + 1; k < end; ++k) put(k);
            }
            if (g.ginitial && p.chunk == 0 && p.valid) {
                each<S>([&](auto s) {
                    if (has_state(g, p, s)) g.ginitial[state_at(g, p, s)] = carry[s];
                });
            }
        }
    }
};

// B's and C's gradients from the channel blocks' parts, in a fixed order.
template <class T>
__device__ __forceinline__ void scan_reduce_bc(const fg_scan_kargs& g) {
    const uint32_t row = g.groups * 2 * g.states;
    const uint64_t n = g.tokens * row;
    const uint64_t e = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= n) return;
    const float v = ordered_sum(g.part_bc + e, n, g.group_blocks);
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
        const int64_t start = scan_row_of(g, lo);
        if ((int64_t)tok < start || (int64_t)tok >= g.offsets[lo + 1] || (int64_t)tok - start >= g.length) return;
    }
    const fg_ssm_view& w = which ? g.gc : g.gb;
    if (w.p) {
        ((typename T::raw*)w.p)[(int64_t)seq * w.seq + (int64_t)t * w.row + grp * g.states + s] = T::down(v);
    }
}

// The parameters' gradients from the chunks' parts, in a fixed order.
__device__ __forceinline__ void scan_reduce_p(const fg_scan_kargs& g) {
    const uint64_t n = (uint64_t)g.channels * (g.states + 2);
    const uint64_t e = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= n) return;
    // without sequences there are no places (and packed, no first one to begin at)
    const uint64_t first = g.seqs ? scan_places_before(g, 0) : 0, end = g.seqs ? scan_places_before(g, g.seqs) : 0;
    const float v = ordered_sum(g.part_p + first * n + e, n, end > first ? end - first : 0);
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
// states of a channel, LANES neighbouring lanes a channel, and walks through
// g.each_wave rows, the next row's loads on their way.  Bound by the states,
// read and written once.  WIDE: four states and their A, B and C load together
// and every channel has 4 LANES states; else any alignment and number.
template <class T, int LANES, bool WIDE>
__device__ __forceinline__ void scan_step_body(const fg_scan_step_kargs& g) {
    using raw = typename T::raw;
    struct __attribute__((aligned(4 * sizeof(raw)))) Raw4 {
        raw v[4];
    };
    const uint32_t per_row = (g.channels * LANES + 63) / 64;  // waves
    const uint32_t wave = uniform(blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64);
    const uint32_t row0 = wave / per_row * g.each_wave;
    if (row0 >= g.rows) return;
    const uint32_t rows = g.rows - row0 < g.each_wave ? g.rows - row0 : g.each_wave;
    const uint32_t id = wave % per_row * 64 + (threadIdx.x & 63), part = id % LANES, n0 = 4 * part;
    const bool valid = id / LANES < g.channels;  // the others take part in the sums of none
    const uint32_t ch = valid ? id / LANES : g.channels - 1;
    const uint32_t bc = ch / g.group_channels * g.states + n0;
    auto has = [&](int k) { return WIDE || n0 + k < g.states; };

    float a2[4];
    if constexpr (WIDE) {
        *(float4*)a2 = *(const float4*)(g.a + (uint64_t)ch * g.states + n0);
        each<4>([&](auto k) { a2[k] *= kLog2e; });
    } else {
        each<4>([&](auto k) { a2[k] = has(k) ? g.a[(uint64_t)ch * g.states + n0 + k] * kLog2e : 0.0f; });
    }
    const float bias = g.bias ? g.bias[ch] : 0.0f, skip = g.skip ? g.skip[ch] : 0.0f;

    struct Row {
        float h[4], b[4], c[4], u, delta, z;
        int64_t slot;
    };
    auto fetch = [&](Row& r, uint32_t row) {
        const int64_t slot = g.slots ? g.slots[row] : (int64_t)row;
        r.slot = slot >= 0 && (uint64_t)slot < g.state_rows ? slot : -1;
        auto in = [&](const fg_ssm_view& v, uint32_t i) { return T::up(((const raw*)v.p)[(int64_t)row * v.seq + i]); };
        auto four = [&](float(&x)[4], const fg_ssm_view& v) {
            if constexpr (WIDE) {
                const Raw4 q = *(const Raw4*)((const raw*)v.p + (int64_t)row * v.seq + bc);
                each<4>([&](auto k) { x[k] = T::up(q.v[k]); });
            } else {
                each<4>([&](auto k) { x[k] = has(k) ? in(v, bc + k) : 0.0f; });
            }
        };
        if (r.slot < 0) return;
        const float* from = g.state + ((uint64_t)r.slot * g.channels + ch) * g.states + n0;
        if constexpr (WIDE) *(float4*)r.h = *(const float4*)from;
        else each<4>([&](auto k) { r.h[k] = has(k) ? from[k] : 0.0f; });
        r.u = in(g.u, ch);
        r.delta = in(g.delta, ch);
        if (g.z.p) r.z = in(g.z, ch);
        four(r.b, g.b);
        four(r.c, g.c);
    };
    Row next;
    fetch(next, row0);
    for (uint32_t i = 0; i < rows; ++i) {
        const Row r = next;
        if (i + 1 < rows) fetch(next, row0 + i + 1);
        float y = 0.0f;
        if (r.slot >= 0) {
            const float x = r.delta + bias, dt = g.softplus ? softplus(x).value : x;
            float h[4];
            each<4>([&](auto k) {
                h[k] = fmaf(exp2_(dt * a2[k]), r.h[k], dt * r.u * r.b[k]);
                y = has(k) ? fmaf(r.c[k], h[k], y) : y;
            });
            float* to = g.state_out + ((uint64_t)r.slot * g.channels + ch) * g.states + n0;
            if constexpr (WIDE) {
                if (valid) *(float4*)to = {h[0], h[1], h[2], h[3]};
            } else {
                each<4>([&](auto k) {
                    if (valid && has(k)) to[k] = h[k];
                });
            }
            for (int m = 1; m < LANES; m *= 2) y += __shfl_xor(y, m);
            y = fmaf(skip, r.u, y);
            if (g.z.p) y *= r.z * sigmoid(r.z);
        }  // a row without a slot: zeros out
        if (valid && part == 0) ((raw*)g.out.p)[(int64_t)(row0 + i) * g.out.seq + ch] = T::down(y);
    }
}

}  // namespace ssm
}  // namespace fg
