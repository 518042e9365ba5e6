// ssm_conv.hpp -- the short causal convolution of each channel with its own W
// taps, over sequences (forward and backward) and for single tokens:
//
//   p[t,d] = bias[d] + sum_k w[d,k] x[t - (W-1) + k, d],  y = p sigmoid(p) or p
//
// Rows before a sequence come from its state (the W - 1 rows that preceded it)
// or are zero.  A thread takes V neighbouring channels through a run of
// tokens with the last W - 1 rows in registers, so each row is read once, plus
// W - 1 rows at the start of a run (backward: also at its end).
//
// Bound by memory where there are many rows, else by the chain of loads of one
// run.  Measured (4 taps, bfloat16): 8 x 2048 tokens x 4096 channels forward 48
// us over the same rows again and again (5.6 TB/s, partly from the Infinity
// Cache), 65 behind a backward pass (4.1 TB/s), backward 105 (3.8 TB/s) and 7 for
// the sums over the runs; 2 x 1001 x 2048 forward 8 us; a step of 256 rows x 4096
// channels 6 us.
// Widths of 4 / 5 / 6 / 7 / 8 taps, 8 x 2048 x 4096 backward with its sums, us:
// bfloat16 110 / 105 / 128 / 121 / 221, float32 168 / 169 / 176 / 186 / 191.  Eight
// taps take more than 256 registers backward (264 to 279), so that a SIMD has one wave.
#pragma once

#include "ssm_common.hpp"

namespace fg {
namespace ssm {

template <class T, int V>
struct Vec {
    using raw = typename T::raw;
    struct __attribute__((aligned(V * sizeof(raw)))) pack {
        raw v[V];
    };
    static __device__ __forceinline__ pack fetch(const void* p, int64_t at) { return *(const pack*)((const raw*)p + at); }
    static __device__ __forceinline__ void up(float (&x)[V], const pack& r) {
        each<V>([&](auto i) { x[i] = T::up(r.v[i]); });
    }
    static __device__ __forceinline__ void load(float (&x)[V], const void* p, int64_t at) { up(x, fetch(p, at)); }
    static __device__ __forceinline__ void store(void* p, int64_t at, const float (&x)[V]) {
        pack r;
        each<V>([&](auto i) { r.v[i] = T::down(x[i]); });
        *(pack*)((raw*)p + at) = r;
    }
};

// Where a thread works: its channels, its sequence and its run of tokens.  All
// but the channels are the wave's.
struct ConvPlace {
    uint32_t ch, seq, t0, len, run;
    int64_t start;
    bool any;   // there are such channels
    bool past;  // the run begins beyond the end of its sequence
};
template <int V>
__device__ __forceinline__ ConvPlace conv_place(const fg_conv_kargs& g) {
    ConvPlace p;
    const uint32_t wide = (g.channels / V + 63) / 64;  // waves over the channels
    const uint32_t wave = uniform(blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64);
    p.ch = (wave % wide * 64 + (threadIdx.x & 63)) * V;
    const uint32_t rest = wave / wide;
    p.run = rest % g.runs;
    p.seq = rest / g.runs;
    p.any = p.ch < g.channels && p.seq < g.seqs;
    p.start = 0;
    p.len = g.length;
    if (p.seq < g.seqs && g.offsets) {
        // offsets out of order or beyond the rows give shorter sequences, not accesses outside
        int64_t a = g.offsets[p.seq], b = g.offsets[p.seq + 1];
        const int64_t all = (int64_t)g.tokens;
        a = a < 0 ? 0 : a > all ? all : a;
        b = b < a ? a : b > all ? all : b;
        p.start = uniform(a);
        p.len = uniform((uint32_t)(b - a < (int64_t)g.length ? b - a : (int64_t)g.length));
    }
    p.t0 = p.run * g.run;
    p.past = p.run > 0 && p.t0 >= p.len;  // the first run is never past: it moves the states
    return p;
}

// The first place of packed sequence `seq` among the runs' parts.
__device__ __forceinline__ uint64_t conv_places_before(const fg_conv_kargs& g, uint32_t seq) {
    const int64_t a = g.offsets[seq], all = (int64_t)g.tokens;
    return (uint64_t)(a < 0 ? 0 : a > all ? all : a) / g.run + seq;
}

template <class T, int V, int W>
struct Conv {
    using Io = Vec<T, V>;
    using pack = typename Io::pack;
    // Rows that are loaded ahead: a wave alone waits a microsecond or two for each.
    static constexpr int U = FG_CONV_ROWS;
    static __device__ __forceinline__ int64_t at(const fg_ssm_view& v, const ConvPlace& p, int64_t t) {
        return (int64_t)p.seq * v.seq + (p.start + t) * v.row + p.ch;
    }
    static __device__ __forceinline__ int64_t state_at(const fg_conv_kargs& g, const ConvPlace& p, int j) {
        return ((int64_t)p.seq * (W - 1) + j) * g.channels + p.ch;
    }
    // The lane's V channels' weights, [channel][tap] in memory: V W adjacent
    // floats a lane.  Loaded straight, each instruction would touch a cache line
    // for each lane, more than the rows of a run do; so the wave loads its 64 V
    // W floats in order and turns them in LDS.
    static constexpr int FLOATS = V * W, STRIDE = FLOATS + 4;  // keeps lanes on banks of their own
    struct Turn {
        float v[V > 1 ? 4 * 64 * STRIDE : 4];
    };
    static __device__ __forceinline__ void weights(Turn& turn, const float* weight, const float* biases, uint32_t ch,
                                                   uint32_t channels, float (&w)[W][V], float (&bias)[V]) {
        const uint32_t lane = threadIdx.x & 63;
        const bool any = ch < channels;
        if constexpr (V > 1) {
            static_assert(FLOATS % 4 == 0, "moved four at a time");
            struct __attribute__((aligned(4))) Four {  // weights are aligned to floats only
                float v[4];
            };
            float* to = turn.v + threadIdx.x / 64 * (64 * STRIDE);
            const uint32_t first = ch - lane * V;  // the wave's first channel
            const uint64_t left = first < channels ? (uint64_t)(channels - first) * W : 0;
            Four f[FLOATS / 4];
            each<FLOATS / 4>([&](auto j) {
                const uint64_t e = 4 * (j * 64 + lane);
                if (e < left) f[j] = *(const Four*)(weight + (uint64_t)first * W + e);
            });
            each<FLOATS / 4>([&](auto j) {
                const uint32_t e = 4 * (j * 64 + lane);
                *(float4*)(to + e / FLOATS * STRIDE + e % FLOATS) = {f[j].v[0], f[j].v[1], f[j].v[2], f[j].v[3]};
            });
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            float x[FLOATS];
            each<FLOATS / 4>([&](auto j) { *(float4*)(x + 4 * j) = *(const float4*)(to + lane * STRIDE + 4 * j); });
            each<V>([&](auto i) {
                each<W>([&](auto k) { w[k][i] = x[i * W + k]; });
            });
        } else if (any) {
            each<W>([&](auto k) { w[k][0] = weight[(uint64_t)ch * W + k]; });
        }
        each<V>([&](auto i) { bias[i] = biases && any ? biases[ch + i] : 0.0f; });
    }
    // Row t of the sequence, or of the state before it.
    static __device__ __forceinline__ void row(float (&x)[V], const fg_conv_kargs& g, const ConvPlace& p, int64_t t) {
        if (t >= 0) Io::load(x, g.x.p, at(g.x, p, t));
        else if (g.initial) Io::load(x, g.initial, state_at(g, p, (int)t + W - 1));
        else each<V>([&](auto i) { x[i] = 0.0f; });
    }
    // U rows from row t on; beyond the last of `end` rows the last.
    static __device__ __forceinline__ void fetch(pack (&r)[U], const fg_ssm_view& v, const ConvPlace& p, uint32_t t,
                                                 uint32_t end) {
        each<U>([&](auto j) { r[j] = Io::fetch(v.p, at(v, p, t + j < end ? t + j : end - 1)); });
    }

    static __device__ __forceinline__ void forward(const fg_conv_kargs& g) {
        __shared__ __attribute__((aligned(16))) Turn turn;
        const ConvPlace p = conv_place<V>(g);
        if (p.past || p.seq >= g.seqs) return;
        const uint32_t t1 = p.len - p.t0 < g.run ? p.len : p.t0 + g.run;
        pack next[U];
        if (p.any && p.t0 < t1) fetch(next, g.x, p, p.t0, t1);
        float w[W][V], bias[V], x[W - 1 + U][V];
        weights(turn, g.weight, g.bias, p.ch, g.channels, w, bias);
        if (!p.any) return;
        each<W - 1>([&](auto k) { row(x[k], g, p, (int64_t)p.t0 - (W - 1) + k); });
        if (p.t0 == 0 && g.final) {
            // rows len - (W - 1) ... len - 1; all are read before any is
            // written, so final may be initial
            float f[W - 1][V];
            each<W - 1>([&](auto k) { row(f[k], g, p, (int64_t)p.len - (W - 1) + k); });
            each<W - 1>([&](auto k) { Io::store(g.final, state_at(g, p, k), f[k]); });
        }
        // ALL: U tokens; else the last ones of the run
        auto group = [&](auto all, uint32_t t) {
            float y[U][V];
            each<U>([&](auto j) {
                each<V>([&](auto i) {
                    float s = bias[i];
                    each<W>([&](auto k) { s = fmaf(w[k][i], x[j + k][i], s); });
                    const float act = s * sigmoid(s);
                    y[j][i] = g.silu ? act : s;
                });
            });
            each<U>([&](auto j) {
                if (decltype(all)::value || t + j < t1) Io::store(g.out.p, at(g.out, p, t + j), y[j]);
            });
        };
        for (uint32_t t = p.t0; t < t1; t += U) {
            each<U>([&](auto j) { Io::up(x[W - 1 + j], next[j]); });
            if (t + U < t1) fetch(next, g.x, p, t + U, t1);
            if (t + U <= t1) group(std::true_type{}, t);
            else group(std::false_type{}, t);
            each<W - 1>([&](auto k) {
                each<V>([&](auto i) { x[k][i] = x[k + U][i]; });
            });
        }
    }

    // dx[r] = sum_k w[k] dp[r + W - 1 - k], dp = dy act'(p): the run emits the
    // rows t0 ... t1 - 1 (the first run also those of the state before the
    // sequence) and works out p for W - 1 tokens beyond its end.
    static __device__ __forceinline__ void backward(const fg_conv_kargs& g) {
        __shared__ __attribute__((aligned(16))) Turn turn;
        const ConvPlace p = conv_place<V>(g);
        if (p.seq >= g.seqs) return;
        float gw[W][V], gbias[V];
        each<V>([&](auto i) {
            gbias[i] = 0.0f;
            each<W>([&](auto k) { gw[k][i] = 0.0f; });
        });
        if (!p.past) backward_run(g, p, turn, gw, gbias);
        if (!p.any) return;
        const auto put = [&](uint64_t k) {
            float* to = g.part + k * g.channels * (W + 1);
            each<V>([&](auto i) {
                each<W>([&](auto k) { to[(uint64_t)(p.ch + i) * W + k] = gw[k][i]; });
                to[(uint64_t)g.channels * W + p.ch + i] = gbias[i];
            });
        };
        if (!g.offsets) return put((uint64_t)p.seq * g.runs + p.run);
        // Packed: a place for every run's length of rows and one more for each
        // sequence, not for each sequence's longest.  What is left before the
        // next sequence's first is zeros; that sequence begins where this one
        // ends, or later where this one is cut.
        const uint64_t first = (uint64_t)p.start / g.run + p.seq, end = conv_places_before(g, p.seq + 1);
        uint64_t k = first + p.run;
        if (k < end) put(k);
        if (p.run + 1 < g.runs) return;
        each<V>([&](auto i) {
            gbias[i] = 0.0f;
            each<W>([&](auto k) { gw[k][i] = 0.0f; });
        });
        while (++k < end) put(k);
    }
    static __device__ __forceinline__ void backward_run(const fg_conv_kargs& g, const ConvPlace& p, Turn& turn,
                                                        float (&gw)[W][V], float (&gbias)[V]) {
        const uint32_t t1 = p.len - p.t0 < g.run ? p.len : p.t0 + g.run;
        const uint32_t end = t1 + W - 1, rows = end < p.len ? end : p.len;  // rows that exist
        pack nx[U], ny[U];
        auto ahead = [&](uint32_t t) {
            if (t < rows) {
                fetch(nx, g.x, p, t, rows);
                fetch(ny, g.out, p, t, rows);
            }
        };
        if (p.any) ahead(p.t0);
        float w[W][V], bias[V], x[W - 1 + U][V], dp[W - 1 + U][V];
        weights(turn, g.weight, g.bias, p.ch, g.channels, w, bias);
        if (!p.any) return;
        each<V>([&](auto i) {
            each<W - 1>([&](auto k) { dp[k][i] = 0.0f; });
        });
        each<W - 1>([&](auto k) { row(x[k], g, p, (int64_t)p.t0 - (W - 1) + k); });
        // INNER: U tokens and U emitted rows of the run's own, and none that
        // the final state took; else any, each looked at.
        auto group = [&](auto inner, uint32_t t) {
            constexpr bool INNER = decltype(inner)::value;
            float dx[U][V];
            each<U>([&](auto j) {
                float(&d)[V] = dp[W - 1 + j];
                const bool there = INNER || t + j < p.len, own = INNER || t + j < t1;
                each<V>([&](auto i) {
                    float s = bias[i];
                    each<W>([&](auto k) { s = fmaf(w[k][i], x[j + k][i], s); });
                    const float sg = sigmoid(s), slope = sg * fmaf(s, 1.0f - sg, 1.0f);
                    const float v = g.silu ? d[i] * slope : d[i];
                    d[i] = there ? v : 0.0f;
                    const float mine = own ? d[i] : 0.0f;
                    gbias[i] += mine;
                    each<W>([&](auto k) { gw[k][i] = own ? fmaf(mine, x[j + k][i], gw[k][i]) : gw[k][i]; });
                });
                each<V>([&](auto i) {
                    float s = 0.0f;
                    each<W>([&](auto k) { s = fmaf(w[W - 1 - k][i], dp[j + k][i], s); });
                    dx[j][i] = s;
                });
            });
            each<U>([&](auto j) {
                const int64_t r = (int64_t)t + j - (W - 1);  // its W outputs are all known now
                if constexpr (INNER) {
                    if (g.gx.p) Io::store(g.gx.p, at(g.gx, p, r), dx[j]);
                } else if (r < (int64_t)t1 && (r >= (int64_t)p.t0 || (r < 0 && g.ginitial && p.t0 == 0))) {
                    const int64_t f = r - ((int64_t)p.len - (W - 1));  // the row of the final state that r became
                    if (g.gfinal && f >= 0) {
                        float more[V];
                        Io::load(more, g.gfinal, state_at(g, p, (int)f));
                        each<V>([&](auto i) { dx[j][i] += more[i]; });
                    }
                    if (r < 0) Io::store(g.ginitial, state_at(g, p, (int)r + W - 1), dx[j]);
                    else if (g.gx.p) Io::store(g.gx.p, at(g.gx, p, r), dx[j]);
                }
            });
        };
        for (uint32_t t = p.t0; t < end; t += U) {
            each<U>([&](auto j) {
                Io::up(x[W - 1 + j], nx[j]);
                Io::up(dp[W - 1 + j], ny[j]);
            });
            ahead(t + U);
            if (t >= p.t0 + W - 1 && t + U <= t1) group(std::true_type{}, t);
            else group(std::false_type{}, t);
            each<W - 1>([&](auto k) {
                each<V>([&](auto i) { x[k][i] = x[k + U][i], dp[k][i] = dp[k + U][i]; });
            });
        }
    }

    // One token of each row, the W - 1 rows before it in a cache of slots.  A
    // wave takes g.each_wave rows, for which it loads the weights once.
    static __device__ __forceinline__ void step(const fg_conv_step_kargs& g) {
        __shared__ __attribute__((aligned(16))) Turn turn;
        const uint32_t wide = (g.channels / V + 63) / 64;
        const uint32_t wave = uniform(blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64);
        const uint32_t ch = (wave % wide * 64 + (threadIdx.x & 63)) * V;
        const uint32_t row0 = wave / wide * g.each_wave;
        if (row0 >= g.rows) return;
        const uint32_t rows = g.rows - row0 < g.each_wave ? g.rows - row0 : g.each_wave;
        struct Row {
            pack x[W];
            int64_t slot;
            __device__ __forceinline__ void fetch(const fg_conv_step_kargs& g, uint32_t row, uint32_t ch) {
                slot = g.slots ? g.slots[row] : (int64_t)row;
                if (slot < 0 || (uint64_t)slot >= g.state_rows) slot = -1;
                const int64_t at = (slot < 0 ? 0 : slot) * (W - 1) * (int64_t)g.channels + ch;
                if (slot >= 0) each<W - 1>([&](auto k) { x[k] = Io::fetch(g.state, at + k * (int64_t)g.channels); });
                x[W - 1] = Io::fetch(g.x.p, (int64_t)row * g.x.seq + ch);
            }
        } next;
        const bool any = ch < g.channels;
        if (any) next.fetch(g, row0, ch);
        float w[W][V], bias[V];
        weights(turn, g.weight, g.bias, ch, g.channels, w, bias);
        if (!any) return;
        for (uint32_t r = 0; r < rows; ++r) {
            const Row now = next;
            if (r + 1 < rows) next.fetch(g, row0 + r + 1, ch);
            float y[V];
            if (now.slot >= 0) {
                float x[W][V];
                each<W>([&](auto k) { Io::up(x[k], now.x[k]); });
                const int64_t at = now.slot * (W - 1) * (int64_t)g.channels + ch;
                each<W - 1>([&](auto k) { *(pack*)((typename T::raw*)g.state_out + at + k * (int64_t)g.channels) = now.x[k + 1]; });
                each<V>([&](auto i) {
                    float s = bias[i];
                    each<W>([&](auto k) { s = fmaf(w[k][i], x[k][i], s); });
                    y[i] = g.silu ? s * sigmoid(s) : s;
                });
            } else {  // a row without a slot: zeros out
                each<V>([&](auto i) { y[i] = 0.0f; });
            }
            Io::store(g.out.p, (int64_t)(row0 + r) * g.out.seq + ch, y);
        }
    }
};

// The parameters' gradients from the runs' parts, in a fixed order: four waves
// of a workgroup take 64 values and a quarter of the parts each.
__device__ __forceinline__ void conv_reduce(const fg_conv_kargs& g, uint32_t width, float* gweight, float* gbias) {
    __shared__ float parts[4][64];
    const uint64_t n = (uint64_t)g.channels * (width + 1);
    uint64_t start = 0, count = (uint64_t)g.seqs * g.runs;
    if (g.offsets) {
        const uint64_t end = conv_places_before(g, g.seqs);
        start = conv_places_before(g, 0);
        count = end > start ? end - start : 0;
    }
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t e = (uint64_t)blockIdx.x * 64 + lane, each_wave = (count + 3) / 4, first = wave * each_wave;
    float v = 0.0f;
    if (e < n && first < count)
        v = ordered_sum(g.part + (start + first) * n + e, n, count - first < each_wave ? count - first : each_wave);
    parts[wave][lane] = v;
    __syncthreads();
    if (wave > 0 || e >= n) return;
    v = (parts[0][lane] + parts[1][lane]) + (parts[2][lane] + parts[3][lane]);
    if (e < (uint64_t)g.channels * width) {
        if (gweight) gweight[e] = v;
    } else if (gbias) {
        gbias[e - (uint64_t)g.channels * width] = v;
    }
}

}  // namespace ssm
}  // namespace fg
