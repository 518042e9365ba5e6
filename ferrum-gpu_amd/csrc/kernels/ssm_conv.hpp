// ssm_conv.hpp -- the short causal convolution of each channel with its own W
// taps, over sequences (forward and backward) and for single tokens:
//
//   p[t,d] = bias[d] + sum_k w[d,k] x[t - (W-1) + k, d],  y = p sigmoid(p) or p
//
// Rows before a sequence come from its state (the W - 1 rows that preceded it)
// or are zero.  A thread takes V neighbouring channels through a run of
// tokens with the last W - 1 rows in registers, so each row is read once, plus
// W - 1 rows at the start of a run.
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
    static __device__ __forceinline__ void load(float (&x)[V], const void* p, int64_t at) {
        const pack r = *(const pack*)((const raw*)p + at);
        each<V>([&](auto i) { x[i] = T::up(r.v[i]); });
    }
    static __device__ __forceinline__ void store(void* p, int64_t at, const float (&x)[V]) {
        pack r;
        each<V>([&](auto i) { r.v[i] = T::down(x[i]); });
        *(pack*)((raw*)p + at) = r;
    }
};

// Where a thread works: its channels, its sequence and its run of tokens.
struct ConvPlace {
    uint32_t ch, seq, t0, len;
    int64_t start;
    bool any;
};
template <int V>
__device__ __forceinline__ ConvPlace conv_place(const fg_conv_kargs& g) {
    ConvPlace p;
    const uint32_t wide = (g.channels / V + 63) / 64;  // waves over the channels
    const uint64_t wave = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) / 64;
    p.ch = (uint32_t)(wave % wide * 64 + (threadIdx.x & 63)) * V;
    const uint64_t rest = wave / wide;
    const uint32_t run = (uint32_t)(rest % g.runs);
    p.seq = (uint32_t)(rest / g.runs);
    p.any = p.ch < g.channels && p.seq < g.seqs;
    p.start = 0;
    p.len = g.length;
    if (p.any && g.offsets) {
        // offsets out of order or beyond the rows give shorter sequences, not accesses outside
        int64_t a = g.offsets[p.seq], b = g.offsets[p.seq + 1];
        const int64_t all = (int64_t)g.tokens;
        a = a < 0 ? 0 : a > all ? all : a;
        b = b < a ? a : b > all ? all : b;
        p.start = a;
        p.len = (uint32_t)(b - a < (int64_t)g.length ? b - a : (int64_t)g.length);
    }
    const uint64_t first = (uint64_t)run * g.run;
    if (first > 0 && first >= p.len) p.any = false;  // the first run stays: it moves the states
    p.t0 = (uint32_t)first;
    return p;
}

template <class T, int V, int W>
struct Conv {
    using Io = Vec<T, V>;
    static __device__ __forceinline__ int64_t at(const fg_ssm_view& v, const ConvPlace& p, int64_t t) {
        return (int64_t)p.seq * v.seq + (p.start + t) * v.row + p.ch;
    }
    static __device__ __forceinline__ int64_t state_at(const fg_conv_kargs& g, const ConvPlace& p, int j) {
        return ((int64_t)p.seq * (W - 1) + j) * g.channels + p.ch;
    }
    static __device__ __forceinline__ void weights(const fg_conv_kargs& g, const ConvPlace& p, float (&w)[W][V],
                                                   float (&bias)[V]) {
        each<V>([&](auto i) {
            each<W>([&](auto k) { w[k][i] = g.weight[(uint64_t)(p.ch + i) * W + k]; });
            bias[i] = g.bias ? g.bias[p.ch + i] : 0.0f;
        });
    }
    // Row t of the sequence, or of the state before it.
    static __device__ __forceinline__ void row(float (&x)[V], const fg_conv_kargs& g, const ConvPlace& p, int64_t t) {
        if (t >= 0) Io::load(x, g.x.p, at(g.x, p, t));
        else if (g.initial) Io::load(x, g.initial, state_at(g, p, (int)t + W - 1));
        else each<V>([&](auto i) { x[i] = 0.0f; });
    }

    static __device__ __forceinline__ void forward(const fg_conv_kargs& g) {
        const ConvPlace p = conv_place<V>(g);
        if (!p.any) return;
        float w[W][V], bias[V], x[W][V];
        weights(g, p, w, bias);
        each<W - 1>([&](auto k) { row(x[k], g, p, (int64_t)p.t0 - (W - 1) + k); });
        const uint32_t t1 = p.len - p.t0 < g.run ? p.len : p.t0 + g.run;
        if (p.t0 == 0 && g.final) {
            // rows len - (W - 1) ... len - 1; all are read before any is
            // written, so final may be initial
            float f[W - 1][V];
            each<W - 1>([&](auto k) { row(f[k], g, p, (int64_t)p.len - (W - 1) + k); });
            each<W - 1>([&](auto k) { Io::store(g.final, state_at(g, p, k), f[k]); });
        }
        for (uint32_t t = p.t0; t < t1; ++t) {
            Io::load(x[W - 1], g.x.p, at(g.x, p, t));
            float y[V];
            each<V>([&](auto i) {
                float s = bias[i];
                each<W>([&](auto k) { s = fmaf(w[k][i], x[k][i], s); });
                y[i] = g.silu ? s * sigmoid(s) : s;
            });
            Io::store(g.out.p, at(g.out, p, t), y);
            each<W - 1>([&](auto k) {
                each<V>([&](auto i) { x[k][i] = x[k + 1][i]; });
            });
        }
    }

    // dx[r] = sum_k w[k] dp[r + W - 1 - k], dp = dy act'(p): the run emits the
    // rows t0 ... t1 - 1 (the first run also those of the state before the
    // sequence) and works out p for W - 1 tokens beyond its end.
    static __device__ __forceinline__ void backward(const fg_conv_kargs& g) {
        const ConvPlace p = conv_place<V>(g);
        if (!p.any) return;
        float w[W][V], bias[V], x[W][V], dp[W][V], gw[W][V], gbias[V];
        weights(g, p, w, bias);
        each<V>([&](auto i) {
            gbias[i] = 0.0f;
            each<W>([&](auto k) { gw[k][i] = dp[k][i] = 0.0f; });
        });
        each<W - 1>([&](auto k) { row(x[k], g, p, (int64_t)p.t0 - (W - 1) + k); });
        const uint32_t t1 = p.len - p.t0 < g.run ? p.len : p.t0 + g.run;
        const int64_t end = (int64_t)t1 + W - 1;
        for (int64_t t = p.t0; t < end; ++t) {
            // dp[W - 1] of token t
            each<V>([&](auto i) { x[W - 1][i] = dp[W - 1][i] = 0.0f; });
            if (t < p.len) {
                float dy[V];
                Io::load(x[W - 1], g.x.p, at(g.x, p, t));
                Io::load(dy, g.out.p, at(g.out, p, t));
                each<V>([&](auto i) {
                    float s = bias[i];
                    each<W>([&](auto k) { s = fmaf(w[k][i], x[k][i], s); });
                    if (g.silu) {
                        const float sg = sigmoid(s);
                        dy[i] *= sg * fmaf(s, 1.0f - sg, 1.0f);
                    }
                    dp[W - 1][i] = dy[i];
                    if (t < t1) {
                        gbias[i] += dy[i];
                        each<W>([&](auto k) { gw[k][i] = fmaf(dy[i], x[k][i], gw[k][i]); });
                    }
                });
            }
            const int64_t r = t - (W - 1);  // its W outputs are all known now
            if (r >= (int64_t)p.t0 || (r < 0 && g.ginitial && p.t0 == 0)) {
                float dx[V];
                each<V>([&](auto i) {
                    float s = 0.0f;
                    each<W>([&](auto k) { s = fmaf(w[W - 1 - k][i], dp[k][i], s); });
                    dx[i] = s;
                });
                const int64_t j = r - ((int64_t)p.len - (W - 1));  // the row of the final state that r became
                if (g.gfinal && j >= 0) {
                    float f[V];
                    Io::load(f, g.gfinal, state_at(g, p, (int)j));
                    each<V>([&](auto i) { dx[i] += f[i]; });
                }
                if (r < 0) Io::store(g.ginitial, state_at(g, p, (int)r + W - 1), dx);
                else if (g.gx.p) Io::store(g.gx.p, at(g.gx, p, r), dx);
            }
            each<W - 1>([&](auto k) {
                each<V>([&](auto i) { x[k][i] = x[k + 1][i], dp[k][i] = dp[k + 1][i]; });
            });
        }
        float* to = g.part + ((uint64_t)p.seq * g.runs + p.t0 / g.run) * g.channels * (W + 1);
        each<V>([&](auto i) {
            each<W>([&](auto k) { to[(uint64_t)(p.ch + i) * W + k] = gw[k][i]; });
            to[(uint64_t)g.channels * W + p.ch + i] = gbias[i];
        });
    }

    // One token of each row, the W - 1 rows before it in a cache of slots.
    static __device__ __forceinline__ void step(const fg_conv_step_kargs& g) {
        const uint32_t wide = (g.channels / V + 63) / 64;
        const uint64_t wave = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) / 64;
        const uint32_t ch = (uint32_t)(wave % wide * 64 + (threadIdx.x & 63)) * V;
        const uint64_t row = wave / wide;
        if (ch >= g.channels || row >= g.rows) return;
        const int64_t slot = g.slots ? g.slots[row] : (int64_t)row;
        float y[V];
        if (slot >= 0 && (uint64_t)slot < g.state_rows) {
            float x[W][V];
            const int64_t at = slot * (W - 1) * (int64_t)g.channels + ch;
            each<W - 1>([&](auto k) { Io::load(x[k], g.state, at + k * (int64_t)g.channels); });
            Io::load(x[W - 1], g.x.p, (int64_t)row * g.x.seq + ch);
            each<W - 1>([&](auto k) { Io::store(g.state_out, at + k * (int64_t)g.channels, x[k + 1]); });
            each<V>([&](auto i) {
                float s = g.bias ? g.bias[ch + i] : 0.0f;
                each<W>([&](auto k) { s = fmaf(g.weight[(uint64_t)(ch + i) * W + k], x[k][i], s); });
                y[i] = g.silu ? s * sigmoid(s) : s;
            });
        } else {  // a row without a slot: zeros out
            each<V>([&](auto i) { y[i] = 0.0f; });
        }
        Io::store(g.out.p, (int64_t)row * g.out.seq + ch, y);
    }
};

// The parameters' gradients from the runs' parts, in the order of the runs.
// Runs beyond the end of a packed sequence have written none.
__device__ __forceinline__ void conv_reduce(const fg_conv_kargs& g, uint32_t width, float* gweight, float* gbias) {
    const uint64_t n = (uint64_t)g.channels * (width + 1);
    const uint64_t e = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= n) return;
    float v = 0.0f;
    for (uint32_t s = 0; s < g.seqs; ++s) {
        uint32_t len = g.length;
        if (g.offsets) {
            int64_t a = g.offsets[s], b = g.offsets[s + 1];
            const int64_t all = (int64_t)g.tokens;
            a = a < 0 ? 0 : a > all ? all : a;
            b = b < a ? a : b > all ? all : b;
            len = (uint32_t)(b - a < (int64_t)g.length ? b - a : (int64_t)g.length);
        }
        const uint32_t runs = len ? (len - 1) / g.run + 1 : 0;
        for (uint32_t k = 0; k < runs; ++k) v += g.part[((uint64_t)s * g.runs + k) * n + e];
    }
    if (e < (uint64_t)g.channels * width) {
        if (gweight) gweight[e] = v;
    } else if (gbias) {
        gbias[e - (uint64_t)g.channels * width] = v;
    }
}

}  // namespace ssm
}  // namespace fg
