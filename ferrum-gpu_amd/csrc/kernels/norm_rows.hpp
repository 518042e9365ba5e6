// norm_rows.hpp -- the root-mean-square norm of rows with what stands before it
// on a residual stream, its gradient, and dropout on its own:
//
//   v = dropout(x) + residual,  s = 1 / sqrt(mean(v^2) + eps),  out = v s weight
//   sum = v, rounded to the rows' type
//
// out in 8 bits (e4m3): out / scale, scale = max |out| / 448 over a row or a group of
// its elements.  With w = v weight and its largest m, both are w 448 / m and m s /
// 448, so that one pass finds all that the other needs.
//
// Backward, from the stored sum u: with s of u and g = grad_out weight,
//   dv = s (g - u s^2 mean(g u)) + grad_sum,  dx = dropout(dv),  dresidual = dv
//   dweight = sum over rows of grad_out u s
//
// A team of threads takes a row, each thread chunks of 16 bytes of it: the row is
// read once and stays in registers, the weight too, and the next row is loaded while
// one is summed and written.  Rows that do not fit are read again (C = 0).  The weight's
// gradient is summed by each team over its rows and then over the teams, in a fixed order.
//
// out is taken of the unrounded v; the backward pass, which reads the stored sum, is the
// gradient at what was stored.
//
// Bound by memory.  Measured (8192 rows x 4096, bfloat16, us; a copy of as many bytes would take):
// with the residual to 8 bits 45 (35), with dropout and the residual 50 (40), backward 70 (50) and 5
// for the weight's gradient; dropout alone 22 (20).  Dropout is 18 vector instructions of an
// element, most of them the generator's 64-bit products, backward 24 others: 36 us of the 70.
// Teams of 256 with two chunks a thread 51, without the next row's loads 53, with ordinary stores 57.
//
// Dropout keeps element e (row-major) where 32 bits are at least p 2^32: half e % 2 of
// the seed's splitmix64 number offset + e / 2 (fill.hpp), so no mask is stored.
#pragma once

#include "norm_args.h"
#include "ssm_common.hpp"

#include "fill.hpp"

namespace fg {
namespace norm {

using namespace ssm;

constexpr float kMost = 448.0f;            // e4m3's largest
constexpr float kLeast = 7.888609e-31f;    // 2^-100: what 448 / m is taken of at least

typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t HalfWords __attribute__((ext_vector_type(2), aligned(1)));

// A store past the caches.  The statements around it keep the compiler from making one
// ordinary store of this one and of that on the branch's other side.
#define FG_PAST_THE_CACHES(TYPE, v, to)                                \
    do {                                                               \
        asm volatile("; past the caches");                             \
        __builtin_nontemporal_store(__builtin_bit_cast(TYPE, v), (TYPE*)(to)); \
        asm volatile("; past the caches");                             \
    } while (0)

// Chunks of 16 bytes at any address of their elements: the GPU's loads and stores take them.
// EVEN: all of them are whole.
template <class T, bool EVEN>
struct Chunk {
    using raw = typename T::raw;
    static constexpr int E = 16 / sizeof(raw);
    struct __attribute__((packed, aligned(sizeof(raw)))) Raw {
        raw v[E];
    };
    struct __attribute__((packed, aligned(4))) Floats {
        float v[E];
    };
    struct __attribute__((packed, aligned(1))) Bytes {
        uint32_t v[E / 4];
    };
    // n of E elements, 0 for the others.
    static __device__ __forceinline__ Raw load(const void* p, int64_t at, uint32_t n) {
        const raw* from = (const raw*)p + at;
        Raw r;
        if (EVEN || n >= E) return *(const Raw*)from;
        each<E>([&](auto i) { r.v[i] = i < n ? from[i] : raw(0); });
        return r;
    }
    static __device__ __forceinline__ void store(void* p, int64_t at, uint32_t n, const float (&x)[E],
                                                 uint32_t stream) {
        raw* to = (raw*)p + at;
        Raw r;
        each<E>([&](auto i) { r.v[i] = T::down(x[i]); });
        if (EVEN || n >= E) {
            if (stream) FG_PAST_THE_CACHES(Words, r, to);
            else *(Raw*)to = r;
        } else {
            each<E>([&](auto i) {
                if (i < n) to[i] = r.v[i];
            });
        }
    }
    // Whole chunks: not for n = 0.
    static __device__ __forceinline__ void floats(float (&x)[E], const float* p, uint32_t at, uint32_t n) {
        if (!p) {
            each<E>([&](auto i) { x[i] = 1.0f; });
        } else if (EVEN || n >= E) {
            const Floats f = *(const Floats*)(p + at);
            each<E>([&](auto i) { x[i] = f.v[i]; });
        } else {
            each<E>([&](auto i) { x[i] = i < n ? p[at + i] : 0.0f; });
        }
    }
    static __device__ __forceinline__ void store8(void* p, int64_t at, uint32_t n, const float (&x)[E], uint32_t stream) {
        uint8_t* to = (uint8_t*)p + at;
        Bytes b;
        each<E / 4>([&](auto i) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
            b.v[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
        });
        if (EVEN || n >= E) {
            if constexpr (E == 8) {
                if (stream) FG_PAST_THE_CACHES(HalfWords, b, to);
                else *(Bytes*)to = b;
            } else {
                *(Bytes*)to = b;
            }
        } else {
            each<E>([&](auto i) {
                if (i < n) to[i] = (uint8_t)(b.v[i / 4] >> (8 * (i % 4)));
            });
        }
    }
    // x where it is kept times 1 / (1 - p), else 0, of elements e, e + 1, ...
    static __device__ __forceinline__ void drop(float (&x)[E], uint64_t seed, uint64_t first, uint64_t e, uint32_t drop,
                                                uint32_t all, float keep) {
        const auto one = [&](float& v, uint32_t bits) { v = !all && bits >= drop ? v * keep : 0.0f; };
        if (e & 1) {
            each<E>([&](auto i) {
                const uint64_t z = splitmix64_at(seed, first + (e + i) / 2);
                one(x[i], (uint32_t)((e + i) & 1 ? z >> 32 : z));
            });
        } else {
            const uint64_t state = seed + (first + e / 2 + 1) * kSplitmixStep;
            each<E / 2>([&](auto i) {
                const uint64_t z = splitmix64_mix(state + i * kSplitmixStep);
                one(x[2 * i], (uint32_t)z);
                one(x[2 * i + 1], (uint32_t)(z >> 32));
            });
        }
    }
};

// Two sums, or a sum and a largest value, over a team's threads.
template <int TEAM, bool MAX>
__device__ __forceinline__ void over_team(float& a, float& b, float2 (&lds)[TEAM / 64]) {
    each<6>([&](auto i) {
        a += __shfl_xor(a, 1 << i);
        const float o = __shfl_xor(b, 1 << i);
        b = MAX ? fmaxf(b, o) : b + o;
    });
    if constexpr (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x % TEAM / 64] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
        each<TEAM / 64>([&](auto w) {
            const float2 v = lds[w];
            a += v.x;
            b = MAX ? fmaxf(b, v.y) : b + v.y;
        });
    }
}

// C: chunks of a thread; 0: any number of them, read again.
template <class T, int C, int TEAM, bool EVEN>
struct Rows {
    using Io = Chunk<T, EVEN>;
    using Raw = typename Io::Raw;
    static constexpr int E = Io::E, TEAMS = FG_NORM_THREADS(TEAM) / TEAM, KEPT = C ? C : 1;

    static __device__ __forceinline__ uint32_t count(const fg_norm_kargs& g, uint32_t col) {
        return col >= g.width ? 0 : g.width - col;
    }
    template <class F>
    static __device__ __forceinline__ void chunks(const fg_norm_kargs& g, F&& f) {
        const uint32_t first = (threadIdx.x % TEAM) * E;
        if constexpr (C > 0) {
            each<C>([&](auto k) {
                const uint32_t col = first + k * (TEAM * E);
                f(k, col, count(g, col));
            });
        } else {
            // every thread of the team passes as often: lanes exchange values within
            for (uint32_t at = 0; at < g.width; at += TEAM * E) f(Int<0>{}, at + first, count(g, at + first));
        }
    }

    // A chunk of x and of the residual, and their sum.
    struct Pair {
        Raw x, residual;
    };
    static __device__ __forceinline__ Pair fetch(const fg_norm_kargs& g, uint64_t row, uint32_t col, uint32_t n) {
        Pair p{};
        p.x = Io::load(g.x.p, (int64_t)row * g.x.row + col, n);
        if (g.residual.p) p.residual = Io::load(g.residual.p, (int64_t)row * g.residual.row + col, n);
        return p;
    }
    static __device__ __forceinline__ void value(const fg_norm_kargs& g, const Pair& p, uint64_t row, uint32_t col,
                                                 uint64_t numbers, float (&v)[E]) {
        each<E>([&](auto i) { v[i] = T::up(p.x.v[i]); });
        if (g.drop) Io::drop(v, g.seed, numbers, row * g.width + col, g.drop, g.drop_all, g.keep);
        if (g.residual.p) each<E>([&](auto i) { v[i] += T::up(p.residual.v[i]); });
    }

    static __device__ __forceinline__ void forward(const fg_norm_kargs& g) {
        __shared__ float2 lds[2][TEAM / 64];
        const uint64_t numbers = g.offset + (g.counter ? (uint64_t)*g.counter : 0);
        const uint64_t stride = (uint64_t)gridDim.x * TEAMS;
        uint64_t row = (uint64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
        float w[KEPT][E], v[KEPT][E];
        Pair next[KEPT];  // the next row, on its way while this one is worked on
        if constexpr (C > 0) {
            chunks(g, [&](auto k, uint32_t col, uint32_t n) {
                if (row < g.rows && n) next[k] = fetch(g, row, col, n);
            });
            // A team may have more threads than the row has chunks: those load the weight's first one and use
            // nothing of it (8192 x 4096 to 8 bits 44.6 us so, 45.5 with a branch around the load).
            chunks(g, [&](auto k, uint32_t col, uint32_t n) { Io::floats(w[k], g.weight, n ? col : 0, n); });
        }
        uint32_t turn = 0;
        for (uint64_t at = (uint64_t)blockIdx.x * TEAMS; at < g.rows; at += stride, row += stride, turn ^= 1) {
            const bool some = row < g.rows;  // a whole team's
            float squares = 0.0f, most = 0.0f;
            chunks(g, [&](auto k, uint32_t col, uint32_t n) {
                each<E>([&](auto i) { v[k][i] = 0.0f; });
                if (!some || !n) return;
                if constexpr (C == 0) {
                    Io::floats(w[k], g.weight, col, n);
                    next[k] = fetch(g, row, col, n);
                }
                value(g, next[k], row, col, numbers, v[k]);
                if (C > 0 && row + stride < g.rows) next[k] = fetch(g, row + stride, col, n);
                each<E>([&](auto i) {
                    if (!EVEN && i >= n) v[k][i] = 0.0f;  // a dropped place beyond the row holds nothing else
                    squares = fmaf(v[k][i], v[k][i], squares);
                    most = fmaxf(most, fabsf(v[k][i] * w[k][i]));
                });
                if (g.sum.p && C) Io::store(g.sum.p, (int64_t)row * g.sum.row + col, n, v[k], g.stream);
            });
            over_team<TEAM, true>(squares, most, lds[turn]);
            const float s = __builtin_amdgcn_rsqf(fmaf(squares, g.over_width, g.eps));
            // s of scales: of an infinite sum it is 0, with which a group beside the infinity, and a row whose
            // squares pass the range, would be read back as 0
            const float known = squares < __builtin_inff() ? s : __builtin_nanf("");
            if (g.scales && !g.group_lanes && some && threadIdx.x % TEAM == 0)
                g.scales[row] = most == 0.0f ? 0.0f * known : fmaxf(most, kLeast) * known * (1.0f / kMost);
            chunks(g, [&](auto k, uint32_t col, uint32_t n) {
                if (C == 0) {
                    each<E>([&](auto i) { v[k][i] = 0.0f; });
                    if (some && n) {
                        Io::floats(w[k], g.weight, col, n);
                        value(g, fetch(g, row, col, n), row, col, numbers, v[k]);
                        if (g.sum.p) Io::store(g.sum.p, (int64_t)row * g.sum.row + col, n, v[k], g.stream);
                    }
                }
                float y[E];
                if (!g.scales) {
                    each<E>([&](auto i) { y[i] = v[k][i] * s * w[k][i]; });
                    if (some && n) Io::store(g.out.p, (int64_t)row * g.out.row + col, n, y, g.stream);
                    return;
                }
                float m = most;
                if (g.group_lanes) {
                    m = 0.0f;
                    each<E>([&](auto i) { m = fmaxf(m, EVEN || i < n ? fabsf(v[k][i] * w[k][i]) : 0.0f); });
                    for (uint32_t far = 1; far < g.group_lanes; far *= 2) m = fmaxf(m, __shfl_xor(m, far));
                    if (some && n && (threadIdx.x & (g.group_lanes - 1)) == 0)
                        g.scales[row * g.groups + col / (g.group_lanes * E)] =
                            m == 0.0f ? 0.0f * known : fmaxf(m, kLeast) * known * (1.0f / kMost);
                }
                const float up = kMost / fmaxf(m, kLeast);
                each<E>([&](auto i) { y[i] = v[k][i] * w[k][i] * up; });
                if (some && n) Io::store8(g.out.p, (int64_t)row * g.out.row + col, n, y, g.stream);
            });
        }
    }

    static __device__ __forceinline__ void backward(const fg_norm_kargs& g) {
        __shared__ float2 lds[2][TEAM / 64];
        const uint64_t numbers = g.offset + (g.counter ? (uint64_t)*g.counter : 0);
        float w[KEPT][E], dw[KEPT][E], u[KEPT][E], dy[KEPT][E];
        float* part = g.part ? g.part + (uint64_t)(blockIdx.x * TEAMS + threadIdx.x / TEAM) * g.width : nullptr;
        chunks(g, [&](auto k, uint32_t col, uint32_t n) {
            if (C > 0 && (!EVEN || n)) Io::floats(w[k], g.weight, col, n);
            each<E>([&](auto i) { dw[k][i] = 0.0f; });
            if (C == 0 && part) each<E>([&](auto i) { if (i < n) part[col + i] = 0.0f; });
        });
        const uint64_t stride = (uint64_t)gridDim.x * TEAMS;
        uint64_t row = (uint64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
        Raw next[KEPT][3];  // the next row of the sum and of both gradients
        const auto fetch = [&](uint64_t r, int k, uint32_t col, uint32_t n) {
            next[k][0] = Io::load(g.x.p, (int64_t)r * g.x.row + col, n);
            next[k][1] = Io::load(g.out.p, (int64_t)r * g.out.row + col, n);
            if (g.residual.p) next[k][2] = Io::load(g.residual.p, (int64_t)r * g.residual.row + col, n);
        };
        Raw later[KEPT];  // this row's gradient of the sum
        const auto take = [&](auto k, uint32_t col, uint32_t n) {
            if constexpr (C == 0) {
                Io::floats(w[k], g.weight, col, n);
                fetch(row, k, col, n);
            }
            each<E>([&](auto i) { u[k][i] = T::up(next[k][0].v[i]), dy[k][i] = T::up(next[k][1].v[i]); });
            later[k] = next[k][2];
        };
        if constexpr (C > 0) {
            chunks(g, [&](auto k, uint32_t col, uint32_t n) {
                if (row < g.rows && n) fetch(row, k, col, n);
            });
        }
        uint32_t turn = 0;
        for (uint64_t at = (uint64_t)blockIdx.x * TEAMS; at < g.rows; at += stride, row += stride, turn ^= 1) {
            const bool some = row < g.rows;
            float squares = 0.0f, along = 0.0f;
            chunks(g, [&](auto k, uint32_t col, uint32_t n) {
                if (!some || !n) return;
                take(k, col, n);
                if (C > 0 && row + stride < g.rows) fetch(row + stride, k, col, n);
                each<E>([&](auto i) {
                    squares = fmaf(u[k][i], u[k][i], squares);
                    if (EVEN || i < n) along = fmaf(dy[k][i] * w[k][i], u[k][i], along);
                });
            });
            over_team<TEAM, false>(squares, along, lds[turn]);
            const float s = __builtin_amdgcn_rsqf(fmaf(squares, g.over_width, g.eps));
            const float back = along * g.over_width * s * s;
            chunks(g, [&](auto k, uint32_t col, uint32_t n) {
                if (!some || !n) return;
                if constexpr (C == 0) take(k, col, n);
                float dv[E];
                each<E>([&](auto i) { dv[i] = s * fmaf(-u[k][i], back, dy[k][i] * w[k][i]); });
                if (g.residual.p) each<E>([&](auto i) { dv[i] += T::up(later[k].v[i]); });
                if (g.dresidual.p) Io::store(g.dresidual.p, (int64_t)row * g.dresidual.row + col, n, dv, g.stream);
                if (g.dx.p) {
                    if (g.drop) Io::drop(dv, g.seed, numbers, row * g.width + col, g.drop, g.drop_all, g.keep);
                    Io::store(g.dx.p, (int64_t)row * g.dx.row + col, n, dv, g.stream);
                }
                if constexpr (C > 0) {
                    each<E>([&](auto i) { dw[k][i] = fmaf(dy[k][i], u[k][i] * s, dw[k][i]); });
                } else if (part) {
                    each<E>([&](auto i) {
                        if (i < n) part[col + i] = fmaf(dy[k][i], u[k][i] * s, part[col + i]);
                    });
                }
            });
        }
        if (C > 0 && part) {
            chunks(g, [&](auto k, uint32_t col, uint32_t n) {
                each<E>([&](auto i) { if (i < n) part[col + i] = dw[k][i]; });
            });
        }
    }
};

// The weight's gradient from the teams' parts: 64 columns of a workgroup, whose
// waves share the parts.
__device__ __forceinline__ void reduce(const float* part, float* to, uint32_t width, uint32_t parts) {
    __shared__ float sums[16][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const uint64_t col = (uint64_t)blockIdx.x * 64 + lane;
    const uint32_t each_wave = (parts + waves - 1) / waves, a = min(parts, wave * each_wave), b = min(parts, a + each_wave);
    sums[wave][lane] = col < width ? ordered_sum(part + (uint64_t)a * width + col, width, b - a) : 0.0f;
    __syncthreads();
    if (wave == 0 && col < width) {
        float v = 0.0f;
        for (uint32_t k = 0; k < waves; ++k) v += sums[k][lane];
        to[col] = v;
    }
}

template <class T>
__device__ __forceinline__ void dropout(const fg_dropout_kargs& g) {
    using Io = Chunk<T, false>;
    constexpr int E = Io::E;
    const uint64_t numbers = g.offset + (g.counter ? (uint64_t)*g.counter : 0);
    const uint64_t step = (uint64_t)gridDim.x * blockDim.x * E;
    for (uint64_t at = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) * E; at < g.n; at += step) {
        const uint32_t n = g.n - at < E ? (uint32_t)(g.n - at) : E;
        const typename Io::Raw x = Io::load(g.x, (int64_t)at, n);
        float v[E];
        each<E>([&](auto i) { v[i] = T::up(x.v[i]); });
        if (g.drop) Io::drop(v, g.seed, numbers, at, g.drop, g.drop_all, g.keep);
        Io::store(g.out, (int64_t)at, n, v, g.stream);
    }
}

}  // namespace norm
}  // namespace fg
