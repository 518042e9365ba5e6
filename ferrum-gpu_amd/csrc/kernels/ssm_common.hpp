// ssm_common.hpp -- element types, activations and lane exchanges of the
// sequence filters' kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "ssm_args.h"

namespace fg {
namespace ssm {

struct F32 {
    using raw = float;
    static __device__ __forceinline__ float up(raw x) { return x; }
    static __device__ __forceinline__ raw down(float x) { return x; }
};
struct BF16 {
    using raw = unsigned short;
    static __device__ __forceinline__ float up(raw x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }
};
struct F16 {
    using raw = unsigned short;
    static __device__ __forceinline__ float up(raw x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(unsigned short, (_Float16)x); }
};

template <int I>
struct Int {
    static constexpr int value = I;
    constexpr operator int() const { return I; }
};
// f(Int<0>), f(Int<1>), ... f(Int<N - 1>): a loop whose index is a constant.
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F&& f) {
    if constexpr (I < N) {
        f(Int<I>{});
        each<N, I + 1>(f);
    }
}

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// h 2^(2 x) + add, also where 2^(2 x) alone passes the type's range: by 2^x
// twice.  The largest number stands for an infinite 2^x, which takes no 0 to NaN.
__device__ __forceinline__ float times_exp2_twice(float h, float x, float add) {
    const float f = fminf(exp2_(x), 3.402823466e38f);
    return fmaf(h * f, f, add);
}

// 1 / (1 + exp(-x)).
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + exp2_(-kLog2e * x));
}

// log(1 + exp(x)) and its derivative 1 / (1 + exp(-x)), both from
// e = exp(-|x|): max(x, 0) + log1p(e), and (x >= 0 ? 1 : e) / (1 + e).
// log1p(e) = log(w) + (e - (w - 1)) / w for the rounded w = 1 + e: the second
// term is what the rounding took away, so time steps far below 1 keep their
// relative accuracy.
struct Softplus {
    float value, slope;
};
__device__ __forceinline__ Softplus softplus(float x) {
    const float e = exp2_(-kLog2e * fabsf(x));
    const float w = 1.0f + e, r = __builtin_amdgcn_rcpf(w);
    const float l = fmaf(e - (w - 1.0f), r, kLn2 * __builtin_amdgcn_logf(w));
    return {fmaxf(x, 0.0f) + l, x >= 0.0f ? r : e * r};
}

// A value that is the same in every lane, as a scalar: what is worked out from
// it (addresses, loop bounds) stays out of the vector registers.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)(((uint64_t)uniform((uint32_t)((uint64_t)x >> 32)) << 32) | uniform((uint32_t)x));
}

// A 32-bit offset that the compiler takes as new here: it then adds it to a
// uniform address within the load or store, where an offset extended to 64
// bits far above costs a vector addition for each of them.
__device__ __forceinline__ uint32_t fresh(uint32_t off) {
    asm volatile("" : "+v"(off));
    return off;
}

// Lane I of each row of 16 lanes to the whole row.  The compiler folds the
// move into a product that takes it.
template <int I>
__device__ __forceinline__ float row_bcast(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + I, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e;

// Two wait states behind the instructions that wrote v, which lane exchanges
// need.  The compiler keeps them by itself, but not for what a statement of
// assembly wrote.
__device__ __forceinline__ void settle(float& a) { asm("s_nop 1" : "+v"(a)); }
__device__ __forceinline__ void settle(float& a, float& b, float& c, float& d) {
    asm("s_nop 1" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
}

// Both values settled.
__device__ __forceinline__ float swap32_add(float a, float b) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(a), __float_as_int(b), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// p[0] + p[stride] + ... of n values, in this order of eight running sums.
__device__ __forceinline__ float ordered_sum(const float* p, uint64_t stride, uint64_t n) {
    float v[8] = {};
    uint64_t k = 0;
    for (; k + 8 <= n; k += 8) each<8>([&](auto j) { v[j] += p[(k + j) * stride]; });
    each<7>([&](auto j) {
        if (k + j < n) v[j] += p[(k + j) * stride];
    });
    return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

}  // namespace ssm
}  // namespace fg
