// Stands in for <hip/hip_runtime.h> where a test builds a kernel's header for the
// CPU: a launch runs one workgroup after another, each thread as a context of its own
// that goes on to the next barrier or lane exchange before another one runs.  Which
// wave goes first is the caller's choice (launch(), last), so that what only the order of
// waves keeps right shows, and arrays that end where nothing is mapped (Guarded) show
// every access behind them.
#pragma once

#include <sys/mman.h>
#include <ucontext.h>
#include <unistd.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <type_traits>
#include <vector>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline __attribute__((always_inline))
#define __launch_bounds__(...)
#define __shared__ static

struct Index {
    uint32_t x;
};
inline Index threadIdx, blockIdx, blockDim, gridDim;

struct float2 {
    float x, y;
};
struct alignas(16) float4 {
    float x, y, z, w;
};
inline float2 make_float2(float x, float y) { return {x, y}; }
inline uint32_t __float_as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }
inline float __uint_as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
inline int __float_as_int(float x) { return __builtin_bit_cast(int, x); }
inline float __int_as_float(int x) { return __builtin_bit_cast(float, x); }
inline uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)((uint64_t)a * b >> 32); }
inline uint64_t __umul64hi(uint64_t a, uint64_t b) { return (uint64_t)((unsigned __int128)a * b >> 64); }
inline int __popcll(unsigned long long x) { return __builtin_popcountll(x); }
template <class A, class B>
std::common_type_t<A, B> min(A a, B b) {
    return std::min<std::common_type_t<A, B>>(a, b);
}
template <class A, class B>
std::common_type_t<A, B> max(A a, B b) {
    return std::max<std::common_type_t<A, B>>(a, b);
}

namespace on_cpu {

struct Thread {
    ucontext_t context;
    std::vector<char> stack;
    bool ended = true;
    uint32_t exchanges = 0, barriers = 0;
};
inline std::vector<Thread> threads;
inline ucontext_t scheduler;
inline uint32_t current, alive;
inline std::function<void()> body;
// of each wave: lanes that have come to its n-th exchange, and what they brought to the last two
struct Wave {
    std::vector<uint32_t> come;
    uint64_t brought[2][64];
};
inline std::vector<Wave> waves;
inline std::vector<uint32_t> at_barrier;

inline void pause() { swapcontext(&threads[current].context, &scheduler); }
inline uint32_t lanes_of(uint32_t wave) { return min(64u, blockDim.x - 64 * wave); }

// What all lanes of the wave bring, to be read before the exchange after the next one.
inline const uint64_t* exchange(uint64_t mine) {
    Wave& w = waves[threadIdx.x / 64];
    const uint32_t lane = threadIdx.x % 64, n = threads[current].exchanges++, all = lanes_of(threadIdx.x / 64);
    if (w.come.size() <= n) w.come.resize(n + 1);
    w.brought[n % 2][lane] = mine;
    ++w.come[n];
    while (w.come[n] < all) pause();
    return w.brought[n % 2];
}
inline void barrier() {
    const uint32_t n = threads[current].barriers++;
    if (at_barrier.size() <= n) at_barrier.resize(n + 1);
    ++at_barrier[n];
    while (at_barrier[n] < blockDim.x) pause();
}
inline void entry() {
    body();
    threads[current].ended = true;
    --alive;
    swapcontext(&threads[current].context, &scheduler);
}

// Workgroups one after another; last: the last wave goes first.  between(b) runs ahead of workgroup b.
template <class F>
void launch(uint32_t blocks, uint32_t size, bool last, F&& kernel, const std::function<void(uint32_t)>& between = {}) {
    body = kernel;
    if (threads.size() < size) threads.resize(size);
    gridDim.x = blocks;
    blockDim.x = size;
    for (uint32_t b = 0; b < blocks; ++b) {
        if (between) between(b);
        blockIdx.x = b;
        waves.assign((size + 63) / 64, {});
        at_barrier.clear();
        for (uint32_t t = 0; t < size; ++t) {
            Thread& th = threads[t];
            th.stack.resize(96 << 10);
            getcontext(&th.context);
            th.context.uc_stack.ss_sp = th.stack.data();
            th.context.uc_stack.ss_size = th.stack.size();
            th.context.uc_link = nullptr;
            makecontext(&th.context, entry, 0);
            th.ended = false;
            th.exchanges = th.barriers = 0;
        }
        alive = size;
        for (uint32_t turns = 0; alive; ++turns) {
            if (turns == 100000) {
                fprintf(stderr, "workgroup %u: threads wait for one another for good\n", b);
                exit(3);
            }
            for (uint32_t k = 0; k < size; ++k) {
                const uint32_t t = last ? (size - 1 - k) / 64 * 64 + k % 64 : k;
                if (t >= size || threads[t].ended) continue;
                current = threadIdx.x = t;
                swapcontext(&scheduler, &threads[t].context);
            }
        }
    }
}

// n elements, the last one's end where nothing is mapped; bytes of 0xff (NaN) until written.
template <class T>
class Guarded {
public:
    explicit Guarded(size_t n) : n_(n) {
        const size_t page = sysconf(_SC_PAGESIZE), bytes = (n * sizeof(T) + page - 1) / page * page;
        mapped_ = bytes + 2 * page;
        base_ = (char*)mmap(nullptr, mapped_, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
        if (base_ == MAP_FAILED || (bytes && mprotect(base_ + page, bytes, PROT_READ | PROT_WRITE))) abort();
        p_ = (T*)(base_ + page + bytes - n * sizeof(T));
        if (bytes) memset(base_ + page, 0xff, bytes);
    }
    Guarded(const Guarded&) = delete;
    ~Guarded() { munmap(base_, mapped_); }
    // an array of one size begins its page, others do not: bytes before it must hold what they held
    bool before_kept() const {
        for (const char* c = base_ + sysconf(_SC_PAGESIZE); c < (const char*)p_; ++c)
            if (*c != (char)0xff) return false;
        return true;
    }
    T* data() { return p_; }
    T& operator[](size_t i) { return p_[i]; }
    size_t size() const { return n_; }

private:
    char* base_;
    T* p_;
    size_t n_, mapped_;
};

template <class T>
uint64_t bits(T v) {
    uint64_t b = 0;
    memcpy(&b, &v, sizeof(T));
    return b;
}
template <class T>
T value(uint64_t b) {
    T v;
    memcpy(&v, &b, sizeof(T));
    return v;
}

// e4m3's numbers by their bits; to the nearest, ties to even, as the instruction rounds.
inline float e4m3(uint32_t code) {
    const int e = code >> 3 & 15, m = code & 7;
    const float v = e ? std::ldexp(1.0f + m / 8.0f, e - 7) : std::ldexp(m / 8.0f, -6);
    return code & 0x80 ? -v : v;
}
inline uint32_t to_e4m3(float x) {
    const uint32_t sign = __float_as_uint(x) >> 31 << 7;
    const float a = std::fabs(x);
    if (!(a <= 464.0f)) return sign | 0x7f;
    uint32_t lo = 0, hi = 0x7e;  // neighbours, in the end
    while (hi - lo > 1) (e4m3((lo + hi) / 2) <= a ? lo : hi) = (lo + hi) / 2;
    const float below = a - e4m3(lo), above = e4m3(hi) - a;
    return sign | (below < above || (below == above && lo % 2 == 0) ? lo : hi);
}

}  // namespace on_cpu

template <class T>
T __shfl_xor(T v, int mask) {
    return on_cpu::value<T>(on_cpu::exchange(on_cpu::bits(v))[threadIdx.x % 64 ^ mask]);
}
inline unsigned long long __ballot(int p) {
    const uint64_t* all = on_cpu::exchange(p != 0);
    unsigned long long b = 0;
    for (uint32_t i = 0; i < on_cpu::lanes_of(threadIdx.x / 64); ++i) b |= (unsigned long long)all[i] << i;
    return b;
}
inline int __all(int p) {
    const uint32_t lanes = on_cpu::lanes_of(threadIdx.x / 64);
    return __ballot(p) == (lanes == 64 ? ~0ull : (1ull << lanes) - 1);
}
inline void __syncthreads() { on_cpu::barrier(); }

// What a value that is the same in all lanes is taken by.
inline uint32_t cpu_readfirstlane(uint32_t x) { return x; }
inline uint32_t cpu_cvt_pk_fp8(float a, float b, int old, bool high) {
    const uint32_t two = on_cpu::to_e4m3(a) | on_cpu::to_e4m3(b) << 8;
    return high ? ((uint32_t)old & 0xffff) | two << 16 : ((uint32_t)old & 0xffff0000) | two;
}
// Tickets are drawn in the workgroups' order and each ends before the next begins, so nobody waits.
inline void cpu_waits() {
    fprintf(stderr, "workgroup %u waits for one that has ended\n", blockIdx.x);
    exit(3);
}
struct CpuPair {
    int v[2];
    int operator[](int i) const { return v[i]; }
};
inline CpuPair cpu_not_here() { abort(); }

#define __builtin_amdgcn_readfirstlane cpu_readfirstlane
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#define __builtin_amdgcn_rsqf(x) (1.0f / std::sqrt(x))
#define __builtin_amdgcn_sqrtf(x) std::sqrt(x)
#define __builtin_amdgcn_exp2f(x) std::exp2(x)
#define __builtin_amdgcn_logf(x) std::log2(x)
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_s_sleep(x) cpu_waits()
#define __builtin_amdgcn_cvt_pk_fp8_f32 cpu_cvt_pk_fp8
#define __builtin_amdgcn_update_dpp(...) cpu_not_here()[0]
#define __builtin_amdgcn_permlane32_swap(...) cpu_not_here()
#define __HIP_MEMORY_SCOPE_AGENT 0
#define __hip_atomic_fetch_add(p, v, order, scope) __atomic_fetch_add(p, v, order)
#define __hip_atomic_store(p, v, order, scope) __atomic_store_n(p, v, order)
#define __hip_atomic_load(p, order, scope) __atomic_load_n(p, order)
