// ssm_kernels.hip -- the gfx950 code object of the sequence filters: the short
// causal convolution (ssm_conv.hpp) and the selective scan (ssm_scan.hpp).
//
// Names: fg_<operator>_<element type>[_...]; the host composes them
// (ssm_ops.cpp).  Built like the FFT code object, by ferrum-gpu_amd/csrc/Makefile.
#include "ssm_conv.hpp"
#include "ssm_scan.hpp"

using namespace fg::ssm;

// S: states of a lane, W: waves that share a channel's states; _any: for any
// alignment, and channels with fewer than 4 S W states.  The backward kernel holds two states
// and decays for each of its 16 S, so S = 4 is held to two waves per SIMD.  That takes
// all 256 registers and leaves a few in scratch memory: 27 of a lane (_any 65), 2 (26)
// on two waves, none (4) on four.
#define FG_SCAN_KERNEL(NAME, T, S, W, WIDE, CALL)                                                               \
    extern "C" __global__ __launch_bounds__((Scan<T, S, W, WIDE>::THREADS))                                     \
    __attribute__((amdgpu_waves_per_eu(2, 3))) void NAME(fg_scan_kargs g) {                                    \
        Scan<T, S, W, WIDE>::CALL(g);                                                                           \
    }
#define FG_SCAN_ONE(NAME, T, S, W, SUFFIX, WIDE)                                                                \
    FG_SCAN_KERNEL(fg_scan_local_##NAME##_s##S##w##W##SUFFIX, T, S, W, WIDE, template forward<true>)            \
    FG_SCAN_KERNEL(fg_scan_##NAME##_s##S##w##W##SUFFIX, T, S, W, WIDE, template forward<false>)                 \
    FG_SCAN_KERNEL(fg_scan_back_local_##NAME##_s##S##w##W##SUFFIX, T, S, W, WIDE, template backward<true>)      \
    extern "C" __global__ __launch_bounds__((Scan<T, S, W, WIDE>::THREADS))                                     \
    __attribute__((amdgpu_waves_per_eu(2))) void fg_scan_back_##NAME##_s##S##w##W##SUFFIX(fg_scan_kargs g) {   \
        Scan<T, S, W, WIDE>::template backward<false>(g);                                                       \
    }
#define FG_SCAN(NAME, T, S, W) FG_SCAN_ONE(NAME, T, S, W, , true) FG_SCAN_ONE(NAME, T, S, W, _any, false)

// W taps, V channels of a thread: eight (16-bit rows, up to four taps, not
// backward: more would not fit the registers), four, or one for any stride and
// alignment.
#define FG_CONV_KERNEL(NAME, T, W, V, CALL, ARGS)                                                               \
    extern "C" __global__ __launch_bounds__(256) void NAME##_w##W##_v##V(ARGS g) { Conv<T, V, W>::CALL(g); }
#define FG_CONV_FORWARD(NAME, T, W, V)                                                                          \
    FG_CONV_KERNEL(fg_conv_##NAME, T, W, V, forward, fg_conv_kargs)                                             \
    FG_CONV_KERNEL(fg_conv_step_##NAME, T, W, V, step, fg_conv_step_kargs)
#define FG_CONV_BACK(NAME, T, W, V) FG_CONV_KERNEL(fg_conv_back_##NAME, T, W, V, backward, fg_conv_kargs)
#define FG_CONV(NAME, T, W)                                                                                     \
    FG_CONV_FORWARD(NAME, T, W, 4)                                                                              \
    FG_CONV_FORWARD(NAME, T, W, 1)                                                                              \
    FG_CONV_BACK(NAME, T, W, 4)                                                                                 \
    FG_CONV_BACK(NAME, T, W, 1)
#define FG_CONV_EIGHT(NAME, T) FG_CONV_FORWARD(NAME, T, 2, 8) FG_CONV_FORWARD(NAME, T, 3, 8) FG_CONV_FORWARD(NAME, T, 4, 8)

// L: lanes of a channel, four states each; _any as for the scan.
#define FG_SCAN_STEP(NAME, T, L)                                                                                \
    extern "C" __global__ __launch_bounds__(256) void fg_scan_step_##NAME##_l##L(fg_scan_step_kargs g) {        \
        scan_step_body<T, L, true>(g);                                                                         \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void fg_scan_step_##NAME##_l##L##_any(fg_scan_step_kargs g) {  \
        scan_step_body<T, L, false>(g);                                                                        \
    }

#define FG_SSM_TYPE(NAME, T)                                                                                    \
    FG_SCAN(NAME, T, 1, 1)                                                                                      \
    FG_SCAN(NAME, T, 2, 1)                                                                                      \
    FG_SCAN(NAME, T, 4, 1)                                                                                      \
    FG_SCAN(NAME, T, 4, 2)                                                                                      \
    FG_SCAN(NAME, T, 4, 4)                                                                                      \
    FG_CONV(NAME, T, 2)                                                                                         \
    FG_CONV(NAME, T, 3)                                                                                         \
    FG_CONV(NAME, T, 4)                                                                                         \
    FG_CONV(NAME, T, 5)                                                                                         \
    FG_CONV(NAME, T, 6)                                                                                         \
    FG_CONV(NAME, T, 7)                                                                                         \
    FG_CONV(NAME, T, 8)                                                                                         \
    extern "C" __global__ __launch_bounds__(256) void fg_scan_reduce_bc_##NAME(fg_scan_kargs g) {                \
        scan_reduce_bc<T>(g);                                                                                  \
    }                                                                                                          \
    FG_SCAN_STEP(NAME, T, 1)                                                                                    \
    FG_SCAN_STEP(NAME, T, 2)                                                                                    \
    FG_SCAN_STEP(NAME, T, 4)                                                                                    \
    FG_SCAN_STEP(NAME, T, 8)                                                                                    \
    FG_SCAN_STEP(NAME, T, 16)

// The sums that are float32 whatever the rows' type, in each code object.
extern "C" __global__ __launch_bounds__(256) void fg_scan_reduce_p(fg_scan_kargs g) { scan_reduce_p(g); }
extern "C" __global__ __launch_bounds__(256) void fg_conv_reduce(fg_conv_kargs g, uint32_t width, float* gweight,
                                                                float* gbias) {
    conv_reduce(g, width, gweight, gbias);
}

// One code object, three builds of this file in parallel: FG_SSM_F32, _BF16, _F16.
#if defined(FG_SSM_F32)
FG_SSM_TYPE(f32, F32)
#elif defined(FG_SSM_BF16)
FG_SSM_TYPE(bf16, BF16)
FG_CONV_EIGHT(bf16, BF16)
#elif defined(FG_SSM_F16)
FG_SSM_TYPE(f16, F16)
FG_CONV_EIGHT(f16, F16)
#else
#error "build with FG_SSM_F32, FG_SSM_BF16 or FG_SSM_F16"
#endif
