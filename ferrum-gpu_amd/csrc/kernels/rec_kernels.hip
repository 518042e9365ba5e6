// rec_kernels.hip -- the gfx950 code object of the gated linear recurrence
// (rec_scan.hpp).  Names: fg_rec_<...>_<element type>[_packed][_any]; the host
// composes them (rec_ops.cpp).
#include "rec_scan.hpp"

using namespace fg::rec;

// _any: for any stride, alignment and number of channels; _stream: rows past the caches.
#define FG_REC_ONE(NAME, T, SUFFIX, WIDE, PACKED, STREAM)                                                       \
    extern "C" __global__ __launch_bounds__(64 * FG_REC_WAVES) __attribute__((amdgpu_waves_per_eu(4)))          \
    void fg_rec_##NAME##SUFFIX(fg_rec_kargs g) {                                                               \
        Rec<T, WIDE, PACKED, STREAM>::forward(g);                                                 \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(64 * FG_REC_BACK_WAVES) __attribute__((amdgpu_waves_per_eu(3)))     \
    void fg_rec_back_##NAME##SUFFIX(fg_rec_kargs g) {                                                          \
        Rec<T, WIDE, PACKED, STREAM>::backward(g);                                           \
    }
#define FG_REC_STEP(NAME, T, V)                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void fg_rec_step_##NAME##_v##V(fg_rec_step_kargs g) { step<T, V>(g); }
#define FG_REC_TYPE(NAME, T)                                                                                    \
    FG_REC_ONE(NAME, T, , true, false, false)                                                                   \
    FG_REC_ONE(NAME, T, _stream, true, false, true)                                                             \
    FG_REC_ONE(NAME, T, _any, false, false, false)                                                              \
    FG_REC_ONE(NAME, T, _packed, true, true, false)                                                             \
    FG_REC_ONE(NAME, T, _packed_stream, true, true, true)                                                       \
    FG_REC_ONE(NAME, T, _packed_any, false, true, false)                                                        \
    FG_REC_STEP(NAME, T, 4)                                                                                     \
    FG_REC_STEP(NAME, T, 1)

extern "C" __global__ __launch_bounds__(1024) void fg_rec_reduce(fg_rec_kargs g) { reduce(g); }

// One code object, three builds of this file in parallel: FG_REC_F32, _BF16, _F16.
#if defined(FG_REC_F32)
FG_REC_TYPE(f32, fg::ssm::F32)
#elif defined(FG_REC_BF16)
FG_REC_TYPE(bf16, fg::ssm::BF16)
#elif defined(FG_REC_F16)
FG_REC_TYPE(f16, fg::ssm::F16)
#else
#error "build with FG_REC_F32, FG_REC_BF16 or FG_REC_F16"
#endif
