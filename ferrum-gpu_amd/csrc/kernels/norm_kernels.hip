// norm_kernels.hip -- the gfx950 code object of the residual norm and of dropout
// (norm_rows.hpp).  Names: fg_norm_[back_]<element type>_c<chunks>_t<team>; the host
// composes them (norm_ops.cpp).
#include "norm_rows.hpp"

using namespace fg::norm;

// _any: for widths that are not whole chunks.
#define FG_NORM_FORM(NAME, T, C, TEAM, SUFFIX, EVEN)                                                            \
    extern "C" __global__ __launch_bounds__(FG_NORM_THREADS(TEAM))                                                  \
    void fg_norm_##NAME##_c##C##_t##TEAM##SUFFIX(fg_norm_kargs g) {                                            \
        Rows<T, C, TEAM, EVEN>::forward(g);                                                                    \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(FG_NORM_THREADS(TEAM))                                                  \
    void fg_norm_back_##NAME##_c##C##_t##TEAM##SUFFIX(fg_norm_kargs g) {                                       \
        Rows<T, C, TEAM, EVEN>::backward(g);                                                                   \
    }
#define FG_NORM_ONE(NAME, T, C, TEAM) FG_NORM_FORM(NAME, T, C, TEAM, , true) FG_NORM_FORM(NAME, T, C, TEAM, _any, false)
#define FG_NORM_TYPE(NAME, T)                                                                                   \
    FG_NORM_ONE(NAME, T, 1, 64)                                                                                 \
    FG_NORM_ONE(NAME, T, 2, 64)                                                                                 \
    FG_NORM_ONE(NAME, T, 1, 256)                                                                                \
    FG_NORM_ONE(NAME, T, 1, 512)                                                                                \
    FG_NORM_ONE(NAME, T, 1, 1024)                                                                               \
    FG_NORM_ONE(NAME, T, 2, 1024)                                                                               \
    FG_NORM_ONE(NAME, T, 0, 1024)                                                                               \
    extern "C" __global__ __launch_bounds__(256) void fg_dropout_##NAME(fg_dropout_kargs g) { dropout<T>(g); }

extern "C" __global__ __launch_bounds__(1024) void fg_norm_reduce(const float* part, float* to, uint32_t width,
                                                                 uint32_t parts) {
    reduce(part, to, width, parts);
}

// One code object, three builds of this file in parallel: FG_NORM_F32, _BF16, _F16.
#if defined(FG_NORM_F32)
FG_NORM_TYPE(f32, fg::ssm::F32)
#elif defined(FG_NORM_BF16)
FG_NORM_TYPE(bf16, fg::ssm::BF16)
#elif defined(FG_NORM_F16)
FG_NORM_TYPE(f16, fg::ssm::F16)
#else
#error "build with FG_NORM_F32, FG_NORM_BF16 or FG_NORM_F16"
#endif
