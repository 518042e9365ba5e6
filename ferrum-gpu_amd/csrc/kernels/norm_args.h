/* norm_args.h -- kernel arguments and tile sizes of the residual norm and of
 * dropout (norm_rows.hpp), shared by the kernels and their host launchers
 * (norm_ops.cpp). */
#ifndef FG_NORM_ARGS_H
#define FG_NORM_ARGS_H

#include "ssm_args.h"

#define FG_NORM_THREADS(team) ((team) < 256 ? 256 : (team)) /* of a workgroup, whose teams have a row each */

typedef struct {
    fg_ssm_view x, residual, out, sum; /* .seq unused; may be null: residual, sum.  backward: x is the sum,
                                          residual its gradient, out the output's gradient */
    fg_ssm_view dx, dresidual;         /* backward; may be null */
    const float* weight;               /* null: 1 */
    float* scales;                     /* null: out has the rows' type; else e4m3 */
    float* part;                       /* backward: [workgroups][width], null: no weight's gradient */
    const int64_t* counter;            /* added to offset; may be null */
    uint64_t rows, seed, offset;
    uint32_t width, groups;            /* groups: scales of a row */
    uint32_t group_lanes;              /* lanes that share a scale; 0: a row does */
    uint32_t drop;                     /* kept where the 32 bits are at least this; 0: no dropout */
    uint32_t drop_all;
    uint32_t stream;                   /* store past the caches */
    float keep;                        /* 1 / (1 - p) */
    float eps, over_width;
} fg_norm_kargs;

typedef struct {
    const void* x;
    void* out;
    const int64_t* counter;
    uint64_t n, seed, offset;
    uint32_t drop, drop_all, stream;
    float keep;
} fg_dropout_kargs;

#endif
