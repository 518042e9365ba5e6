/* ssm_args.h -- kernel arguments and tile sizes of the sequence filters
 * (ssm_conv.hpp, ssm_scan.hpp), shared by the kernels and their host
 * launchers (ssm_ops.cpp). */
#ifndef FG_SSM_ARGS_H
#define FG_SSM_ARGS_H

#include <stdint.h>

#define FG_SSM_SEGMENT 16         /* tokens that the scan works through at a time; the
                                    states before each segment are what a forward
                                    pass leaves for its backward pass */
#define FG_SSM_MAX_STATES 64
#define FG_CONV_MAX_WIDTH 8
#define FG_CONV_ROWS 4            /* rows that the convolution loads at a time */

/* A scan's workgroup has FG_SSM_BLOCKS(W) blocks of 16 channels with W waves
 * each; 4 W rows of 16 lanes share a channel's states. */
#define FG_SSM_BLOCKS(w) ((w) == 1 ? 4 : 2)

/* Rows of a [sequences, tokens, n] array, strides in elements. */
typedef struct {
    void* p;
    int64_t seq, row;
} fg_ssm_view;

typedef struct {
    fg_ssm_view u, delta, b, c, z, out;      /* z.p null: no gate */
    fg_ssm_view gu, gdelta, gb, gc, gz, gout; /* gradients; out.p and those may be null */
    const float *a, *skip, *bias, *initial;
    float* final;
    const float* gfinal;
    float *ga, *gskip, *gbias, *ginitial;
    const int32_t* offsets; /* packed: sequences + 1 of them; null: dense */
    float* check;           /* states at segment starts */
    float* carry;           /* [places + sequences][blocks of 16 channels][16 * 4 W S]: what a chunk adds;
                               behind the chunks' places: each sequence's initial states */
    float* carry_dt;        /* [places][blocks of 16 channels][16]: its summed time steps */
    float* part_bc;         /* [channel blocks of a group][tokens][groups][2][states] */
    float* part_p;          /* [places][channels * (states + 2)] */
    uint64_t tokens;        /* packed: of all sequences */
    uint64_t places;        /* of chunks, over all sequences */
    uint32_t seqs, length, channels, states, groups;
    uint32_t group_channels, group_blocks; /* channels of a group, workgroups over them */
    uint32_t chunks, chunk_len;            /* chunk_len: a multiple of the segment */
    uint32_t check_segs;                   /* dense: segments of a sequence */
    uint32_t softplus;
} fg_scan_kargs;

typedef struct {
    fg_ssm_view u, delta, b, c, z, out; /* .seq: of rows; .row unused */
    const float *a, *skip, *bias, *state;
    float* state_out;
    const int32_t* slots;
    uint64_t state_rows;
    uint32_t rows, channels, states, groups, group_channels;
    uint32_t softplus;
    uint32_t each_wave; /* rows of a wave */
} fg_scan_step_kargs;

typedef struct {
    fg_ssm_view x, out;       /* backward: x and the output's gradient */
    fg_ssm_view gx;
    const float *weight, *bias;
    const void* initial;      /* [sequences][width - 1][channels] */
    void* final;
    const void* gfinal;
    void* ginitial;
    float* part;              /* [parts][channels * (width + 1)] */
    const int32_t* offsets;
    uint64_t tokens;
    uint32_t seqs, length, channels, run; /* run: tokens of a thread */
    uint32_t runs;                        /* runs of the longest sequence */
    uint32_t silu;
} fg_conv_kargs;

typedef struct {
    fg_ssm_view x, out;
    const float *weight, *bias;
    const void* state;
    void* state_out;
    const int32_t* slots;
    uint64_t state_rows;
    uint32_t rows, channels, silu;
    uint32_t each_wave; /* rows of a wave */
} fg_conv_step_kargs;

#endif
