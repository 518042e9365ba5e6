/* rec_args.h -- kernel arguments and tile sizes of the gated linear recurrence
 * (rec_scan.hpp), shared by the kernels and their host launchers (rec_ops.cpp). */
#ifndef FG_REC_ARGS_H
#define FG_REC_ARGS_H

#include "ssm_args.h"

#define FG_REC_CHANNELS 64                        /* of a workgroup */
#define FG_REC_LANE_CHANNELS 2                    /* of a lane */
#define FG_REC_ROWS 2                             /* rows of lanes of a wave, each a segment of tokens */
#define FG_REC_WAVES 8                            /* of a workgroup, at most */
#define FG_REC_BACK_WAVES 4                       /* backward */
#define FG_REC_SEGMENT(bytes) ((bytes) == 2 ? 16 : 8) /* tokens of a lane, by its elements' bytes */
#define FG_REC_BACK_SEGMENT 8
#define FG_REC_AHEAD(segment) ((segment) / 2)     /* tokens whose rows a lane has on their way */
#define FG_REC_CHECK (FG_REC_ROWS * FG_REC_BACK_SEGMENT * FG_REC_BACK_WAVES) /* tokens between the states that a
                                                    forward pass leaves for its backward pass, at the
                                                    starts of waves of both */

/* Tiles whose pairs a workgroup composes itself, see rec_scan.hpp. */
#define FG_REC_GROUP 4
/* What a plan's tiles pass on: for each chain of a workgroup's channels the tickets drawn,
 * in a line of 64 bytes of its own, and behind all of them for each tile FG_REC_WORDS
 * 8-byte words of each channel. */
#define FG_REC_WORDS 3
#define FG_REC_CHAIN_BYTES(across, tiles) ((across) * (64 + 8ull * FG_REC_WORDS * FG_REC_CHANNELS * (tiles)))

typedef struct {
    fg_ssm_view x, ga, gx, out; /* backward: out is the output's gradient */
    fg_ssm_view dx, dga, dgx;   /* gradients; may be null */
    const float *decay, *bias_a, *bias_x, *initial;
    float* final;
    const float* gfinal;
    float *ginitial, *gdecay, *gbias_a, *gbias_x;
    const int32_t* offsets; /* packed: sequences + 1 of them; null: dense */
    float* check;           /* [chains][checks][channels], states before each FG_REC_CHECK tokens;
                               packed, behind them: [sequences][channels] initial states */
    float* part;            /* [parts][3][channels] */
    unsigned long long* chain; /* FG_REC_CHAIN_BYTES(chains * blocks, tiles); null where a chain is one tile */
    uint64_t over_tiles;    /* (2^64 - 1) / tiles */
    uint32_t over_across, over_blocks; /* (2^32 - 1) / (chains * blocks), / blocks */
    uint64_t tokens;        /* of a chain: a dense sequence's, packed those of all */
    uint64_t checks;        /* of a chain */
    uint64_t parts;
    uint32_t seqs, chains, channels;
    uint32_t blocks;        /* workgroups over the channels */
    uint32_t tiles;         /* of a chain */
    float rate;
} fg_rec_kargs;

/* What the kernels divide by (place_of), once blocks, chains and tiles are known. */
static inline void fg_rec_set_divisors(fg_rec_kargs* g) {
    const uint64_t across = (uint64_t)g->blocks * g->chains;
    g->over_tiles = ~0ull / g->tiles;
    g->over_across = across ? (uint32_t)(0xffffffffull / across) : 0;
    g->over_blocks = g->blocks ? 0xffffffffu / g->blocks : 0;
}

typedef struct {
    fg_ssm_view x, ga, gx, out; /* .seq: of rows; .row unused */
    const float *decay, *bias_a, *bias_x, *state;
    float* state_out;
    const int32_t* slots;
    uint64_t state_rows;
    uint32_t rows, channels;
    float rate;
} fg_rec_step_kargs;

#endif
