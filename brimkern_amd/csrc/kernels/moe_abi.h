// What the kernels of a mixture-of-experts layer (moe_*.hip, quant_i8.hip, gemm_i8.hip) and the host runtime share: the launch
// arguments, and how assignments are divided over blocks.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "../../../include/brik.h"

// Blocks that route and sort: chunks of whole tokens, each with a row of counts per expert in the workspace.
#define BRIK_MOE_CHUNKS 256
#define BRIK_MOE_WS_BYTES (BRIK_MOE_CHUNKS * BRIK_MOE_EXPERTS * 4)

typedef struct brik_route_launch {
    brik_moe_route_args r;       // logit_stride filled in
    int32_t *counts;             // [chunks, experts]: assignments of a chunk by expert (more than one chunk)
    int32_t chunks, chunk;       // blocks, and tokens of each
} brik_route_launch;

typedef struct brik_spread_launch {
    const float *x, *y, *res, *weights;
    const int32_t *slot;
    float *out, *rows, *dweights;
    int32_t tokens, k, quads;    // quads: width / 4
} brik_spread_launch;

typedef struct brik_quant_launch {
    const float *x, *gate;
    int64_t x_stride, gate_stride;
    int8_t *codes;
    float *scales;
    int32_t M, K, gelu;
} brik_quant_launch;

typedef struct brik_i8_launch {
    const int8_t *x, *w;
    const float *xs, *ws, *res;
    float *y;
    int32_t *part;               // partial sums [split][M][N], where K is split over blocks
    const int32_t *src, *row_off;    // by experts
    int32_t M, K, N;             // M: rows of y
    int32_t E, k, x_rows;
    int32_t row_tiles, col_tiles, splits;
    int32_t steps;               // K steps of a split
} brik_i8_launch;
