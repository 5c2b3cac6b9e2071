// How the calls of a mixture-of-experts layer and the 8-bit products are divided over the device. Plain functions of the sizes,
// apart from any context.
#pragma once
#include "kernels/moe_abi.h"

#include <algorithm>

namespace brik_plan {

// Chunks of a routing or sorting call: one block of all assignments where they are few, else as many as BRIK_MOE_CHUNKS.
inline void moe_chunks(brik_route_launch& a, int alone)
{
    const long n = (long)a.r.tokens * a.r.k;
    a.chunk = n <= alone ? std::max(1, a.r.tokens) : (int)std::max(16l, ((long)a.r.tokens + BRIK_MOE_CHUNKS - 1) / BRIK_MOE_CHUNKS);
    a.chunks = (a.r.tokens + a.chunk - 1) / a.chunk;
}

// Index of a kernel among those of 1, 2, 4, 8 and 16 experts a lane.
inline int moe_lanes(int E)
{
    int v = 0;
    while ((64 << v) < E) ++v;
    return v;
}

// Kernels of the 8-bit product: few rows (16 rows x 1, 2, 4 at once, by 16 x 1, 2 channels), tiles of dense products, tiles by
// experts.
enum I8Kind { I8_FEW, I8_TILE, I8_MOE };
struct I8Kernel {
    I8Kind kind;
    int bm, bn, threads;
    const char* name;
};
constexpr I8Kernel kI8Kernels[] = {
    {I8_FEW, 16, 16, 512, "brik_i8_few_1_1_8"},        {I8_FEW, 32, 16, 512, "brik_i8_few_2_1_8"},
    {I8_FEW, 64, 16, 512, "brik_i8_few_4_1_8"},        {I8_FEW, 16, 32, 512, "brik_i8_few_1_2_8"},
    {I8_FEW, 32, 32, 512, "brik_i8_few_2_2_8"},        {I8_FEW, 64, 32, 512, "brik_i8_few_4_2_8"},
    {I8_TILE, 256, 256, 256, "brik_i8_tile_256x256"},  {I8_TILE, 256, 128, 256, "brik_i8_tile_256x128"},
    {I8_TILE, 128, 128, 256, "brik_i8_tile_128x128"},  {I8_TILE, 64, 128, 256, "brik_i8_tile_64x128"},
    {I8_MOE, 256, 128, 256, "brik_i8_moe_256x128"},    {I8_MOE, 128, 128, 256, "brik_i8_moe_128x128"},
    {I8_MOE, 128, 128, 256, "brik_i8_moe_128x128k"},   {I8_MOE, 64, 128, 256, "brik_i8_moe_64x128"},
};
constexpr int kI8Count = sizeof(kI8Kernels) / sizeof(kI8Kernels[0]);

// The kernel of a call, and its grid in `a`. forced: 0, or 1 + index of a kernel (one of the other kind's tiles: as 0).
inline int i8_plan(brik_i8_launch& a, int forced)
{
    int t;
    const long rows = a.E ? (a.M + a.E - 1) / a.E : a.M;       // of an expert, in the mean
    const I8Kind other = a.E ? I8_TILE : I8_MOE;
    if (a.K == 0) t = a.E ? 13 : 9;                             // (a tile without steps: sums of 0)
    else if (forced && kI8Kernels[forced - 1].kind != other) t = forced - 1;
    else if (a.E) t = rows <= 8 ? 0 : rows <= 64 ? 13 : 11;
    else if (rows <= 64) t = rows <= 16 ? 0 : rows <= 32 ? 1 : 2;
    else t = a.M >= 2048 && (long)a.M * a.N >= 32l << 20 ? 6 : 8;
    const I8Kernel& g = kI8Kernels[t];
    a.col_tiles = (a.N + g.bn - 1) / g.bn;
    a.splits = 1;
    a.steps = (a.K + 63) / 64;
    if (g.kind == I8_FEW) a.row_tiles = std::max(1, a.E);
    else a.row_tiles = (int)((a.M + g.bm - 1) / g.bm + (a.E ? std::min(a.E, a.M) : 0));
    return t;
}

}  // namespace brik_plan
