// How the calls of a mixture-of-experts layer and the 8-bit products are divided over the device. Plain functions of the sizes,
// apart from any context.
#pragma once
#include "kernels/moe_abi.h"

#include <algorithm>
#include <cmath>

namespace brik_plan {

// Chunks of a routing or sorting call: one block of all assignments where they are few (`alone`), else as many as BRIK_MOE_CHUNKS.
inline void moe_chunks(brik_route_launch& a, int alone)
{
    const long n = (long)a.r.tokens * a.r.k;
    a.chunk = n <= alone ? std::max(1, a.r.tokens) : (int)std::max(64l, ((long)a.r.tokens + BRIK_MOE_CHUNKS - 1) / BRIK_MOE_CHUNKS);
    a.chunks = (a.r.tokens + a.chunk - 1) / a.chunk;
}

// Index of a kernel among those of 1, 2, 4, 8 and 16 experts a lane of a team of `lanes`.
inline int moe_lanes(int E, int lanes)
{
    int v = 0;
    while ((lanes << v) < E) ++v;
    return v;
}

// Index of a routing kernel: by teams of 16 lanes, then by whole waves.
inline int moe_route(int E, int k) { return E <= 256 && k <= 16 ? moe_lanes(E, 16) : 5 + moe_lanes(E, 64); }

// Kernels of the 8-bit product: few rows (16 rows x 1 or 2 at once, 16 channels a block), tiles of dense products, tiles by experts.
enum I8Kind { I8_FEW, I8_TILE, I8_MOE };
struct I8Kernel {
    I8Kind kind;
    int bm, bn, threads;
    const char* name;
};
constexpr I8Kernel kI8Kernels[] = {
    {I8_FEW, 16, 16, 256, "brik_i8_few_1_4"},         {I8_FEW, 16, 16, 512, "brik_i8_few_1_8"},
    {I8_FEW, 32, 16, 512, "brik_i8_few_2_8"},         {I8_FEW, 16, 16, 1024, "brik_i8_few_1_16"},
    {I8_FEW, 32, 16, 1024, "brik_i8_few_2_16"},       {I8_TILE, 256, 256, 256, "brik_i8_tile_256x256"},
    {I8_TILE, 256, 128, 256, "brik_i8_tile_256x128"}, {I8_TILE, 128, 128, 256, "brik_i8_tile_128x128"},
    {I8_TILE, 64, 128, 256, "brik_i8_tile_64x128"},   {I8_MOE, 256, 256, 256, "brik_i8_moe_256x256"},
    {I8_MOE, 128, 128, 256, "brik_i8_moe_128x128"},   {I8_MOE, 64, 128, 256, "brik_i8_moe_64x128"},
};
constexpr int kI8Count = sizeof(kI8Kernels) / sizeof(kI8Kernels[0]);
constexpr int kI8Few = 0, kI8Tiles = 5, kI8Moe = 9;

// A tile's times, fitted to measurements (us): `start` for a block (twice where a CU has two), then for a step of 128 of K from `alone`, where few blocks run, to
// `full` with one on every CU (the matrix cores' clock falls under load), and `two` where CUs have two, which share its paths.
struct I8Times {
    double start, alone, full, two;
    bool square;                 // how the step's time grows with the blocks
};
constexpr I8Times kI8Times[4] = {{11.6, 1.0, 1.7, 0, true}, {7.1, 0.61, 1.0, 0, false}, {4.6, 0.37, 0.66, 0.95, false}, {3.7, 0.27, 0.45, 0.64, true}};
constexpr int kI8CUs = 256;

inline double i8_tile_us(const I8Times& t, double blocks, double steps)
{
    const double slots = t.two > 0 ? 2 * kI8CUs : kI8CUs, rounds = std::floor(blocks / slots), rest = blocks - rounds * slots, x = rest / kI8CUs;
    const double whole = t.two > 0 ? 2 * t.start + steps * t.two : t.start + steps * t.full;
    return rounds * whole + (rest == 0 ? 0 : x > 1 ? whole : t.start + steps * (t.alone + (t.full - t.alone) * (t.square ? x * x : x)));
}

// Up to 64 rows by the few-row kernel: its launch, the waves' steps of 64 of K, w from memory, x from the L2 for every block, and more
// waves than the device holds.
inline double i8_few_us(long M, long K, long N, int waves)
{
    const long steps = (K + 63) / 64, blocks = (N + 15) / 16;
    return 2.9 + 0.28 * ((steps + waves - 1) / waves) + N * (double)K / 7e6 + (double)M * K * blocks / 11e6 + (M > 16 ? 0.8 * ((M - 1) / 16) : 0) +
           (blocks * waves > 32 * kI8CUs ? 2 : 0);
}

// The kernel of a dense product and the splits of its K, by these times. What it weighs (us): 1 x 2560 x 9728 few 7.7, tiles 9.1; 1 x
// 9728 x 2560 few by 16 waves 8.9, by 8 10.8, tiles 23.7, in 8 splits 11.5; 64 x 2560 x 9728 few 20, 64 x 128 tiles 9.6; 128 x 9728 x
// 2560 64 x 128 tiles 23.5, in 4 splits 13.2; 512 x 2560 x 9728 256 x 128 25, 128 x 128 30, 256 x 256 35; 1536 rows of it 54, 57, 45.
inline int i8_dense(brik_i8_launch& a, int forced, int splits)
{
    const long M = a.M, K = a.K, N = a.N, steps = (K + 127) / 128;
    int best = -1, best_splits = 1;
    double us = 1e30;
    for (int t = 0; t < kI8Moe; ++t) {
        const I8Kernel& g = kI8Kernels[t];
        if (forced ? t != forced - 1 : t == kI8Few || (g.kind == I8_FEW && (M > 64 || (M > 16) != (g.bm > 16)))) continue;
        for (int s : {1, 2, 3, 4, 6, 8, 12, 16}) {
            if (splits) s = splits;
            else if (s > 1 && (g.kind == I8_FEW || steps < 4 * s)) break;
            const double tiles = (double)((M + g.bm - 1) / g.bm) * ((N + g.bn - 1) / g.bn);
            double x = g.kind == I8_FEW ? i8_few_us(M, K, N, g.threads / 64) : i8_tile_us(kI8Times[t - kI8Tiles], tiles * s, (double)((steps + s - 1) / s));
            if (s > 1) x += 2 + 0.45 * s + 8.0 * s * M * N / 5e6;        // the sums written and read again by a launch of its own
            if (x < us) {
                us = x;
                best = t;
                best_splits = s;
            }
            if (splits) break;
        }
    }
    const long each = ((K + 63) / 64 + best_splits - 1) / best_splits;
    a.steps = (int)std::max(1l, best_splits > 1 ? (each + 1) / 2 * 2 : each);        // whole steps of 128
    a.splits = (int)std::max(1l, ((K + 63) / 64 + a.steps - 1) / a.steps);
    return best;
}

// The kernel of a product by experts, by the mean of their rows (all rows count, those without an expert too: how many there are stays on
// the device). 64 experts, 8 a token, 2048 x 1536 and 768 x 2048 (us; 256 and 1024 tokens the first alone, 4096 the second; up to 4 tokens
// with the weights in the last-level cache):
//   tokens      1           2           4           8           16          32          256         1024       4096   8192
//   few         9.8   6.7   13.4  8.4   22.4  12.4  31.0  16.3  35.9  20.7  40.5  24.7
//   64 rows     9.1   6.1   12.5  9.3   20.7  13.7  36.1  21.3  37.7  22.4  39.6  24.4  51.1        77.9           156  366   281
//   128 rows    12.0  7.6               25.3  18.4  43.5  27.6              47.2  31.9  52.9        78.1           145  326   254
//   256 rows                                                                                        114            143  319   236
// and by 2048 x 1536 alone 512 tokens 61.2 by 64 rows, 63.7 by 128; 2048 tokens 128, 116, 128 by 256; 4096 215, 193, 209; 6144 268, 264 (128, 256).
// So few rows are right from 8 tokens to 16 and cost up to 11 % at 1 to 4, which the mean cannot tell from 8; with 256 experts, where few rows
// start a block for each, one token takes 15.2 against 9.8 by 64 rows, 8 tokens 36.7 against 38.5. K < 1024 keeps 128 rows, 2 to 8 % behind 256.
// Waves of a few-row block, 4, 8, 16, 8 tokens: 1024 x 2048 22.9, 31.7, 54.0; 2048 x 1536 31.1, 34.9, 47.7; 4096 x 1024 45.2, 39.1, 45.8; 8192 x 512
// 43.0, 43.4, 40.3.
inline int i8_experts(brik_i8_launch& a, int forced)
{
    a.splits = 1;
    a.steps = (a.K + 63) / 64;
    if (forced && kI8Kernels[forced - 1].kind != I8_TILE) return forced - 1;
    const long rows = ((long)a.M + a.E - 1) / a.E;
    if (rows <= 2) return a.K <= 2048 ? 0 : a.K <= 4096 ? 1 : 3;
    return rows <= 160 ? kI8Moe + 2 : rows <= 768 || a.K < 1024 ? kI8Moe + 1 : kI8Moe;
}

// What a launch takes: blocks, and threads, that 32 bits count.
inline bool i8_fits(const brik_i8_launch& a, int kernel, long& blocks)
{
    blocks = (long)a.row_tiles * a.col_tiles * a.splits;
    return blocks < (1l << 23) && blocks * kI8Kernels[kernel].threads < (1l << 32);
}

inline void i8_grid(brik_i8_launch& a, int kernel)
{
    const I8Kernel& g = kI8Kernels[kernel];
    a.col_tiles = (a.N + g.bn - 1) / g.bn;
    if (g.kind == I8_FEW) a.row_tiles = std::max(1, a.E);
    else a.row_tiles = (int)(((long)a.M + g.bm - 1) / g.bm + (a.E ? std::min(a.E, a.M) : 0));
}

// The kernel of a call, and its grid in `a`. forced: 0, or 1 + index of a kernel (a tile of the other kind: 0). A kernel that nobody
// forced gives way to larger tiles where a launch does not hold its blocks.
inline int i8_plan(brik_i8_launch& a, int forced, int splits)
{
    if (!a.E && forced > kI8Moe) forced = 0;
    int t;
    if (a.K == 0) {                      // (a tile without steps: sums of 0)
        forced = 0;
        t = a.E ? kI8Moe + 2 : kI8Tiles + 3;
        a.splits = a.steps = 1;
    } else t = a.E ? i8_experts(a, forced) : i8_dense(a, forced, splits);
    i8_grid(a, t);
    if (forced && t == forced - 1) return t;
    long blocks;
    while (!i8_fits(a, t, blocks)) {
        const int larger = a.E && kI8Kernels[t].kind == I8_FEW ? kI8Moe + 2 : t - 1;
        if (larger < kI8Tiles || larger == kI8Moe - 1) break;
        i8_grid(a, t = larger);
    }
    return t;
}

}  // namespace brik_plan
