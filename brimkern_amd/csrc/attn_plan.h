// How a call of brik_attention is divided over the device: row tiles, splits of the keys, the grid and the partial results. Plain
// functions of the sizes, apart from any context.
#pragma once
#include "kernels/attn_abi.h"

#include <algorithm>
#include <cmath>

namespace brik_plan {

constexpr int kDeviceCUs = 256;           // MI355X compute units

// Row tiles and splits of a section of keys (the own ones, or the prefix's): those with the least time by a model of the kernels,
// fitted to measured times (us). A block takes `start`, then steps of `alone` where the device is not full and of `full` where its
// `slots` are; a step of 16-row tiles is 128 keys (32 a wave), of the others 32 keys. Partial results are written and read
// again at 4.5 TB/s and joined by a launch of 5. What it weighs, 32 heads over 8 of 128, q8, by 16, 128 and 256 rows unsplit:
// a prompt of 1024 rows 68, 89, 93; of 2048 190, 170, 175 (256 in 2 splits 137); of 4096 639, 439, 384; eight prompts of 256
// 80, 41, 37 (65 and more in 2 splits); 512 rows behind 8192 292, 617, 644 (256 in 4 splits 200). One row of 4095: 32 splits
// 12.3, 16 splits 14.4, 8 splits 17.9; of 131072: 64 splits 63, 32 or 128 70.
struct AttnOptions {
    int rows = 0, splits = 0;             // 0: by the sizes
};
struct AttnPlan {
    int rows = 16, splits = 1;
    double us = 1e30;
};
struct AttnSection {
    long KV, G, D, rows, seqs, most;      // most: rows of a sequence
    long keys, window;
    bool prefix, ragged;
    long tiles(int bm) const
    {
        const long bound = (rows * G + bm - 1) / bm;
        if (prefix) return bound;
        const long each = (most * G + bm - 1) / bm * seqs;
        return ragged ? std::min(each, bound + seqs) : each;
    }
};
inline AttnPlan attn_plan(const AttnOptions& opt, const AttnSection& x, bool joined, int beside)
{
    static const int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 40, 48, 64};
    AttnPlan best;
    for (int bm : {16, 128, 256}) {
        if (opt.rows ? bm != (x.D > 128 && opt.rows > 16 ? 128 : opt.rows)
                             : bm > 16 && (x.most * x.G <= 16 || (bm == 256 && x.D > 128)))
            continue;
        const double D = (double)x.D, slots = kDeviceCUs * (bm == 16 ? x.D <= 64 ? 3 : x.D <= 128 ? 2 : 1 : bm == 128 && x.D <= 128 ? 2 : 1);
        const double start = bm == 16 ? 3.8 : 4, alone = bm == 16 ? 0.65 + 0.0086 * D : bm == 128 ? 0.6 + 0.0145 * D : 0.9 + 0.0133 * D;
        const double full = bm == 16 ? 3.3e-5 * D * slots : bm == 256 ? 0.9 + 0.0155 * D : x.D <= 128 ? 1 + 0.018 * D : alone;
        // keys of the tile that sees the most, and of the middle one
        const long far = x.window ? std::min(x.keys, x.window + bm / x.G + 32) : x.keys;
        const long mid = x.prefix ? far : std::min(far, std::max(1l, x.keys - x.most / 2 + bm / x.G));
        const double blocks = (double)x.KV * x.tiles(bm), vectors = (double)x.rows * x.KV * x.G;
        const long most = std::max(1l, std::min(64l, (far + 127) / 128));
        double last = 0;
        for (int q : kSplits) {
            if (opt.splits) q = opt.splits;
            else if (q > most) break;
            // steps of the longest split (four of a tile's, or one of a 16-row tile's, at a time) and of the middle tile's
            const double unit = bm == 16 ? 1 : 4, f = unit * ((far + 128 * q - 1) / (128 * q));
            const double m = mid == far ? f : std::min(f, unit * mid / (128 * q) + 0.5);
            if (f == last && !opt.splits) continue;      // more splits, none of them shorter
            last = f;
            // rounds that blocks of one length do not fill last as long as full ones (half that with several blocks on a CU);
            // where lengths differ the long ones go first, and short ones fill the gaps
            const double rounds = blocks * q / slots, even = std::max(0.0, 2.0 * mid / std::max(1l, far) - 1) * (bm == 256 ? 1 : 0.5);
            double us = std::max(start + f * alone, std::max(1.0, rounds + (std::ceil(rounds) - rounds) * even) * (start + m * full));
            if (q > 1 || joined) us += (joined ? 0 : 5) + vectors * (2 * q + 1) * 4 * D / 4.5e6;
            if (beside && beside != bm) us += 10;            // another kernel's launch
            if (us < best.us) best = AttnPlan{bm, q, us};
            if (opt.splits) break;
        }
    }
    return best;
}

// The launches of a call.
struct AttnGrid {
    int own_rows = 0, prefix_rows = 0;        // rows of a tile: of the own keys, of the prefix's
    long own_blocks = 0, prefix_blocks = 0;
    size_t vectors = 0;                       // partial results
    bool join_few = false;                    // joined by a group of lanes each
};

// Fills in a.tiles_per_seq, own_blocks, own_splits, prefix_tiles, prefix_splits and whole. a.a, a.s and a.c are checked.
inline AttnGrid attn_grid(brik_attn_launch& a, int max_rows, const AttnOptions& opt)
{
    AttnGrid r;
    const long KV = a.c.heads, G = a.a.heads / KV, rows = a.s.rows;
    const long own_keys = std::min<long>((long)a.s.max_len - a.s.prefix_len, (long)a.s.table_cols << a.s.shift);
    const long prefix_keys = std::min(a.s.prefix_len, a.s.max_len);
    const long most = a.s.row_off ? std::min<long>(max_rows ? max_rows : rows, rows) : a.s.per_seq;    // rows of a sequence
    AttnSection own{KV, G, a.c.head_dim, rows, a.s.seqs, most, std::max(0l, own_keys), a.a.window, false, a.s.row_off != nullptr};
    const AttnPlan own_plan = attn_plan(opt, own, prefix_keys > 0, 0);
    r.own_rows = own_plan.rows;
    // row tiles of the sequences: the same number for each where that is not many more than there can be
    const long per_seq = (most * G + r.own_rows - 1) / r.own_rows, bound = (rows * G + r.own_rows - 1) / r.own_rows + a.s.seqs;
    long tiles = per_seq * a.s.seqs;
    a.tiles_per_seq = (int)per_seq;
    if (a.s.row_off && tiles > 2 * bound) {
        a.tiles_per_seq = 0;
        tiles = bound;
    }
    // One tile a sequence and several sequences: their keys in a row, shared out evenly over the blocks that the device takes at
    // once, by the lengths that the call finds. (Splits of the longest length left 32 sequences of 1 to 8192 tokens waiting for
    // the longest.) Only where a block gets 16 blocks of keys and a sequence has over 1024: one that begins a second sequence
    // pays 4 us for it (17 sequences behind a window of 635 tokens, one head of 128: 20 us shared out, 13 by splits).
    const long far = a.a.window ? std::min(own_keys, a.a.window + most) : own_keys, blocks32 = (std::max(0l, far) + 31) / 32;
    const long share = std::max(1l, (a.c.head_dim <= 128 ? 2 : 1) * kDeviceCUs / KV);
    if (r.own_rows == 16 && per_seq == 1 && a.s.seqs > 1 && a.s.seqs <= 1024 && blocks32 > 32 && a.s.seqs * blocks32 >= 16 * share &&
        a.s.seqs * blocks32 < (1l << 30) && !opt.splits) {
        a.own_blocks = (int)share;
        tiles = a.own_blocks;
        a.own_splits = 1;
    } else {
        a.own_splits = own_plan.splits;
    }
    r.prefix_rows = r.own_rows;
    if (prefix_keys > 0) {
        AttnSection pre = own;
        pre.prefix = true;
        pre.most = rows;
        pre.keys = prefix_keys;
        const AttnPlan plan = attn_plan(opt, pre, true, r.own_rows);
        r.prefix_rows = plan.rows;
        a.prefix_tiles = (int)((rows * G + plan.rows - 1) / plan.rows);
        a.prefix_splits = plan.splits;
    }
    a.whole = a.prefix_splits == 0 && a.own_splits == 1 && a.own_blocks == 0;
    const size_t all = (size_t)rows * a.a.heads;
    if (!a.whole)
        r.vectors = a.prefix_splits * all + (a.own_blocks ? (size_t)KV * (a.own_blocks + a.s.seqs) * 16 : a.own_splits * all);
    r.own_blocks = KV * tiles * a.own_splits;
    r.prefix_blocks = KV * a.prefix_tiles * a.prefix_splits;
    // few slots, or rows and heads for every CU: each group of lanes joins a row and head by itself; else a block shares the slots
    // out (32 heads of one row: 16 slots 15.0 us the one way, 12.9 the other, 4 slots 12.5 and 12.8; 1024 rows by 2 slots 68 and 102)
    const int slots = a.prefix_splits + a.own_splits;
    r.join_few = !a.own_blocks && (slots <= 4 || (slots <= 16 && rows * a.a.heads >= 2 * kDeviceCUs));
    return r;
}

}  // namespace brik_plan
