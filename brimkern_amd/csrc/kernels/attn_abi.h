// What the attention side's kernels (kv_rows.hip, attn*.hip) and the host runtime share: the launch arguments and where
// a token lies in the cache. Plain functions, so that the host's tests run the same code.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "../../../include/brik.h"

#ifdef __HIP__
#include <hip/hip_runtime.h>
#define BRIK_HD __host__ __device__ __forceinline__
#else
#define BRIK_HD static inline
#endif

// log2 of a power of two
BRIK_HD int brik_log2(int v)
{
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

// The step as a kernel sees it: the batch, and the cache's paging.
typedef struct brik_step {
    const int32_t *row_off, *kv_len, *table, *prefix_table;
    int32_t seqs, rows, table_cols, max_len, prefix_len;
    int32_t per_seq;       // rows per sequence where row_off is null
    int32_t pages, shift;  // page = 1 << shift
} brik_step;

// The page of token p of sequence b, or -1 where the token does not exist. The token's slot is brik_slot's.
BRIK_HD int32_t brik_page_of(const brik_step& s, int b, int32_t p)
{
    if (p < 0 || p >= s.max_len) return -1;
    int32_t id;
    if (p < s.prefix_len) {
        id = s.prefix_table[p >> s.shift];
    } else {
        const int32_t col = (p - s.prefix_len) >> s.shift;
        if (col >= s.table_cols) return -1;
        id = s.table[(size_t)b * s.table_cols + col];
    }
    return (uint32_t)id < (uint32_t)s.pages ? id : -1;
}

BRIK_HD int32_t brik_slot(const brik_step& s, int32_t p)
{
    return (p < s.prefix_len ? p : p - s.prefix_len) & ((1 << s.shift) - 1);
}

// Rows of sequence b as [first, first + count): clipped to the rows there are, whatever row_off holds.
BRIK_HD void brik_rows_of(const brik_step& s, int b, int32_t& first, int32_t& count)
{
    if (!s.row_off) {
        first = b * s.per_seq;
        count = s.per_seq;
        return;
    }
    const int32_t a = s.row_off[b], e = s.row_off[b + 1];
    first = a < 0 ? 0 : a > s.rows ? s.rows : a;
    const int32_t end = e > s.rows ? s.rows : e;
    count = end > first ? end - first : 0;
}

// Rows before the first sequence's and behind the last one's belong to none.
BRIK_HD bool brik_row_taken(const brik_step& s, int32_t t)
{
    return !s.row_off || (t >= s.row_off[0] && t < s.row_off[s.seqs]);
}

// Index of the vector (token's head) in a cache plane: planes are [pages, heads, page, head_dim].
BRIK_HD size_t brik_vector(const brik_step& s, int heads, int32_t page, int head, int32_t slot)
{
    return (((size_t)page * heads + head) << s.shift) + slot;
}

typedef struct brik_rows_launch {
    brik_qkv_rows r;       // strides filled in
    brik_step s;
    brik_kv_cache c;
    int32_t nq, nk, nv;    // heads of q, k and v to go over
} brik_rows_launch;

typedef struct brik_read_launch {
    brik_step s;
    brik_kv_cache c;
    float *k, *v;
} brik_read_launch;

typedef struct brik_attn_launch {
    brik_attn_args a;      // strides filled in
    brik_step s;
    brik_kv_cache c;
    // Partial results, where keys are split: outputs [vector][head_dim], reference exponents and sums [vector][2]. Vectors:
    // [slot][row][head] with the slots of the prefix, then (own_blocks == 0) those of the own keys; own_blocks > 0: behind the
    // prefix's, [key / value head][own_blocks + seqs parts][16 rows].
    float *part, *ml;
    // The grid: row tiles of the prefix's keys (rows of all sequences) and of the sequences' own keys, each tile's keys
    // split over so many blocks. tiles_per_seq: the tile's sequence by division (0: by a search over the sequences' rows).
    int32_t prefix_tiles, prefix_splits, own_splits, tiles_per_seq;
    // One tile a sequence: own_blocks blocks per key / value head share the sequences' keys out by their lengths.
    int32_t own_blocks;
    int32_t first_block;   // number of the launch's first block
    int32_t whole;         // no splits, no prefix: the kernel writes the output
} brik_attn_launch;
