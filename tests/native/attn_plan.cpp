// Host test of how a call of brik_attention is divided over the device (attn_plan.h), without one: for many batches the blocks of the
// grid are gone through as the kernels number them. Every key block that a row sees is done exactly once, every partial result
// has a place of its own inside the workspace, and the joins read what was written. Prints "ok" and returns 0.
#include "../../brimkern_amd/csrc/attn_plan.h"

#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <vector>

static int failures = 0;
#define EXPECT(c)                                              \
    do {                                                       \
        if (!(c)) {                                            \
            if (++failures < 20) std::printf("line %d: %s (case %d)\n", __LINE__, #c, now); \
        }                                                      \
    } while (0)
static int now = 0;

struct Batch {
    std::vector<int32_t> off, len;
    int cols = 0, shift = 4, prefix = 0, max_len = 0, max_rows = 0, rows = 0;
};

// The blocks of 32 own keys that the rows [r0, r0 + count) of sequence b see: [first, first + n).
static void own_keys(const brik_attn_launch& a, int b, int r0, int count, long& first, long& n)
{
    const long end_row = a.s.row_off ? a.s.row_off[b + 1] : (b + 1) * a.s.per_seq, before = a.s.prefix_len;
    const long pos = a.s.kv_len[b] - end_row + r0;
    const long end = std::min<long>(a.s.max_len - before, (long)a.s.table_cols << a.s.shift);
    const long hi = std::min(pos + count - before, end), lo = a.a.window ? std::max(0l, pos - a.a.window + 1 - before) : 0;
    first = lo / 32;
    n = count > 0 && lo < hi ? (hi + 31) / 32 - first : 0;
}

using Ranges = std::vector<std::pair<long, long>>;

// Whether the ranges are [first, first + n), each part once.
static bool whole(Ranges k, long first, long n)
{
    std::sort(k.begin(), k.end());
    long at = first;
    for (auto& r : k) {
        if (r.first != at || r.second <= r.first) return false;
        at = r.second;
    }
    return at == first + n;
}

static void check(brik_attn_launch a, const Batch& t, const brik_plan::AttnOptions& opt)
{
    const brik_plan::AttnGrid g = brik_plan::attn_grid(a, t.max_rows, opt);
    const int KV = a.c.heads, G = a.a.heads / KV;
    const size_t all = (size_t)a.s.rows * a.a.heads;
    EXPECT(g.own_rows == 16 || g.own_rows == 128 || (g.own_rows == 256 && a.c.head_dim <= 128));
    EXPECT(g.prefix_rows == 16 || g.prefix_rows == 128 || (g.prefix_rows == 256 && a.c.head_dim <= 128));
    EXPECT(g.own_blocks > 0 && g.own_blocks % KV == 0 && a.own_splits >= 1 && (opt.splits ? a.own_splits == opt.splits : a.own_splits <= 64));
    EXPECT(a.whole == (g.vectors == 0));
    EXPECT(a.own_blocks == 0 || (g.own_rows == 16 && a.own_splits == 1));
    EXPECT(g.prefix_blocks == (long)KV * a.prefix_tiles * a.prefix_splits);
    EXPECT(a.prefix_splits == 0 || (long)a.prefix_tiles * g.prefix_rows >= (long)a.s.rows * G);
    EXPECT(!g.join_few || (a.own_blocks == 0 && a.prefix_splits + a.own_splits <= 16));
    std::set<size_t> places;                                     // of partial results, key / value head 0
    std::map<std::pair<int, int>, Ranges> keys;                  // (row tile's sequence, first row): blocks of keys done
    const int blocks = (int)(g.own_blocks / KV);
    if (a.own_blocks) {
        // shared out: the sequences' blocks of keys in a row
        std::vector<long> first(a.s.seqs), n(a.s.seqs), start(a.s.seqs);
        long total = 0;
        for (int b = 0; b < a.s.seqs; ++b) {
            int32_t row, rows;
            brik_rows_of(a.s, b, row, rows);
            own_keys(a, b, row, rows, first[b], n[b]);
            start[b] = total;
            total += n[b];
        }
        const long each = std::max(4l, (total + a.own_blocks - 1) / a.own_blocks);
        EXPECT(blocks == a.own_blocks && total < (1l << 31) && each * a.own_blocks >= total);
        for (int block = 0; block < blocks; ++block)
            for (int b = 0; b < a.s.seqs; ++b) {
                const long lo = std::max(block * each, start[b]), hi = std::min((block + 1) * each, start[b] + n[b]);
                if (lo >= hi) continue;
                keys[{b, 0}].push_back({first[b] + lo - start[b], first[b] + hi - start[b]});
                if (a.prefix_splits == 0 && start[b] / each == (start[b] + n[b] - 1) / each) continue;     // writes the output
                for (int m = 0; m < 16; ++m) {
                    for (int h = 0; h < KV; h += std::max(1, KV - 1)) {
                        const size_t at = a.prefix_splits * all + ((size_t)h * (a.own_blocks + a.s.seqs) + block + b) * 16 + m;
                        EXPECT(at < g.vectors);
                        if (h == 0) EXPECT(places.insert(at).second);
                    }
                }
            }
        for (int b = 0; b < a.s.seqs; ++b) {
            EXPECT(whole(keys[{b, 0}], first[b], n[b]));
        }
        return;
    }
    // tiles of rows, their keys over the splits
    std::map<std::pair<int, int>, int> done;                     // (sequence, first row of a tile): splits that write it
    for (int block = 0; block < blocks; ++block) {
        const int split = block % a.own_splits;
        int tile = block / a.own_splits, b, j;
        if (a.tiles_per_seq) {
            b = tile / a.tiles_per_seq;
            j = tile % a.tiles_per_seq;
        } else {
            for (b = 0; b < a.s.seqs; ++b) {
                int32_t row, rows;
                brik_rows_of(a.s, b, row, rows);
                const int here = (int)(((long)rows * G + g.own_rows - 1) / g.own_rows);
                if (tile < here) break;
                tile -= here;
            }
            j = tile;
            if (b == a.s.seqs) continue;
        }
        EXPECT(b < a.s.seqs);
        int32_t row, rows;
        brik_rows_of(a.s, b, row, rows);
        int tiles = (int)(((long)rows * G + g.own_rows - 1) / g.own_rows);
        if (a.tiles_per_seq) tiles = std::min(tiles, a.tiles_per_seq);
        if (j >= tiles) continue;
        const int r0 = (tiles - 1 - j) * g.own_rows;
        ++done[{b, r0}];
        long first, n;
        const int t0 = r0 / G, t1 = std::min((r0 + g.own_rows - 1) / G + 1, (int)rows);
        own_keys(a, b, row + t0, t1 - t0, first, n);
        const long each = (n + 4 * a.own_splits - 1) / (4 * a.own_splits) * 4;
        if (split * each < n) keys[{b, r0}].push_back({first + split * each, first + std::min(n, (split + 1) * each)});
        if (!a.whole) EXPECT((a.prefix_splits + split) * all + (size_t)(row + rows - 1) * a.a.heads + a.a.heads - 1 < g.vectors);
    }
    for (int b = 0; b < a.s.seqs; ++b) {
        int32_t row, rows;
        brik_rows_of(a.s, b, row, rows);
        const long promised = std::min<long>(rows, t.max_rows ? t.max_rows : rows) * G;
        for (int r0 = 0; r0 < promised; r0 += g.own_rows) EXPECT((done[{b, r0}] == a.own_splits));
        for (int r0 = 0; r0 < promised; r0 += g.own_rows) {
            long first, n;
            own_keys(a, b, row + r0 / G, std::min((r0 + g.own_rows - 1) / G + 1, (int)rows) - r0 / G, first, n);
            EXPECT(whole(keys[{b, r0}], first, n));
        }
    }
}

int main()
{
    std::mt19937 rng(7);
    auto pick = [&](std::initializer_list<int> v) { return *(v.begin() + rng() % v.size()); };
    for (now = 0; now < 1500; ++now) {
        Batch t;
        brik_attn_launch a{};
        a.c.heads = pick({1, 2, 3, 8, 16, 40});
        a.a.heads = a.c.heads * pick({1, 2, 4, 7, 20});
        a.c.head_dim = pick({64, 96, 128, 192, 256});
        a.s.seqs = pick({1, 1, 2, 5, 17, 70, 200, 1100});
        t.shift = pick({4, 6, 8});
        t.prefix = pick({0, 0, 0, 1, 45, 300, 9000});
        const int most = pick({1, 1, 1, 2, 5, 40, 333}), longest = pick({1, 30, 700, 5000, 70000});
        const bool ragged = rng() % 3 != 0;
        int rows = ragged && rng() % 4 == 0 ? (int)(rng() % 50) : 0;                 // rows before the first sequence
        t.off.push_back(rows);
        for (int b = 0; b < a.s.seqs; ++b) {
            rows += ragged ? (int)(rng() % (most + 1)) : most;
            t.off.push_back(rows);
            t.len.push_back((int)(rng() % (longest + 1)) + (rng() % 2 ? t.prefix : 0));
            t.max_len = std::max(t.max_len, t.len.back());
        }
        a.s.rows = std::max(1, rows + (ragged ? (int)(rng() % 3) : 0));
        a.s.row_off = ragged ? t.off.data() : nullptr;
        a.s.kv_len = t.len.data();
        a.s.per_seq = ragged ? 0 : most;
        t.max_rows = rng() % 3 == 0 ? 0 : rng() % 4 ? most : std::max(1, most / 2);  // half: fewer than a sequence may have
        if (!ragged) t.max_rows = most;
        a.s.max_len = t.max_len;
        a.s.prefix_len = t.prefix;
        a.s.shift = t.shift;
        a.s.table_cols = rng() % 5 ? (std::max(0, t.max_len - t.prefix) >> t.shift) + 1 : (int)(rng() % 8);
        a.a.window = pick({0, 0, 1, 50, 1500, INT32_MAX});
        brik_plan::AttnOptions opt;
        if (rng() % 3 == 0) opt.rows = pick({16, 128, 256});
        if (rng() % 3 == 0) opt.splits = pick({1, 2, 3, 17, 64, 256});
        check(a, t, opt);
    }
    // choices that the comments beside the model give as the fastest: 32 heads over 8 of 128
    auto choice = [](int seqs, int rows, int len, int tile, int splits) {
        brik_attn_launch a{};
        a.c.heads = 8;
        a.c.head_dim = 128;
        a.a.heads = 32;
        a.s.seqs = seqs;
        a.s.rows = seqs * rows;
        a.s.per_seq = rows;
        a.s.max_len = len;
        a.s.shift = 6;
        a.s.table_cols = (len + 63) / 64;
        const brik_plan::AttnGrid g = brik_plan::attn_grid(a, 0, {});
        if (g.own_rows != tile || a.own_splits != splits) std::printf("%d x %d of %d: %d rows, %d splits\n", seqs, rows, len, g.own_rows, a.own_splits);
        return g.own_rows == tile && a.own_splits == splits;
    };
    EXPECT(choice(1, 1, 4095, 16, 32));
    EXPECT(choice(1, 1, 131072, 16, 64));
    EXPECT(choice(1, 1024, 1024, 16, 1));
    EXPECT(choice(1, 2048, 2048, 256, 2));
    EXPECT(choice(1, 4096, 4096, 256, 1));
    EXPECT(choice(1, 512, 8192, 256, 4));
    std::printf(failures ? "%d failure(s)\n" : "ok\n", failures);
    return failures != 0;
}
