// Host test of the rows that a step leaves alone (attn_abi.h) and of rows that share a buffer (attn_check.h), without a device.
// Prints "ok" and returns 0 when every check holds.
#include "../../brimkern_amd/csrc/attn_check.h"

#include <cstdio>
#include <vector>

static int failures = 0;
#define EXPECT(c)                                              \
    do {                                                       \
        if (!(c)) {                                            \
            std::printf("line %d: %s\n", __LINE__, #c);        \
            ++failures;                                        \
        }                                                      \
    } while (0)

int main()
{
    // a row belongs to a sequence exactly where some sequence's [row_off[b], row_off[b + 1]) holds it
    const std::vector<std::vector<int32_t>> offs = {{0, 2, 5}, {3, 3, 5}, {1000, 1001, 1002}, {4, 4, 4}, {-3, 1, 9}, {0, 0, 0}, {7, 8, 20}};
    for (const auto& off : offs) {
        brik_step s{};
        s.row_off = off.data();
        s.seqs = 2;
        s.rows = 8;
        for (int32_t t = 0; t < s.rows; ++t) {
            bool in = false;
            for (int b = 0; b < s.seqs; ++b) {
                int32_t first, count;
                brik_rows_of(s, b, first, count);
                in = in || (t >= first && t < first + count);
            }
            EXPECT(brik_row_taken(s, t) == in);
        }
    }
    brik_step s{};
    s.seqs = s.per_seq = 2;
    s.rows = 4;
    for (int32_t t = 0; t < 4; ++t) EXPECT(brik_row_taken(s, t));

    // rows of two kinds in one buffer: overlapping exactly where they share a float
    for (int64_t as : {8, 12, 16})
        for (int64_t bs : {8, 12, 16})
            for (int64_t aw : {4, 8})
                for (int64_t bw : {4, 8})
                    for (int rows : {1, 2, 3})
                        for (int64_t at = 0; at < 120; at += 4) {
                            const float* const p = reinterpret_cast<const float*>((uintptr_t)0x10000);
                            bool meet = false;
                            for (int i = 0; i < rows; ++i)
                                for (int j = 0; j < rows; ++j) {
                                    const int64_t a0 = 60 + i * as, b0 = at + j * bs;
                                    meet = meet || (a0 < b0 + bw && b0 < a0 + aw);
                                }
                            const bool said = brik_check::overlap(p + 60, as, aw, p + at, bs, bw, rows);
                            EXPECT(as == bs ? said == meet : said || !meet);      // of unlike strides: never missed
                        }
    std::printf(failures ? "%d failure(s)\n" : "ok\n", failures);
    return failures != 0;
}
