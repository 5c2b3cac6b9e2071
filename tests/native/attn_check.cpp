// Host test of the attention side's argument checks (attn_check.h) and of where a token lies (attn_abi.h), without a
// device. Prints "ok" and returns 0 when every check holds.
#include "../../brimkern_amd/csrc/attn_check.h"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <limits>
#include <vector>

static int failures = 0;
#define EXPECT(c)                                              \
    do {                                                       \
        if (!(c)) {                                            \
            std::printf("line %d: %s\n", __LINE__, #c);        \
            ++failures;                                        \
        }                                                      \
    } while (0)

template <class T>
static T* at(uintptr_t a) { return reinterpret_cast<T*>(a); }

int main()
{
    using namespace brik_check;
    Why w;
    // pages: every id the device may find in a table, in range or not
    std::vector<int32_t> table = {3, 0, -1, 4, 7, INT32_MAX, INT32_MIN, 1}, prefix = {2, 9}, len = {0, 0}, off = {0, 2, 5};
    brik_step s{};
    s.table = table.data();
    s.prefix_table = prefix.data();
    s.table_cols = 4;
    s.pages = 5;
    s.shift = 4;
    s.prefix_len = 20;
    s.max_len = 80;
    EXPECT(brik_page_of(s, 0, -1) == -1 && brik_page_of(s, 0, INT32_MIN) == -1);
    EXPECT(brik_page_of(s, 0, 0) == 2 && brik_page_of(s, 0, 15) == 2 && brik_slot(s, 15) == 15);
    EXPECT(brik_page_of(s, 0, 16) == -1);                               // page 9 of 5
    EXPECT(brik_page_of(s, 0, 20) == 3 && brik_slot(s, 20) == 0 && brik_slot(s, 35) == 15);
    EXPECT(brik_page_of(s, 0, 36) == 0 && brik_page_of(s, 0, 52) == -1 && brik_page_of(s, 0, 68) == 4);
    EXPECT(brik_page_of(s, 1, 20) == -1 && brik_page_of(s, 1, 36) == -1 && brik_page_of(s, 1, 52) == -1 && brik_page_of(s, 1, 79) == 1);
    EXPECT(brik_page_of(s, 1, 80) == -1 && brik_page_of(s, 1, INT32_MAX) == -1);
    s.max_len = INT32_MAX;
    EXPECT(brik_page_of(s, 1, 83) == 1 && brik_page_of(s, 1, 84) == -1 && brik_page_of(s, 0, INT32_MAX - 1) == -1);
    EXPECT(brik_vector(s, 8, 1 << 20, 7, 15) == (((size_t)(1 << 20) * 8 + 7) << 4) + 15);
    // rows: clipped whatever row_off holds
    s.rows = 4;
    s.row_off = off.data();
    int32_t first, count;
    brik_rows_of(s, 0, first, count);
    EXPECT(first == 0 && count == 2);
    brik_rows_of(s, 1, first, count);
    EXPECT(first == 2 && count == 2);
    off = {-5, 1 << 30, 3};
    brik_rows_of(s, 0, first, count);
    EXPECT(first == 0 && count == 4);
    brik_rows_of(s, 1, first, count);
    EXPECT(first == 4 && count == 0);
    s.row_off = nullptr;
    s.per_seq = 2;
    brik_rows_of(s, 1, first, count);
    EXPECT(first == 2 && count == 2);

    // caches
    brik_kv_cache c{BRIK_FMT_Q4, 2, 128, 64, 10, 0, at<void>(0x1000), at<void>(0x2000), at<uint16_t>(0x3000), at<uint16_t>(0x4000),
                    at<uint16_t>(0x5000), at<uint16_t>(0x6000)};
    EXPECT(cache(w, "t", &c) == BRIK_OK && cache(w, "t", nullptr) == BRIK_EINVAL);
    auto bad_cache = [&](int code, auto change) {
        brik_kv_cache x = c;
        change(x);
        EXPECT(cache(w, "t", &x) == code);
    };
    bad_cache(BRIK_EINVAL, [](brik_kv_cache& x) { x.fmt = BRIK_FMT_Q3; });
    bad_cache(BRIK_EINVAL, [](brik_kv_cache& x) { x.reserved = 1; });
    bad_cache(BRIK_EINVAL, [](brik_kv_cache& x) { x.heads = 0; });
    bad_cache(BRIK_EINVAL, [](brik_kv_cache& x) { x.pages = -1; });
    for (int d : {0, -32, 16, 48, 288}) bad_cache(BRIK_EINVAL, [&](brik_kv_cache& x) { x.head_dim = d; });
    for (int p : {0, 8, 24, 131072, -64, INT32_MIN}) bad_cache(BRIK_EINVAL, [&](brik_kv_cache& x) { x.page = p; });
    bad_cache(BRIK_EINVAL, [](brik_kv_cache& x) { x.heads = 65536, x.page = 65536; });
    bad_cache(BRIK_EINVAL, [](brik_kv_cache& x) { x.k = nullptr; });
    bad_cache(BRIK_EINVAL, [](brik_kv_cache& x) { x.v_mins = nullptr; });
    bad_cache(BRIK_EALIGN, [](brik_kv_cache& x) { x.v = at<void>(0x2008); });
    bad_cache(BRIK_EALIGN, [](brik_kv_cache& x) { x.k_scales = at<uint16_t>(0x3002); });

    // batches
    brik_kv_batch b{2, 4, nullptr, len.data(), table.data(), 4, 100, 0, 0, nullptr};
    EXPECT(batch(w, "t", &b, true, true) == BRIK_OK && batch(w, "t", nullptr, true, true) == BRIK_EINVAL);
    auto bad_batch = [&](int code, auto change) {
        brik_kv_batch x = b;
        change(x);
        EXPECT(batch(w, "t", &x, true, true) == code);
    };
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.rows = 5; });
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.rows = -1; });
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.seqs = 0; });
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.kv_len = nullptr; });
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.table = nullptr; });
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.prefix_len = 5; });
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.prefix_len = -5; });
    bad_batch(BRIK_EINVAL, [](brik_kv_batch& x) { x.max_rows = 1; });
    bad_batch(BRIK_EALIGN, [](brik_kv_batch& x) { x.kv_len = at<int32_t>(0x1002); });
    bad_batch(BRIK_OK, [](brik_kv_batch& x) { x.rows = 0, x.seqs = 0, x.kv_len = nullptr; });

    // rows
    brik_qkv_rows r{};
    r.q = r.k = r.v = at<float>(0x10000);
    r.q_out = at<float>(0x20000);
    r.heads = 4;
    r.kv_heads = 2;
    r.head_dim = 128;
    r.inv_freq = at<float>(0x30000);
    r.rot_dim = 64;
    r.eps = 1e-6f;
    auto rows_code = [&](bool write, auto change) {
        brik_qkv_rows x = r;
        change(x);
        return rows(w, "t", write ? &c : nullptr, &b, x, write);
    };
    EXPECT(rows_code(true, [](brik_qkv_rows&) {}) == BRIK_OK);
    EXPECT(rows_code(false, [](brik_qkv_rows&) {}) == BRIK_EINVAL);               // k without k_out
    EXPECT(rows_code(false, [](brik_qkv_rows& x) { x.k_out = at<float>(0x40000); }) == BRIK_OK);
    for (int d : {0, 64, 100, 512, -128}) EXPECT(rows_code(true, [&](brik_qkv_rows& x) { x.head_dim = d; }) == BRIK_EINVAL);
    for (int d : {0, 4, 12, 136, -8}) EXPECT(rows_code(true, [&](brik_qkv_rows& x) { x.rot_dim = d; }) == BRIK_EINVAL);
    for (float e : {-1.f, std::numeric_limits<float>::quiet_NaN(), std::numeric_limits<float>::infinity()})
        EXPECT(rows_code(true, [&](brik_qkv_rows& x) { x.eps = e; }) == BRIK_EINVAL);
    for (int64_t n : {(int64_t)508, (int64_t)514, (int64_t)-512}) EXPECT(rows_code(true, [&](brik_qkv_rows& x) { x.q_stride = n; }) == BRIK_EINVAL);
    EXPECT(rows_code(true, [](brik_qkv_rows& x) { x.flags = 4; }) == BRIK_EINVAL);
    EXPECT(rows_code(true, [](brik_qkv_rows& x) { x.kv_heads = 3; }) == BRIK_EINVAL);
    EXPECT(rows_code(true, [](brik_qkv_rows& x) { x.q_out = nullptr; }) == BRIK_EINVAL);
    EXPECT(rows_code(true, [](brik_qkv_rows& x) { x.v = at<float>(0x10008); }) == BRIK_EALIGN);
    EXPECT(rows_code(true, [](brik_qkv_rows& x) { x.q_out = const_cast<float*>(x.q), x.q_stride = 516; }) == BRIK_EINVAL);
    EXPECT(rows_code(true, [](brik_qkv_rows& x) { x.q_out = const_cast<float*>(x.q), x.q_stride = x.q_out_stride = 516; }) == BRIK_OK);

    // attention
    brik_attn_args a{at<float>(0x100000), at<float>(0x200000), 0, 0, 4, 0, 0.1f, 0.f};
    auto attn_code = [&](auto change) {
        brik_attn_args x = a;
        change(x);
        return attn(w, "t", &c, &b, x);
    };
    EXPECT(attn_code([](brik_attn_args&) {}) == BRIK_OK);
    for (int h : {0, -2, 3, 1 << 20}) EXPECT(attn_code([&](brik_attn_args& x) { x.heads = h; }) == BRIK_EINVAL);
    EXPECT(attn_code([](brik_attn_args& x) { x.window = -1; }) == BRIK_EINVAL);
    EXPECT(attn_code([](brik_attn_args& x) { x.softcap = NAN; }) == BRIK_EINVAL);
    EXPECT(attn_code([](brik_attn_args& x) { x.scale = INFINITY; }) == BRIK_EINVAL);
    EXPECT(attn_code([](brik_attn_args& x) { x.out = nullptr; }) == BRIK_EINVAL);
    EXPECT(attn_code([](brik_attn_args& x) { x.q = at<float>(0x100004); }) == BRIK_EALIGN);
    EXPECT(attn_code([](brik_attn_args& x) { x.out = at<float>(0x100000 + 4 * 512 * 4 - 16); }) == BRIK_EINVAL);
    EXPECT(attn_code([](brik_attn_args& x) { x.out = at<float>(0x100000 + 4 * 512 * 4); }) == BRIK_OK);
    EXPECT(attn_code([](brik_attn_args& x) { x.out = at<float>(0x100000 - 4 * 512 * 4); }) == BRIK_OK);
    EXPECT(attn_code([](brik_attn_args& x) { x.out_stride = 256; }) == BRIK_EINVAL);
    for (int d : {32, 160, 224}) {
        brik_kv_cache x = c;
        x.head_dim = d;
        brik_attn_args y = a;
        EXPECT(cache(w, "t", &x) == BRIK_OK && attn(w, "t", &x, &b, y) == BRIK_EINVAL);
    }
    std::printf(failures ? "%d failure(s)\n" : "ok\n", failures);
    return failures != 0;
}
