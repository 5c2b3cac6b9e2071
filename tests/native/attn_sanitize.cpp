// Host-code sanitizer run of the attention side's entry points (the runtime's host code with AddressSanitizer and
// UndefinedBehaviorSanitizer, the kernels the ordinary code object): argument validation without a device, then, on a GPU, writes, reads
// and attention of every kind (decoding whole, split and shared out, prompts by every tile, a prefix, a part of a batch), refusals,
// a recorded step and a workspace that moves under it, with loose numeric checks (the parity tests hold the exact ones).
//
// usage: attn_sanitize          (device checks run when a device is present)
//        attn_sanitize nodev    (host checks only)
// Exit status 0 when every check passed.
#include "brik.h"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

extern "C" const char* __asan_default_options()
{
    // the HIP runtime keeps allocations until exit; the check here is for memory errors
    return "detect_leaks=0:verify_asan_link_order=0:abort_on_error=1";
}

namespace {

int fails = 0;
brik_ctx* ctx = nullptr;

#define CHECK(c)                                                                                          \
    do {                                                                                                  \
        if (!(c)) {                                                                                       \
            std::fprintf(stderr, "FAIL line %d: %s (%s)\n", __LINE__, #c, brik_last_error(ctx));          \
            ++fails;                                                                                      \
        }                                                                                                 \
    } while (0)
#define OK(c) CHECK((c) == BRIK_OK)

// A device buffer freed at scope end.
struct Dev {
    void* p = nullptr;
    explicit Dev(size_t bytes) { OK(brik_alloc(ctx, bytes ? bytes : 16, &p)); }
    template <class T>
    explicit Dev(const std::vector<T>& v) : Dev(v.size() * sizeof(T)) { OK(brik_h2d(ctx, p, v.data(), v.size() * sizeof(T))); }
    ~Dev() { if (p) brik_free(ctx, p); }
    Dev(const Dev&) = delete;
    Dev& operator=(const Dev&) = delete;
    template <class T> T* as() const { return static_cast<T*>(p); }
};

std::vector<float> normal(size_t n, int seed)
{
    std::mt19937 rng(seed);
    std::normal_distribution<float> d;
    std::vector<float> v(n);
    for (float& x : v) x = d(rng);
    return v;
}

std::vector<float> download(const void* p, size_t n)
{
    std::vector<float> v(n);
    OK(brik_d2h(ctx, v.data(), p, n * sizeof(float)));
    return v;
}

constexpr int KV = 4, H = 8, D = 64, P = 16;

struct Cache {
    Dev k, v, ks, vs, km, vm;
    brik_kv_cache c{};
    Cache(int fmt, int pages)
        : k((size_t)pages * KV * P * D), v((size_t)pages * KV * P * D), ks((size_t)pages * KV * P * D / 16), vs((size_t)pages * KV * P * D / 16),
          km((size_t)pages * KV * P * D / 16), vm((size_t)pages * KV * P * D / 16)
    {
        c = {fmt, KV, D, P, pages, 0, k.p, v.p, ks.as<uint16_t>(), vs.as<uint16_t>(), nullptr, nullptr};
        if (fmt == BRIK_FMT_Q4) {
            c.k_mins = km.as<uint16_t>();
            c.v_mins = vm.as<uint16_t>();
        }
    }
};

// Sequences of rows[b] rows and len[b] tokens (the prefix among them), the pages of each in a row, those of the prefix first.
struct Batch {
    std::vector<int32_t> off, len, table, pre;
    brik_kv_batch b{};
    int pages;
    Dev *doff = nullptr, *dlen = nullptr, *dtab = nullptr, *dpre = nullptr;
    Batch(const std::vector<int>& rows, const std::vector<int>& lens, int prefix = 0, int lead = 0)
    {
        int cols = 1, most = 1, longest = 0;
        for (size_t i = 0; i < lens.size(); ++i) {
            cols = std::max(cols, (lens[i] - prefix + P - 1) / P);
            most = std::max(most, rows[i]);
            longest = std::max(longest, lens[i]);
        }
        off.push_back(lead);
        for (int r : rows) off.push_back(off.back() + r);
        for (int n : lens) len.push_back(n);
        pages = (prefix + P - 1) / P;
        for (int i = 0; i < pages; ++i) pre.push_back(i);
        for (size_t i = 0; i < lens.size(); ++i)
            for (int k = 0; k < cols; ++k) table.push_back(pages++);
        doff = new Dev(off);
        dlen = new Dev(len);
        dtab = new Dev(table);
        dpre = new Dev(pre);
        b = {(int)rows.size(), off.back() + lead, doff->as<int32_t>(), dlen->as<int32_t>(), dtab->as<int32_t>(), cols, longest, most, prefix,
             prefix ? dpre->as<int32_t>() : nullptr};
    }
    ~Batch() { delete doff; delete dlen; delete dtab; delete dpre; }
    Batch(const Batch&) = delete;
    Batch& operator=(const Batch&) = delete;
};

void without_device()
{
    brik_kv_cache c{};
    brik_kv_batch b{};
    brik_qkv_rows r{};
    brik_attn_args a{};
    CHECK(brik_qk_norm_rope(nullptr, &b, &r) == BRIK_EINVAL);
    CHECK(brik_kv_write(nullptr, &c, &b, &r) == BRIK_EINVAL);
    CHECK(brik_kv_read(nullptr, &c, &b, nullptr, nullptr) == BRIK_EINVAL);
    CHECK(brik_attention(nullptr, &c, &b, &a) == BRIK_EINVAL);
}

// All tokens of the batch written as rows, read back, and attention of its last rows: a row that sees one token gives its values.
void run(int fmt, const std::vector<int>& rows, const std::vector<int>& lens, int prefix = 0, int lead = 0)
{
    Batch t(rows, lens, prefix, lead);
    Cache cache(fmt, t.pages);
    const int seqs = (int)rows.size(), n = t.b.rows;
    // the tokens: the prefix as a sequence of its own, then every sequence's own ones
    std::vector<int> own;
    int total = 0;
    for (int x : lens) {
        own.push_back(x - prefix);
        total += x - prefix;
    }
    std::vector<int32_t> aoff = {0}, alen;
    for (int x : own) {
        aoff.push_back(aoff.back() + x);
        alen.push_back(x);
    }
    Dev doff(aoff), dlen(alen), k(normal((size_t)(total + prefix) * KV * D, 1)), v(normal((size_t)(total + prefix) * KV * D, 2));
    brik_kv_batch all = {seqs, total, doff.as<int32_t>(), dlen.as<int32_t>(), t.b.table, t.b.table_cols, t.b.max_len, 0, 0, nullptr};
    brik_qkv_rows r{};
    r.k = k.as<float>();
    r.v = v.as<float>();
    r.kv_heads = KV;
    r.head_dim = D;
    OK(brik_kv_write(ctx, &cache.c, &all, &r));
    if (prefix) {
        std::vector<int32_t> pl = {prefix};
        Dev dpl(pl);
        brik_kv_batch pre = {1, prefix, nullptr, dpl.as<int32_t>(), t.b.prefix_table, (prefix + P - 1) / P, prefix, 0, 0, nullptr};
        brik_qkv_rows pr = r;
        pr.k += (size_t)total * KV * D;
        pr.v += (size_t)total * KV * D;
        OK(brik_kv_write(ctx, &cache.c, &pre, &pr));
        OK(brik_sync(ctx));
    }
    Dev kb((size_t)total * KV * D * 4), vb((size_t)total * KV * D * 4);
    OK(brik_kv_read(ctx, &cache.c, &all, kb.as<float>(), vb.as<float>()));
    const auto v0 = download(v.p, (size_t)total * KV * D), v1 = download(vb.p, (size_t)total * KV * D);
    double num = 0, den = 0;
    for (size_t i = 0; i < v0.size(); ++i) {
        num += (v0[i] - v1[i]) * (v0[i] - v1[i]);
        den += v0[i] * v0[i];
    }
    CHECK(std::sqrt(num / den) < (fmt == BRIK_FMT_Q8 ? 0.01 : 0.12));
    Dev q(normal((size_t)n * H * D, 3)), qo((size_t)n * H * D * 4), freq(std::vector<float>(D / 2, 0.01f));
    std::vector<float> nan((size_t)n * H * D, std::nanf(""));
    Dev out(nan);
    brik_qkv_rows turn{};
    turn.q = q.as<float>();
    turn.q_out = qo.as<float>();
    turn.heads = H;
    turn.head_dim = D;
    turn.inv_freq = freq.as<float>();
    turn.rot_dim = D;
    OK(brik_qk_norm_rope(ctx, &t.b, &turn));
    for (int tile : {0, 16, 128, 256}) {
        for (int splits : {0, 1, 5}) {
            OK(brik_set_option(ctx, BRIK_OPT_ATTN_ROWS, tile));
            OK(brik_set_option(ctx, BRIK_OPT_ATTN_SPLITS, splits));
            brik_attn_args a = {qo.as<float>(), out.as<float>(), 0, 0, H, 0, 0.125f, 0.f};
            OK(brik_attention(ctx, &cache.c, &t.b, &a));
            const auto y = download(out.p, (size_t)n * H * D);
            for (int row = 0; row < n; ++row) {
                const bool mine = row >= lead && row < t.off.back();
                for (int i = 0; i < H * D; ++i) {
                    const float x = y[(size_t)row * H * D + i];
                    if (mine ? !(std::fabs(x) < 8.f) : !std::isnan(x)) {
                        CHECK(!"outputs of rows, and of no others");
                        return;
                    }
                }
            }
            for (int b = 0; b < seqs; ++b)
                if (rows[b] == lens[b] && !prefix)                           // its first row sees its first token only
                    for (int h = 0; h < H; ++h)
                        for (int i = 0; i < D; ++i)
                            CHECK(std::fabs(y[((size_t)t.off[b] * H + h) * D + i] - v1[((size_t)aoff[b] * KV + h / (H / KV)) * D + i]) < 1e-5);
        }
    }
    OK(brik_set_option(ctx, BRIK_OPT_ATTN_ROWS, 0));
    OK(brik_set_option(ctx, BRIK_OPT_ATTN_SPLITS, 0));
}

void refusals()
{
    Batch t({1}, {5});
    Cache cache(BRIK_FMT_Q8, t.pages);
    Dev q((size_t)H * D * 4), out((size_t)H * D * 4);
    brik_attn_args a = {q.as<float>(), out.as<float>(), 0, 0, H, 0, 0.1f, 0.f};
    auto code = [&](auto change) {
        brik_kv_cache c = cache.c;
        brik_kv_batch b = t.b;
        brik_attn_args x = a;
        change(c, b, x);
        const int r = brik_attention(ctx, &c, &b, &x);
        CHECK(r == BRIK_OK || std::strlen(brik_last_error(ctx)) > 0);
        return r;
    };
    CHECK(code([](auto&, auto&, auto&) {}) == BRIK_OK);
    CHECK(code([](auto&, auto&, auto& x) { x.heads = 7; }) == BRIK_EINVAL);
    CHECK(code([](auto&, auto&, auto& x) { x.out = nullptr; }) == BRIK_EINVAL);
    CHECK(code([](auto& c, auto&, auto&) { c.page = 24; }) == BRIK_EINVAL);
    CHECK(code([](auto&, auto& b, auto&) { b.rows = 1 << 24; }) == BRIK_EINVAL);
    CHECK(code([](auto&, auto& b, auto&) { b.kv_len = nullptr; }) == BRIK_EINVAL);
    CHECK(code([](auto&, auto&, auto& x) { x.q = reinterpret_cast<const float*>(reinterpret_cast<const char*>(x.q) + 4); }) == BRIK_EALIGN);
    CHECK(code([](auto&, auto& b, auto&) { b.rows = 0; }) == BRIK_OK);
    CHECK(brik_attention(ctx, nullptr, &t.b, &a) == BRIK_EINVAL);
    CHECK(brik_attention(ctx, &cache.c, nullptr, &a) == BRIK_EINVAL);
    CHECK(brik_attention(ctx, &cache.c, &t.b, nullptr) == BRIK_EINVAL);
    CHECK(brik_kv_write(ctx, &cache.c, &t.b, nullptr) == BRIK_EINVAL);
}

// A recorded call, replayed; refused once a larger call has moved the workspace; a capture that would grow it.
void recorded()
{
    Batch t({1}, {900}), big({1}, {40000});
    Cache cache(BRIK_FMT_Q8, big.pages);
    Dev q(normal((size_t)H * D, 4)), out((size_t)H * D * 4), codes(std::vector<int8_t>((size_t)big.pages * KV * P * D, 1));
    std::vector<uint16_t> one((size_t)big.pages * KV * P * D / 32, 0x2400);
    OK(brik_d2d(ctx, cache.c.k, codes.p, (size_t)big.pages * KV * P * D));
    OK(brik_d2d(ctx, cache.c.v, codes.p, (size_t)big.pages * KV * P * D));
    OK(brik_h2d(ctx, cache.c.k_scales, one.data(), one.size() * 2));
    OK(brik_h2d(ctx, cache.c.v_scales, one.data(), one.size() * 2));
    brik_attn_args a = {q.as<float>(), out.as<float>(), 0, 0, H, 0, 0.125f, 0.f};
    auto call = [&](Batch& b, int splits) {
        OK(brik_set_option(ctx, BRIK_OPT_ATTN_SPLITS, splits));
        const int r = brik_attention(ctx, &cache.c, &b.b, &a);
        OK(brik_set_option(ctx, BRIK_OPT_ATTN_SPLITS, 0));
        return r;
    };
    auto flat = [&] {
        for (float x : download(out.p, (size_t)H * D)) CHECK(std::fabs(x - 0x1p-6f) < 1e-6f);
    };
    OK(call(t, 8));
    flat();
    brik_graph* g = nullptr;
    OK(brik_graph_begin(ctx));
    OK(call(t, 8));
    OK(brik_graph_end(ctx, &g));
    for (int i = 0; i < 3; ++i) {
        OK(brik_graph_launch(ctx, g));
        flat();
    }
    Dev wide((size_t)2000 * H * D * 4), wout((size_t)2000 * H * D * 4);
    brik_kv_batch b = big.b;
    b.seqs = 1;
    b.rows = b.max_rows = 2000;
    b.row_off = nullptr;
    OK(brik_h2d(ctx, wide.p, std::vector<float>((size_t)2000 * H * D, 0.f).data(), (size_t)2000 * H * D * 4));
    brik_attn_args wa = {wide.as<float>(), wout.as<float>(), 0, 0, H, 0, 0.125f, 0.f};
    OK(brik_set_option(ctx, BRIK_OPT_ATTN_SPLITS, 12));
    brik_graph* none = nullptr;
    OK(brik_graph_begin(ctx));
    CHECK(brik_attention(ctx, &cache.c, &b, &wa) == BRIK_EINVAL);           // the workspace would grow inside a capture
    const int ended = brik_graph_end(ctx, &none);
    if (ended == BRIK_OK && none) brik_graph_destroy(ctx, none);
    OK(brik_attention(ctx, &cache.c, &b, &wa));
    OK(brik_set_option(ctx, BRIK_OPT_ATTN_SPLITS, 0));
    CHECK(brik_graph_launch(ctx, g) == BRIK_EINVAL);                        // the workspace has moved
    brik_graph_destroy(ctx, g);
    OK(call(t, 8));
    flat();
}

}  // namespace

int main(int argc, char** argv)
{
    int devices = 0;
    without_device();
    if ((argc > 1 && std::strcmp(argv[1], "nodev") == 0) || brik_device_count(&devices) != BRIK_OK || devices == 0) {
        std::printf("host checks only (no device): %d failure(s)\n", fails);
        return fails ? 1 : 0;
    }
    for (int round = 0; round < 2; ++round) {
        OK(brik_create(0, &ctx));
        if (!ctx) return 1;
        for (int fmt : {BRIK_FMT_Q8, BRIK_FMT_Q4}) {
            std::printf("round %d, format %d: decoding\n", round, fmt); std::fflush(stdout);
            run(fmt, {1, 1, 0, 1}, {300, 1, 20, 77});
            std::printf("round %d, format %d: prompts\n", round, fmt); std::fflush(stdout);
            run(fmt, {90, 3, 200}, {90, 3, 333});
            std::printf("round %d, format %d: prefix\n", round, fmt); std::fflush(stdout);
            run(fmt, {1, 5, 40}, {150, 131, 190}, 100);
            std::printf("round %d, format %d: part of a batch\n", round, fmt); std::fflush(stdout);
            run(fmt, {2, 30}, {2, 500}, 0, 17);
            std::printf("round %d, format %d: shared out\n", round, fmt); std::fflush(stdout);
            run(fmt, std::vector<int>(64, 1), [] {
                std::vector<int> n(64);
                for (int i = 0; i < 64; ++i) n[i] = 1 + 30 * i;
                return n;
            }());
        }
        std::printf("round %d: refusals\n", round); std::fflush(stdout);
        refusals();
        std::printf("round %d: recorded\n", round); std::fflush(stdout);
        recorded();
        OK(brik_sync(ctx));
        brik_destroy(ctx);
        ctx = nullptr;
    }
    std::printf("device checks done: %d failure(s)\n", fails);
    return fails ? 1 : 0;
}
