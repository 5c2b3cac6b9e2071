// The argument checks of the experts' and 8-bit products' entry points, and how their calls are divided over the device, without one.
// Prints "ok" and returns 0 when every check holds.
#include "../../brimkern_amd/csrc/moe_check.h"
#include "../../brimkern_amd/csrc/moe_plan.h"

#include <cstdint>
#include <cstdio>
#include <limits>
#include <random>

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
    const int most = std::numeric_limits<int>::max(), least = std::numeric_limits<int>::min();

    // routing
    const brik_moe_route_args good{at<float>(0x1000), nullptr, 0, at<int32_t>(0x2000), at<float>(0x3000), nullptr, nullptr, nullptr, 4, 8, 2, 0, 1.f, 0};
    auto route_is = [&](int code, bool grad, auto change) {
        brik_moe_route_args r = good;
        change(r);
        EXPECT(route(w, "t", r, grad) == code);
        return r;
    };
    EXPECT(route_is(BRIK_OK, false, [](brik_moe_route_args&) {}).logit_stride == 8);
    route_is(BRIK_OK, true, [](brik_moe_route_args& r) { r.weights = nullptr; });
    route_is(BRIK_OK, false, [](brik_moe_route_args& r) { r.k = BRIK_MOE_K, r.experts = BRIK_MOE_EXPERTS; });
    route_is(BRIK_OK, false, [](brik_moe_route_args& r) { r.tokens = 0, r.logits = nullptr, r.ids = nullptr, r.weights = nullptr; });
    for (int v : {-1, least, most, 1 << 24}) route_is(BRIK_EINVAL, false, [&](brik_moe_route_args& r) { r.tokens = v; });
    for (int v : {-1, least, most, 9, 65}) route_is(BRIK_EINVAL, false, [&](brik_moe_route_args& r) { r.k = v; });
    for (int v : {-1, least, most, 1, 1025}) route_is(BRIK_EINVAL, false, [&](brik_moe_route_args& r) { r.experts = v; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.tokens = (1 << 24) - 1, r.k = 65; });
    route_is(BRIK_OK, false, [](brik_moe_route_args& r) { r.tokens = (1 << 24) - 1, r.k = 64, r.experts = 64, r.logit_stride = 64; });      // 2^30 - 64 slots
    for (float v : {std::numeric_limits<float>::quiet_NaN(), std::numeric_limits<float>::infinity()})
        route_is(BRIK_EINVAL, false, [&](brik_moe_route_args& r) { r.scale = v; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.flags = 4; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.reserved = 1; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.logit_stride = 7; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.logit_stride = -8; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.logits = nullptr; });
    route_is(BRIK_EINVAL, true, [](brik_moe_route_args& r) { r.ids = nullptr; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.weights = nullptr; });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.src = at<int32_t>(0x4000); });
    route_is(BRIK_EINVAL, false, [](brik_moe_route_args& r) { r.row_off = r.src = at<int32_t>(0x4000); });
    route_is(BRIK_OK, false, [](brik_moe_route_args& r) { r.row_off = r.src = r.slot = at<int32_t>(0x4000); });
    route_is(BRIK_EALIGN, false, [](brik_moe_route_args& r) { r.row_off = r.src = r.slot = at<int32_t>(0x4002); });
    route_is(BRIK_EALIGN, false, [](brik_moe_route_args& r) { r.bias = at<float>(0x4001); });

    // rows
    const int32_t* slot = at<int32_t>(0x1000);
    EXPECT(spread(w, "t", 3, 2, 8, slot, nullptr) == BRIK_OK && spread(w, "t", 3, 2, 0, slot, nullptr) == BRIK_OK);
    for (int v : {-4, 2, 7, least}) EXPECT(spread(w, "t", 3, 2, v, slot, nullptr) == BRIK_EINVAL);
    EXPECT(spread(w, "t", 3, 2, 8, nullptr, nullptr) == BRIK_EINVAL && spread(w, "t", 3, 0, 8, nullptr, nullptr) == BRIK_OK);
    EXPECT(spread(w, "t", 3, 2, 8, slot, at<float>(0x1002)) == BRIK_EALIGN && spread(w, "t", 1 << 24, 2, 8, slot, nullptr) == BRIK_EINVAL);

    // quantization
    auto quant_is = [&](int code, int flags, auto change) {
        brik_quant_launch q{at<float>(0x1000), nullptr, 0, 0, at<int8_t>(0x2000), at<float>(0x3000), 5, 64, 0};
        change(q);
        EXPECT(quantize_i8(w, "t", q, flags) == code);
    };
    quant_is(BRIK_OK, 0, [](brik_quant_launch&) {});
    quant_is(BRIK_OK, BRIK_JOB_ACT_GELU, [](brik_quant_launch& q) { q.gate = q.x, q.gate_stride = 128, q.x_stride = 68; });
    quant_is(BRIK_EINVAL, 1, [](brik_quant_launch&) {});
    for (int v : {-1, least, 1 << 22, most}) quant_is(BRIK_EINVAL, 0, [&](brik_quant_launch& q) { q.M = v; });
    for (int v : {-32, 33, 16, least}) quant_is(BRIK_EINVAL, 0, [&](brik_quant_launch& q) { q.K = v; });
    for (long v : {-64l, 32l, 66l}) quant_is(BRIK_EINVAL, 0, [&](brik_quant_launch& q) { q.x_stride = v; });
    quant_is(BRIK_EINVAL, 0, [](brik_quant_launch& q) { q.x = nullptr; });
    quant_is(BRIK_EINVAL, 0, [](brik_quant_launch& q) { q.codes = nullptr; });
    quant_is(BRIK_EINVAL, 0, [](brik_quant_launch& q) { q.scales = nullptr; });
    quant_is(BRIK_EALIGN, 0, [](brik_quant_launch& q) { q.gate = at<float>(0x1008); });
    quant_is(BRIK_OK, 0, [](brik_quant_launch& q) { q.M = 0, q.x = nullptr; });

    // products
    brik_i8_launch p{};
    p.x = at<int8_t>(0x1000), p.w = at<int8_t>(0x2000), p.xs = at<float>(0x3000), p.ws = at<float>(0x4000), p.y = at<float>(0x5000);
    p.M = 10, p.K = 64, p.N = 7;
    auto product_is = [&](int code, bool moe, auto change) {
        brik_i8_launch x = p;
        if (moe) x.E = 3, x.row_off = at<int32_t>(0x6000), x.x_rows = 10, x.k = 1;
        change(x);
        EXPECT(product_i8(w, "t", x, moe) == code);
    };
    for (bool moe : {false, true}) {
        product_is(BRIK_OK, moe, [](brik_i8_launch&) {});
        product_is(BRIK_OK, moe, [](brik_i8_launch& x) { x.K = BRIK_I8_K; });
        product_is(BRIK_OK, moe, [](brik_i8_launch& x) { x.K = 0, x.x = x.w = nullptr; });
        product_is(BRIK_OK, moe, [](brik_i8_launch& x) { x.N = 0, x.y = nullptr; });
        for (int v : {-1, least, (1 << 30) + 1, most - 16, most}) product_is(BRIK_EINVAL, moe, [&](brik_i8_launch& x) { x.M = v, x.x_rows = most; });
        product_is(BRIK_OK, moe, [](brik_i8_launch& x) { x.M = 1 << 30, x.x_rows = 1 << 30; });
        for (int v : {-32, 16, 33, BRIK_I8_K + 32, most, least}) product_is(BRIK_EINVAL, moe, [&](brik_i8_launch& x) { x.K = v; });
        for (int v : {-1, 1 << 22, most, least}) product_is(BRIK_EINVAL, moe, [&](brik_i8_launch& x) { x.N = v; });
        product_is(BRIK_EINVAL, moe, [](brik_i8_launch& x) { x.N = 40000, x.K = 131040; });
        product_is(BRIK_EINVAL, moe, [](brik_i8_launch& x) { x.w = nullptr; });
        product_is(BRIK_EINVAL, moe, [](brik_i8_launch& x) { x.xs = nullptr; });
        product_is(BRIK_EINVAL, moe, [](brik_i8_launch& x) { x.ws = nullptr, x.K = 0; });
        product_is(BRIK_EALIGN, moe, [](brik_i8_launch& x) { x.w = at<int8_t>(0x2008); });
        product_is(BRIK_EALIGN, moe, [](brik_i8_launch& x) { x.y = at<float>(0x5002); });
    }
    product_is(BRIK_EINVAL, true, [](brik_i8_launch& x) { x.row_off = nullptr; });
    product_is(BRIK_EINVAL, true, [](brik_i8_launch& x) { x.x_rows = 9; });
    product_is(BRIK_EINVAL, true, [](brik_i8_launch& x) { x.E = -1; });
    product_is(BRIK_EINVAL, true, [](brik_i8_launch& x) { x.src = x.row_off, x.k = 0; });
    product_is(BRIK_EINVAL, true, [](brik_i8_launch& x) { x.src = x.row_off, x.x_rows = 1 << 26; });       // offsets past 32 bits
    product_is(BRIK_OK, true, [](brik_i8_launch& x) { x.src = x.row_off, x.x_rows = 3, x.k = 4; });
    product_is(BRIK_OK, true, [](brik_i8_launch& x) { x.src = x.row_off, x.x_rows = 0, x.x = nullptr, x.xs = nullptr; });

    // plans, over sizes of all magnitudes: K and the rows are covered once, kernels are of the call's kind
    std::mt19937_64 rng(1);
    auto some = [&](double from, double to) { return (int)std::exp(std::log(from) + (std::log(to) - std::log(from)) * (double)(rng() % 100000) / 99999); };
    for (int i = 0; i < 200000; ++i) {
        brik_route_launch r{};
        r.r.tokens = some(1, 16777215), r.r.k = some(1, 64);
        brik_plan::moe_chunks(r, i % 2 ? 512 : 0);
        EXPECT(r.chunks >= 1 && r.chunks <= BRIK_MOE_CHUNKS && (long)r.chunks * r.chunk >= r.r.tokens && (long)(r.chunks - 1) * r.chunk < r.r.tokens);
        const int E = some(1, 1024), k = std::min(E, some(1, 64)), t = brik_plan::moe_route(E, k), lanes = t < 5 ? 16 : 64;
        EXPECT(t < 10 && (lanes << t % 5) >= E && (t >= 5 || k <= 16));
        EXPECT((64 << brik_plan::moe_lanes(E, 64)) >= E && brik_plan::moe_lanes(E, 64) < 5);
        brik_i8_launch a{};
        a.M = some(1, 300000), a.K = 32 * some(1, 4095), a.N = std::min(some(1, 300000), (int)((1ll << 32) / a.K) - 1);
        a.E = i % 3 ? 0 : some(1, 1024);
        const int forced = i % 5 ? 0 : 1 + (int)(rng() % brik_plan::kI8Count), splits = i % 7 ? 0 : 1 + (int)(rng() % 64);
        const int n = brik_plan::i8_plan(a, forced, splits);
        if (n < 0 || n >= brik_plan::kI8Count) {
            EXPECT(false);
            continue;
        }
        const brik_plan::I8Kernel& g = brik_plan::kI8Kernels[n];
        EXPECT(g.kind == brik_plan::I8_FEW || (g.kind == brik_plan::I8_MOE) == (a.E > 0));
        EXPECT(forced == 0 || n == forced - 1 || brik_plan::kI8Kernels[forced - 1].kind == (a.E ? brik_plan::I8_TILE : brik_plan::I8_MOE));
        EXPECT((long)a.col_tiles * g.bn >= a.N && (long)(a.col_tiles - 1) * g.bn < a.N);
        long blocks = 0;
        if (brik_plan::i8_fits(a, n, blocks)) EXPECT(blocks * g.threads <= 4294967295l && blocks == (long)a.row_tiles * a.col_tiles * a.splits);
        else EXPECT(blocks >= 1 << 22);
        const long steps = (a.K + 63) / 64;
        EXPECT(a.steps >= 1 && a.splits >= 1 && (long)a.splits * a.steps >= steps && (long)(a.splits - 1) * a.steps < steps);
        EXPECT(a.E == 0 || a.splits == 1);
        if (g.kind == brik_plan::I8_FEW) EXPECT(a.row_tiles == std::max(1, a.E));
        else if (a.E == 0) EXPECT((long)a.row_tiles * g.bm >= a.M && (long)(a.row_tiles - 1) * g.bm < a.M);
        else {
            // however the rows lie among the experts: each of them ends at most one tile early
            long tiles = 0, left = a.M;
            for (int e = 0; e < a.E; ++e) {
                const long rows = e + 1 < a.E ? std::min<long>(left, rng() % (2 * a.M / a.E + 2)) : left;
                tiles += (rows + g.bm - 1) / g.bm;
                left -= rows;
            }
            EXPECT(tiles <= a.row_tiles);
        }
    }
    // forced onto many experts and channels: more threads than a launch has
    brik_i8_launch many{};
    many.E = 65536, many.M = 65536, many.K = 64, many.N = 1280;
    long blocks = 0;
    EXPECT(!brik_plan::i8_fits(many, brik_plan::i8_plan(many, 4, 0), blocks) && blocks == 65536 * 80l);
    EXPECT(brik_plan::i8_fits(many, brik_plan::i8_plan(many, 1, 0), blocks) && blocks == 65536 * 80l);
    std::printf(failures ? "%d failures\n" : "ok\n", failures);
    return failures != 0;
}
