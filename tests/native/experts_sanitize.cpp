// Host-code sanitizer run of the experts' and 8-bit products' entry points (the runtime's host code with AddressSanitizer and
// UndefinedBehaviorSanitizer, the kernels the ordinary code object): argument validation without a device, then, on a GPU, a whole layer of few and
// of many tokens with its gradients, products by every kernel with K whole and split, refusals, a recorded step and a workspace
// that moves under it, with loose numeric checks (the parity tests hold the exact ones).
//
// usage: experts_sanitize          (device checks run when a device is present)
//        experts_sanitize nodev    (host checks only)
// Exit status 0 when every check passed.
#include "brik.h"

#include <algorithm>
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
            std::fprintf(stderr, "FAIL line %d: %s (%s)\n", __LINE__, #c, ctx ? brik_last_error(ctx) : ""); \
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
    float* f() const { return static_cast<float*>(p); }
    int32_t* i() const { return static_cast<int32_t*>(p); }
    int8_t* c() const { return static_cast<int8_t*>(p); }
};

std::vector<float> normal(size_t n, int seed)
{
    std::mt19937 rng(seed);
    std::normal_distribution<float> d;
    std::vector<float> v(n);
    for (float& x : v) x = d(rng);
    return v;
}

template <class T>
std::vector<T> download(const Dev& b, size_t n)
{
    std::vector<T> v(n);
    OK(brik_d2h(ctx, v.data(), b.p, n * sizeof(T)));
    return v;
}

void without_device()
{
    brik_moe_route_args r{};
    CHECK(brik_moe_route(nullptr, &r) == BRIK_EINVAL);
    CHECK(brik_moe_route_grad(nullptr, &r, nullptr, nullptr) == BRIK_EINVAL);
    CHECK(brik_moe_sort(nullptr, nullptr, 1, 1, 1, nullptr, nullptr, nullptr) == BRIK_EINVAL);
    CHECK(brik_moe_dispatch(nullptr, nullptr, nullptr, nullptr, nullptr, 1, 1, 4) == BRIK_EINVAL);
    CHECK(brik_moe_combine(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1, 1, 4) == BRIK_EINVAL);
    CHECK(brik_moe_combine_grad(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1, 1, 4) == BRIK_EINVAL);
    CHECK(brik_quantize_i8(nullptr, nullptr, 0, nullptr, 0, 0, nullptr, nullptr, 1, 32) == BRIK_EINVAL);
    CHECK(brik_matmul_t_i8(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1, 32, 1) == BRIK_EINVAL);
    CHECK(brik_moe_matmul_t_i8(nullptr, nullptr, nullptr, 1, nullptr, 1, nullptr, nullptr, nullptr, nullptr, 1, 1, 32, 1) == BRIK_EINVAL);
}

// A layer: routed, tokens quantized, gate and up by experts, SwiGLU into 8 bits, down by experts, back; the experts are all the same, so
// that what comes back is the sum of a token's weights times one feed-forward of it. Then the gradients.
void layer(int T, int E, int k, bool bias, int flags)
{
    const int H = 96, F = 64, n = T * k;
    const auto x = normal((size_t)T * H, 1), one = normal((size_t)2 * F * H, 2), down = normal((size_t)H * F, 3);
    std::vector<float> wgu, wd;
    for (int e = 0; e < E; ++e) {
        wgu.insert(wgu.end(), one.begin(), one.end());
        wd.insert(wd.end(), down.begin(), down.end());
    }
    Dev xd(x), logits(normal((size_t)T * E, 4)), b(normal(E, 5)), gus(wgu), ds(wd), guc((size_t)E * 2 * F * H), gusc((size_t)4 * E * 2 * F), dc((size_t)E * H * F), dsc((size_t)4 * E * H);
    OK(brik_quantize_i8(ctx, gus.f(), 0, nullptr, 0, 0, guc.c(), gusc.f(), E * 2 * F, H));
    OK(brik_quantize_i8(ctx, ds.f(), 0, nullptr, 0, 0, dc.c(), dsc.f(), E * H, F));
    Dev ids(4 * (size_t)n), w(4 * (size_t)n), off(4 * (size_t)(E + 1)), src(4 * (size_t)n), slot(4 * (size_t)n);
    brik_moe_route_args r{};
    r.logits = logits.f();
    r.bias = bias ? b.f() : nullptr;
    r.ids = ids.i();
    r.weights = w.f();
    r.row_off = off.i();
    r.src = src.i();
    r.slot = slot.i();
    r.tokens = T;
    r.experts = E;
    r.k = k;
    r.flags = flags;
    r.scale = 1.f;
    OK(brik_moe_route(ctx, &r));
    const auto order = download<int32_t>(slot, n), rows = download<int32_t>(off, E + 1);
    CHECK(rows[0] == 0 && rows[E] == n && std::is_sorted(rows.begin(), rows.end()));
    OK(brik_moe_sort(ctx, ids.i(), T, k, E, off.i(), src.i(), slot.i()));
    CHECK(download<int32_t>(slot, n) == order);
    Dev xc((size_t)T * H), xs(4 * (size_t)T), gu((size_t)4 * n * 2 * F), hc((size_t)n * F), hs(4 * (size_t)n), y((size_t)4 * n * H), out((size_t)4 * T * H), dense((size_t)4 * T * H);
    OK(brik_quantize_i8(ctx, xd.f(), 0, nullptr, 0, 0, xc.c(), xs.f(), T, H));
    OK(brik_moe_matmul_t_i8(ctx, xc.c(), xs.f(), T, src.i(), k, off.i(), guc.c(), gusc.f(), gu.f(), E, n, H, 2 * F));
    for (int gelu : {BRIK_JOB_ACT_GELU, 0}) OK(brik_quantize_i8(ctx, gu.f() + F, 2 * F, gu.f(), 2 * F, gelu, hc.c(), hs.f(), n, F));
    OK(brik_moe_matmul_t_i8(ctx, hc.c(), hs.f(), n, nullptr, 1, off.i(), dc.c(), dsc.f(), y.f(), E, n, F, H));
    OK(brik_moe_combine(ctx, y.f(), slot.i(), w.f(), nullptr, out.f(), T, k, H));
    // the same by dense products of the first expert
    OK(brik_matmul_t_i8(ctx, xc.c(), xs.f(), guc.c(), gusc.f(), nullptr, gu.f(), T, H, 2 * F));
    OK(brik_quantize_i8(ctx, gu.f() + F, 2 * F, gu.f(), 2 * F, 0, hc.c(), hs.f(), T, F));
    OK(brik_matmul_t_i8(ctx, hc.c(), hs.f(), dc.c(), dsc.f(), nullptr, dense.f(), T, F, H));
    const auto got = download<float>(out, (size_t)T * H), want = download<float>(dense, (size_t)T * H), weights = download<float>(w, n);
    for (int t = 0; t < T; ++t) {
        double sum = 0;
        for (int j = 0; j < k; ++j) sum += weights[(size_t)t * k + j];
        for (int i = 0; i < H; ++i) {
            const size_t at = (size_t)t * H + i;
            if (!(std::fabs(got[at] - sum * want[at]) <= 1e-4 * (1 + std::fabs(sum * want[at])))) {
                CHECK(!"a layer of equal experts");
                return;
            }
        }
    }
    Dev dw(4 * (size_t)n), dl((size_t)4 * T * E), sorted((size_t)4 * n * H);
    OK(brik_moe_dispatch(ctx, xd.f(), slot.i(), w.f(), sorted.f(), T, k, H));
    OK(brik_moe_combine_grad(ctx, xd.f(), y.f(), slot.i(), w.f(), y.f(), dw.f(), T, k, H));
    CHECK(download<float>(y, (size_t)n * H) == download<float>(sorted, (size_t)n * H));
    OK(brik_moe_route_grad(ctx, &r, dw.f(), dl.f()));
    for (float v : download<float>(dl, (size_t)T * E)) CHECK(std::isfinite(v));
}

void products()
{
    const int M = 70, K = 1120, N = 45;
    std::mt19937 rng(7);
    std::vector<int8_t> x((size_t)M * K), w((size_t)N * K);
    for (auto& v : x) v = (int8_t)(rng() & 255);
    for (auto& v : w) v = (int8_t)(rng() & 255);
    Dev xd(x), wd(w), one(std::vector<float>(M, 1.f)), y((size_t)4 * M * N);
    const std::vector<float> res = normal((size_t)M * N, 1);
    Dev rd(res);
    for (int kernel = 0; kernel <= 12; ++kernel)
        for (int splits : {0, 3}) {
            OK(brik_set_option(ctx, BRIK_OPT_I8_KERNEL, kernel));
            OK(brik_set_option(ctx, BRIK_OPT_I8_SPLITS, splits));
            OK(brik_matmul_t_i8(ctx, xd.c(), one.f(), wd.c(), one.f(), rd.f(), y.f(), M, K, N));
            const auto got = download<float>(y, (size_t)M * N);
            for (int m = 0; m < M; ++m)
                for (int n = 0; n < N; ++n) {
                    int sum = 0;
                    for (int i = 0; i < K; ++i) sum += x[(size_t)m * K + i] * w[(size_t)n * K + i];
                    if (got[(size_t)m * N + n] != (float)sum + res[(size_t)m * N + n]) {
                        CHECK(!"sums and added values");
                        m = M;
                        break;
                    }
                }
        }
    OK(brik_set_option(ctx, BRIK_OPT_I8_KERNEL, 0));
    OK(brik_set_option(ctx, BRIK_OPT_I8_SPLITS, 0));
}

void refusals()
{
    Dev b((size_t)1 << 16);
    int8_t* const odd = b.c() + 4;
    auto refused = [](int code, int r) { CHECK(r == code && std::strlen(brik_last_error(ctx)) > 0); };
    brik_moe_route_args r{};
    r.logits = b.f();
    r.ids = b.i();
    r.weights = b.f();
    r.tokens = 4;
    r.experts = 8;
    r.k = 9;
    refused(BRIK_EINVAL, brik_moe_route(ctx, &r));
    refused(BRIK_EINVAL, brik_moe_route(ctx, nullptr));
    refused(BRIK_EINVAL, brik_moe_route_grad(ctx, &r, b.f(), b.f()));
    refused(BRIK_EINVAL, brik_moe_route_grad(ctx, nullptr, b.f(), b.f()));
    refused(BRIK_EINVAL, brik_moe_sort(ctx, b.i(), 4, 2, BRIK_MOE_EXPERTS + 1, b.i(), b.i(), b.i()));
    refused(BRIK_EINVAL, brik_moe_dispatch(ctx, b.f(), b.i(), nullptr, b.f(), 2, 2, 6));
    refused(BRIK_EINVAL, brik_moe_combine(ctx, b.f(), b.i(), nullptr, nullptr, nullptr, 2, 2, 8));
    refused(BRIK_EALIGN, brik_moe_combine_grad(ctx, reinterpret_cast<float*>(odd), b.f(), b.i(), nullptr, b.f(), b.f(), 2, 2, 8));
    refused(BRIK_EINVAL, brik_quantize_i8(ctx, b.f(), 0, nullptr, 0, 1, b.c(), b.f(), 2, 64));
    refused(BRIK_EALIGN, brik_quantize_i8(ctx, b.f(), 0, nullptr, 0, 0, odd, b.f(), 2, 64));
    refused(BRIK_EINVAL, brik_matmul_t_i8(ctx, b.c(), b.f(), b.c(), b.f(), nullptr, b.f(), 2, 33, 4));
    refused(BRIK_EINVAL, brik_moe_matmul_t_i8(ctx, b.c(), b.f(), 3, nullptr, 1, b.i(), b.c(), b.f(), b.f(), 2, 4, 64, 4));
    refused(BRIK_EINVAL, brik_set_option(ctx, BRIK_OPT_I8_KERNEL, 13));
    refused(BRIK_EINVAL, brik_set_option(ctx, BRIK_OPT_I8_SPLITS, 65));
    OK(brik_moe_combine(ctx, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 2, 8));
    OK(brik_matmul_t_i8(ctx, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 64, 4));
}

// A recorded product with split K, replayed; refused once a larger call has moved the workspace; a capture that would grow it.
void recorded()
{
    const int M = 130, K = 4096, N = 1100;
    Dev x(std::vector<int8_t>((size_t)M * K, 1)), w(std::vector<int8_t>((size_t)N * K, 1)), one(std::vector<float>(N, 1.f)), y((size_t)4 * M * N);
    auto call = [&](int rows, int splits) {
        OK(brik_set_option(ctx, BRIK_OPT_I8_KERNEL, 9));
        OK(brik_set_option(ctx, BRIK_OPT_I8_SPLITS, splits));
        const int rc = brik_matmul_t_i8(ctx, x.c(), one.f(), w.c(), one.f(), nullptr, y.f(), rows, K, N);
        OK(brik_set_option(ctx, BRIK_OPT_I8_KERNEL, 0));
        OK(brik_set_option(ctx, BRIK_OPT_I8_SPLITS, 0));
        return rc;
    };
    auto flat = [&](int rows) {
        for (float v : download<float>(y, (size_t)rows * N)) CHECK(v == 4096.f);
    };
    OK(call(40, 4));
    flat(40);
    brik_graph *g = nullptr, *none = nullptr;
    OK(brik_graph_begin(ctx));
    OK(call(40, 4));
    OK(brik_graph_end(ctx, &g));
    for (int i = 0; i < 3; ++i) {
        OK(brik_graph_launch(ctx, g));
        flat(40);
    }
    OK(brik_graph_begin(ctx));
    CHECK(call(M, 16) == BRIK_EINVAL);                                      // the workspace would grow inside a capture
    if (brik_graph_end(ctx, &none) == BRIK_OK && none) brik_graph_destroy(ctx, none);
    OK(call(M, 16));
    flat(M);
    CHECK(brik_graph_launch(ctx, g) == BRIK_EINVAL);                        // the workspace has moved
    brik_graph_destroy(ctx, g);
    OK(call(40, 4));
    flat(40);
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
        std::printf("round %d: layers\n", round); std::fflush(stdout);
        layer(1, 8, 2, false, BRIK_ROUTE_RENORM);
        layer(33, 8, 4, true, BRIK_ROUTE_SIGMOID);
        layer(700, 20, 3, true, 0);
        std::printf("round %d: products\n", round); std::fflush(stdout);
        products();
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
