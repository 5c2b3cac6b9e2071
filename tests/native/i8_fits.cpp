// The kernel of a product of 8-bit integers, where one would need more blocks than a launch has and another does not. Prints "ok" and
// returns 0 when every check holds.
#include "../../brimkern_amd/csrc/moe_check.h"
#include "../../brimkern_amd/csrc/moe_plan.h"

#include <cstdio>
#include <random>

int main()
{
    using namespace brik_plan;
    int failures = 0;
    auto call = [](int E, int M, int K, int N) {
        brik_i8_launch a{};
        a.E = E, a.M = M, a.K = K, a.N = N;
        return a;
    };
    // whether the call is taken, and whether any kernel of its kind would take it
    auto check = [&](const brik_i8_launch& a) {
        long blocks = 0;
        brik_i8_launch own = a;
        const bool taken = i8_fits(own, i8_plan(own, 0, 0), blocks);
        for (int f = 1; f <= kI8Count && !taken; ++f) {
            brik_i8_launch other = a;
            const int t = i8_plan(other, f, 1);
            if ((a.E && kI8Kernels[t].kind == I8_TILE) || (!a.E && kI8Kernels[t].kind == I8_MOE)) continue;
            if (i8_fits(other, t, blocks)) {
                std::printf("E=%d M=%d K=%d N=%d is refused, %s takes it\n", a.E, a.M, a.K, a.N, kI8Kernels[t].name);
                ++failures;
                break;
            }
        }
        return taken;
    };
    for (const brik_i8_launch& a : {call(65536, 1, 32, 2048), call(4096, 8, 32, 131072), call(33480, 78193, 32, 60840), call(65536, 1 << 20, 32, 16384),
                                    call(65536, 40, 0, 1 << 20), call(0, 1 << 30, 32, 1), call(0, 1 << 30, 0, 1), call(0, 1 << 30, 32, 256)})
        if (!check(a)) {
            std::printf("E=%d M=%d K=%d N=%d is refused\n", a.E, a.M, a.K, a.N);
            ++failures;
        }
    std::mt19937_64 rng(1);
    auto some = [&](double from, double to) { return (int)std::exp(std::log(from) + (std::log(to) - std::log(from)) * (double)(rng() % 100000) / 99999); };
    long held = 0;
    for (int i = 0; i < 600000 && failures < 20; ++i) {
        const int E = i % 3 ? some(1, 65536) : 0, M = some(1, 1 << 30), K = i % 50 ? 32 * some(1, 4095) : 0;
        const int most = (int)std::min<long>((1l << 22) - 1, K ? ((1l << 32) - 1) / K : 1l << 30);
        const brik_i8_launch a = call(E, M, K, some(1, most));
        if (4.0 * a.M * a.N + ((double)a.M + (double)std::max(1, E) * a.N) * K < 288e9) check(a), ++held;      // what the device holds
    }
    if (held < 200000) ++failures;
    std::printf(failures ? "%d failures\n" : "ok\n", failures);
    return failures != 0;
}
