// Rows to 8-bit codes and a scale each: s = f32(max|h| / 127), c = floor(h / s + 1/2), h = x or act(gate) x in 64 bits.
//
// A row is held in registers between its maximum and its codes: by a wave up to 1024 values, by a block of 256 or 1024 threads
// up to 4096 or 16384, longer ones are read again. The values go in f32 first, which without a gate is exact; with one, SiLU is within
// 2^-21 of itself. What depends on the last bits is then done in 64: the maximum among the values next to the f32 one, and the codes
// whose f32 quotient lies nearer to a border than its error. A row with values that f32 does not hold to 2^-21 (gates below -64 or
// subnormal, overflow, NaN) and one under GELU take 64 bits throughout. 4 bytes are read a value (8 with a gate), one written: without a gate
// memory bounds it, 8192 x 9728 84 us, 4.75 TB/s, vector instructions in 79 % of the cycles. With one vector instructions do: under SiLU
// 32768 x 768 55 us, 4.1 TB/s and 84 %, 8192 x 9728 251 us (2.9 TB/s); under GELU, two exponentials of 64 bits a value, 121 and 474 us.
// 512 x 2560 4 us and one row 3, a launch's latency.
#include "attn_common.h"
#include "moe_abi.h"

namespace {

constexpr int QV = 4;            // quads of a thread

// g s(y), s the logistic function: SiLU with y = g; tanh-GELU with y = 2 sqrt(2 / pi) (g + 0.044715 g^3), as (1 + tanh z) / 2 = s(2 z).
__device__ __forceinline__ double act64(double g, bool gelu)
{
    const double y = gelu ? 1.5957691216057308 * (g + 0.044715 * g * g * g) : g;
    return g / (1.0 + exp(-y));
}

struct Quad {
    f32x4_t x, g;
};

template <bool GATE>
__device__ __forceinline__ Quad quant_load(const brik_quant_launch& a, int row, int q)
{
    Quad d;
    d.x = *(const f32x4_t*)(a.x + row * a.x_stride + 4 * q);
    if constexpr (GATE) d.g = *(const f32x4_t*)(a.gate + row * a.gate_stride + 4 * q);
    return d;
}

// exp(-g) = 2^t 2^u with t = -g log2(e) rounded and u its rest, so that only the exponential itself, the sum, the reciprocal and two
// products round: 3.5 units of 2^-23 together. Half of the smallest normal gates is subnormal, where a product may be off by a whole unit, but
// there only the two products round. What is left of a subnormal gate has fewer bits than that: GATE_SUBNORMAL tells them.
constexpr int GATE_SUBNORMAL = 0x90;                         // classes of both signs
template <bool GATE>
__device__ __forceinline__ float value32(const Quad& d, int i)
{
    if constexpr (!GATE) return d.x[i];
    const float g = d.g[i], t = -ATTN_LOG2E * g;
    const float u = fmaf(-1.92596299e-8f, g, fmaf(-ATTN_LOG2E, g, -t));          // log2(e) = its f32 + 1.926e-8
    const float e = __builtin_amdgcn_exp2f(t);
    return g * __builtin_amdgcn_rcpf(1.f + fmaf(e, u * 0.693147181f, e)) * d.x[i];
}
template <bool GATE>
__device__ __forceinline__ double value64(const Quad& d, int i, bool gelu)
{
    if constexpr (!GATE) return d.x[i];
    return act64(d.g[i], gelu) * (double)d.x[i];
}

// The larger size, NaN above all.
template <class H>
__device__ __forceinline__ H max_of(H m, H v)
{
    v = v < 0 ? -v : v;
    return v > m || v != v ? v : m;
}

// Over the T threads of a row.
template <int T, class H>
__device__ __forceinline__ H team_max(H m, H* tops)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) m = max_of(m, (H)__shfl_xor(m, o, 64));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
        __syncthreads();
        m = tops[0];
#pragma unroll
        for (int w = 1; w < T / 64; ++w) m = max_of(m, tops[w]);
    }
    return m;
}

// A block of NT threads takes ROWS rows.
template <int NT, int ROWS, bool GATE>
__device__ __forceinline__ void quant_body(const brik_quant_launch& a)
{
    constexpr int T = NT / ROWS;                             // threads of a row
    __shared__ float top32[T > 64 ? T / 64 : 1];
    __shared__ double top64[T > 64 ? T / 64 : 1];
    const int row = blockIdx.x * ROWS + (int)threadIdx.x / T, tid = threadIdx.x % T, quads = row < a.M ? a.K >> 2 : 0;
    const bool whole = a.K >> 2 <= QV * T, gelu = GATE && a.gelu;
    Quad d[QV];
    // f(quad, its number) over the row's quads of this thread
    auto each = [&](bool first, auto f) {
        if (whole) {
#pragma unroll
            for (int v = 0; v < QV; ++v)
                if (tid + v * T < quads) {
                    if (first) d[v] = quant_load<GATE>(a, row, tid + v * T);
                    f(d[v], tid + v * T);
                }
        } else {
            for (int q = tid; q < quads; q += T) f(quant_load<GATE>(a, row, q), q);
        }
    };
    // infinity: f32 does not hold the row
    float m32 = gelu ? __builtin_inff() : 0.f;
    each(true, [&](const Quad& v, int) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float h = fabsf(value32<GATE>(v, i));
            const bool held = h <= 3.0e38f && (!GATE || (v.g[i] >= -64.f && !__builtin_amdgcn_classf(v.g[i], GATE_SUBNORMAL)));
            m32 = fmaxf(m32, held || (!GATE && h <= 3.4028235e38f) ? h : __builtin_inff());
        }
    });
    m32 = team_max<T>(m32, top32);
    const bool held = m32 < __builtin_inff();
    double m = m32;
    if (GATE) {
        double mine = 0;
        const float near = m32 * (1.f - 0x1p-19f);
        each(false, [&](const Quad& v, int) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!held || fabsf(value32<GATE>(v, i)) >= near) mine = max_of(mine, value64<GATE>(v, i, gelu));
        });
        m = team_max<T>(mine, top64);
    }
    // (the quotient in 64 bits is never so near the middle of two f32 values that it rounds another way than the exact one)
    float s = (float)(m / 127.0);
    const bool fine = s <= 3.4028235e38f && m <= 1.7976931348623157e308, some = fine && s >= 0x1p-126f;
    if (!fine) s = __builtin_nanf("");
    else if (!some) s = 0.f;
    if (row < a.M && tid == 0) a.scales[row] = s;
    const float r = some ? 1.f / s : 0.f;
    uint32_t* const to = (uint32_t*)(a.codes + (size_t)row * a.K);
    each(false, [&](const Quad& v, int q) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // |h / s| <= 127: its f32 value, the reciprocal, the product and the sum are off by less than 2^-13 together
            const float u = fmaf(value32<GATE>(v, i), r, 0.5f), f = floorf(u);
            int c = (int)f;
            if ((GATE && !held) || fabsf(u - f - 0.5f) > 0.5f - 0x1p-13f) c = (int)floor(value64<GATE>(v, i, gelu) / (double)s + 0.5);
            w |= (uint32_t)(max(-127, min(127, c)) & 255) << (8 * i);
        }
        to[q] = some ? w : 0u;
    });
}

}  // namespace

#define BRIK_QUANT_I8(NAME, NT, ROWS)                                                                                        \
    extern "C" __global__ __launch_bounds__(NT) void brik_quant_i8_##NAME(brik_quant_launch a) { quant_body<NT, ROWS, false>(a); } \
    extern "C" __global__ __launch_bounds__(NT) void brik_quant_i8_glu_##NAME(brik_quant_launch a) { quant_body<NT, ROWS, true>(a); }
BRIK_QUANT_I8(wave, 256, 4)
BRIK_QUANT_I8(256, 256, 1)
BRIK_QUANT_I8(1024, 1024, 1)
