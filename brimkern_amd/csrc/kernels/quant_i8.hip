// Rows to 8-bit codes and a scale each: s = f32(max|h| / 127), c = floor(h / s + 1/2), h = x or act(gate) x in 64 bits.
//
// A row is held in registers between its maximum and its codes: by a wave up to 1024 values, by a block of 256 or 1024 threads
// up to 4096 or 16384, longer ones are read twice. A code is taken from an f32 quotient where that is further from the next
// border than its error (|h / s| <= 127: the reciprocal, its product and the addition are off by less than 2^-15 together), else
// from the 64-bit one, whose border no f32 quotient meets without being on it. Bound by memory: 4 bytes read a value (8 with a
// gate), one written.
#include "attn_common.h"
#include "moe_abi.h"

namespace {

constexpr int QV = 4;            // quads of a thread

__device__ __forceinline__ double act64(double g, bool gelu)
{
    if (gelu) return 0.5 * g * (1.0 + tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)));
    return g / (1.0 + exp(-g));
}

__device__ __forceinline__ float magnitude(float h) { return fabsf(h); }
__device__ __forceinline__ double magnitude(double h) { return fabs(h); }

template <bool GATE>
struct QuantValue {
    typedef float type;
};
template <>
struct QuantValue<true> {
    typedef double type;
};

template <bool GATE>
__device__ __forceinline__ void quant_load(const brik_quant_launch& a, int row, int q, typename QuantValue<GATE>::type (&h)[4])
{
    const f32x4_t x = *(const f32x4_t*)(a.x + row * a.x_stride + 4 * q);
    if constexpr (GATE) {
        const f32x4_t g = *(const f32x4_t*)(a.gate + row * a.gate_stride + 4 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = act64(g[i], a.gelu) * (double)x[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = x[i];
    }
}

// max that NaN wins.
template <class H>
__device__ __forceinline__ H max_of(H m, H v)
{
    v = magnitude(v);
    return v > m || v != v ? v : m;
}

template <class H>
__device__ __forceinline__ uint32_t codes_of(const H (&h)[4], float s, float r)
{
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float u = fmaf((float)h[i], r, 0.5f), f = floorf(u);
        int c = (int)f;
        if (fabsf(u - f - 0.5f) > 0.5f - 0x1p-13f) c = (int)floor((double)h[i] / (double)s + 0.5);
        c = max(-127, min(127, c));
        w |= (uint32_t)(c & 255) << (8 * i);
    }
    return w;
}

// ROWS rows of a block of NT threads; whole: the row fits the registers.
template <int NT, int ROWS, bool GATE>
__device__ __forceinline__ void quant_body(const brik_quant_launch& a)
{
    typedef typename QuantValue<GATE>::type H;
    constexpr int T = NT / ROWS;                             // threads of a row
    const int row = blockIdx.x * ROWS + (int)threadIdx.x / T, tid = threadIdx.x % T, quads = a.K >> 2;
    const bool real = row < a.M;
    H h[QV][4], m = 0;
    const bool whole = quads <= QV * T;
    if (real && whole) {
#pragma unroll
        for (int v = 0; v < QV; ++v)
            if (tid + v * T < quads) {
                quant_load<GATE>(a, row, tid + v * T, h[v]);
#pragma unroll
                for (int i = 0; i < 4; ++i) m = max_of(m, h[v][i]);
            }
    } else if (real) {
        for (int q = tid; q < quads; q += T) {
            quant_load<GATE>(a, row, q, h[0]);
#pragma unroll
            for (int i = 0; i < 4; ++i) m = max_of(m, h[0][i]);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) m = max_of(m, (H)__shfl_xor(m, o, 64));
    if constexpr (T > 64) {
        __shared__ H tops[T / 64];
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
        __syncthreads();
        m = tops[0];
#pragma unroll
        for (int w = 1; w < T / 64; ++w) m = max_of(m, tops[w]);
    }
    if (!real) return;
    // the quotient in 64 bits, rounded once more: two f32 values' quotient is not so near a border of f32 that this shows
    float s = (float)((double)m / 127.0);
    const bool fine = magnitude(s) <= 3.4028235e38f, some = fine && s >= 0x1p-126f;
    if (!fine) s = __builtin_nanf("");
    else if (!some) s = 0.f;
    if (tid == 0) a.scales[row] = s;
    const float r = some ? 1.f / s : 0.f;
    uint32_t* const to = (uint32_t*)(a.codes + (size_t)row * a.K);
    if (whole) {
#pragma unroll
        for (int v = 0; v < QV; ++v)
            if (tid + v * T < quads) to[tid + v * T] = some ? codes_of(h[v], s, r) : 0u;
    } else {
        for (int q = tid; q < quads; q += T) {
            quant_load<GATE>(a, row, q, h[0]);
            to[q] = some ? codes_of(h[0], s, r) : 0u;
        }
    }
}

}  // namespace

#define BRIK_QUANT_I8(NAME, NT, ROWS)                                                                                        \
    extern "C" __global__ __launch_bounds__(NT) void brik_quant_i8_##NAME(brik_quant_launch a) { quant_body<NT, ROWS, false>(a); } \
    extern "C" __global__ __launch_bounds__(NT) void brik_quant_i8_glu_##NAME(brik_quant_launch a) { quant_body<NT, ROWS, true>(a); }
BRIK_QUANT_I8(wave, 256, 4)
BRIK_QUANT_I8(256, 256, 1)
BRIK_QUANT_I8(1024, 1024, 1)
