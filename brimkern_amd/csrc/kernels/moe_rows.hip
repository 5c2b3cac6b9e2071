// Tokens' rows to their experts' rows and back, weighted and summed, and the gradient of that.
//
//   dispatch: xs[slot_j] = w_j x     combine: out = res + sum_j w_j y[slot_j]     gradient: dy[slot_j] = w_j dout, dw_j = dout . y[slot_j]
//
// All three go by token: a row of the token is read once and its k sorted rows are named by the slots, so nothing is read
// twice and no sum depends on an order. Bound by memory: a token's row and its k sorted ones, read or written once. Rows of 2048: 16384
// tokens, 6 places, three quarters of them elsewhere, there 66 us (5.1 TB/s) and back 100 (4.7); 4096 tokens, 8 places, the gradient 104
// (5.5 TB/s) and the sum of its rows 79; 256 tokens 6 each, the latency of slot, row, store.
#include "attn_common.h"
#include "moe_abi.h"

namespace {

constexpr int SPREAD_J = 8;      // sorted rows on the way at once

// The slots of a token from place j0 on, -1 where there are none.
__device__ __forceinline__ void slots_of(const brik_spread_launch& a, int t, int j0, int (&s)[SPREAD_J], float (&w)[SPREAD_J])
{
    const int all = a.tokens * a.k;
    const size_t at = (size_t)t * a.k + j0;
#pragma unroll
    for (int j = 0; j < SPREAD_J; ++j) {
        const int v = j0 + j < a.k ? a.slot[at + j] : -1;
        s[j] = uniform((uint32_t)v < (uint32_t)all ? v : -1);
        w[j] = s[j] < 0 ? 0.f : a.weights ? a.weights[at + j] : 1.f;
    }
}

__device__ __forceinline__ float dot4(f32x4_t a, f32x4_t b) { return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, a.w * b.w))); }

}  // namespace

extern "C" __global__ __launch_bounds__(256) void brik_rows_dispatch(brik_spread_launch a)
{
    const int t = blockIdx.x, step = 256 * gridDim.y;
    for (int j0 = 0; j0 < a.k; j0 += SPREAD_J) {
        int s[SPREAD_J];
        float w[SPREAD_J];
        slots_of(a, t, j0, s, w);
        for (int q = blockIdx.y * 256 + threadIdx.x; q < a.quads; q += step) {
            const f32x4_t v = ((const f32x4_t*)a.x)[(size_t)t * a.quads + q];
#pragma unroll
            for (int j = 0; j < SPREAD_J; ++j)
                if (s[j] >= 0) ((f32x4_t*)a.rows)[(size_t)s[j] * a.quads + q] = a.weights ? v * w[j] : v;
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void brik_rows_combine(brik_spread_launch a)
{
    const int t = blockIdx.x, step = 256 * gridDim.y;
    for (int q = blockIdx.y * 256 + threadIdx.x; q < a.quads; q += step) {
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
        if (a.res) sum = ((const f32x4_t*)a.res)[(size_t)t * a.quads + q];
        for (int j0 = 0; j0 < a.k; j0 += SPREAD_J) {
            int s[SPREAD_J];
            float w[SPREAD_J];
            slots_of(a, t, j0, s, w);
            f32x4_t v[SPREAD_J];
#pragma unroll
            for (int j = 0; j < SPREAD_J; ++j)
                if (s[j] >= 0) v[j] = ((const f32x4_t*)a.y)[(size_t)s[j] * a.quads + q];
#pragma unroll
            for (int j = 0; j < SPREAD_J; ++j)
                if (s[j] >= 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] = fmaf(w[j], v[j][i], sum[i]);
                }
        }
        ((f32x4_t*)a.out)[(size_t)t * a.quads + q] = sum;
    }
}

// A block has the whole row of a token: the products' sums stay in it.
extern "C" __global__ __launch_bounds__(256) void brik_rows_combine_grad(brik_spread_launch a)
{
    __shared__ float part[4][SPREAD_J];
    const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j0 = 0; j0 < a.k; j0 += SPREAD_J) {
        int s[SPREAD_J];
        float w[SPREAD_J], dot[SPREAD_J];
        slots_of(a, t, j0, s, w);
#pragma unroll
        for (int j = 0; j < SPREAD_J; ++j) dot[j] = 0.f;
        for (int q = threadIdx.x; q < a.quads; q += 256) {
            const f32x4_t d = ((const f32x4_t*)a.x)[(size_t)t * a.quads + q];
            f32x4_t v[SPREAD_J];
            if (a.dweights) {
#pragma unroll
                for (int j = 0; j < SPREAD_J; ++j)
                    if (s[j] >= 0) v[j] = ((const f32x4_t*)a.y)[(size_t)s[j] * a.quads + q];
#pragma unroll
                for (int j = 0; j < SPREAD_J; ++j)
                    if (s[j] >= 0) dot[j] += dot4(d, v[j]);
            }
            if (a.rows) {
#pragma unroll
                for (int j = 0; j < SPREAD_J; ++j)
                    if (s[j] >= 0) ((f32x4_t*)a.rows)[(size_t)s[j] * a.quads + q] = d * w[j];
            }
        }
        if (!a.dweights) continue;
#pragma unroll
        for (int j = 0; j < SPREAD_J; ++j) {
            const float v = quarters_sum(sum16(dot[j]));
            if (lane == 0) part[wave][j] = v;
        }
        __syncthreads();
        if (threadIdx.x < SPREAD_J && j0 + (int)threadIdx.x < a.k) {
            const int j = threadIdx.x;
            a.dweights[(size_t)t * a.k + j0 + j] = (part[0][j] + part[1][j]) + (part[2][j] + part[3][j]);
        }
        __syncthreads();
    }
}
