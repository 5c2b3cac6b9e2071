// Joins the partial results of split keys: out = sum_s f_s O_s / sum_s f_s l_s with f_s = exp2(M_s - max M), the slots in order
// (the same bits every time). A block per row and head; its threads are (quad of values) x (every n-th slot).
#include "attn_common.h"

extern "C" __global__ __launch_bounds__(256) void brik_attn_join(brik_attn_launch a)
{
    __shared__ float f[256];
    __shared__ f32x4_t sums[256];
    const int D = a.c.head_dim, quads = D / 4, groups = 256 / quads, slots = a.prefix_splits + a.own_splits;
    const int h = blockIdx.y, t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    if (a.s.row_off && t >= a.s.row_off[a.s.seqs]) return;          // behind the last sequence
    const size_t all = (size_t)a.s.rows * a.a.heads, row = (size_t)t * a.a.heads + h;
    // every wave: the reference exponent, then the weights (slots <= 256)
    float M = ATTN_NONE;
    for (int s = lane; s < slots; s += 64) M = fmaxf(M, a.ml[2 * (s * all + row)]);
    for (int m = 1; m < 64; m <<= 1) M = fmaxf(M, __shfl_xor(M, m));
    float L = 0.f;
    for (int s = lane; s < slots; s += 64) {
        const float l = a.ml[2 * (s * all + row) + 1], w = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(a.ml[2 * (s * all + row)] - M);
        f[s] = w;                                                    // every wave writes the same
        L += l * w;
    }
    for (int m = 1; m < 64; m <<= 1) L += __shfl_xor(L, m);
    __syncthreads();
    const int g = tid / quads, d = 4 * (tid - g * quads);
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (g < groups)
        for (int s = g; s < slots; s += groups)
            if (f[s] != 0.f) v += *(const f32x4_t*)(a.part + (s * all + row) * D + d) * f[s];
    sums[tid] = v;
    __syncthreads();
    if (g != 0) return;
    for (int k = 1; k < groups; ++k) v += sums[k * quads + tid];
    *(f32x4_t*)(a.a.out + t * a.a.out_stride + (size_t)h * D + d) = L == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : v / L;
}
