// Attention over the quantized cache, the plain kernel: one wave per row and query head, 64 keys at a time, a key per lane
// for the scores and a value column per lane for the sums, the running maximum and sum of the softmax in f32.
#include "attn_abi.h"
#include "common.h"

namespace {

template <int FMT>
__device__ __forceinline__ float cached(const uint8_t* code, const uint16_t* sc, const uint16_t* mn, size_t vec, int D, int d)
{
    const size_t g = vec * (size_t)(D / BRIK_GROUP) + d / BRIK_GROUP;
    if constexpr (FMT == FMT_Q8) return (float)((const int8_t*)code)[vec * D + d] * f16_bits_to_f32(sc[g]);
    return fmaf((float)((code[vec * (D / 2) + d / 2] >> (4 * (d & 1))) & 15), f16_bits_to_f32(sc[g]), f16_bits_to_f32(mn[g]));
}

template <int FMT>
__device__ __forceinline__ void plain_body(const brik_attn_launch& a)
{
    __shared__ float q[4][256], p[4][64];
    __shared__ size_t at[4][64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, D = a.c.head_dim;
    const int h = blockIdx.y * 4 + w, t = blockIdx.x;
    const int b = seq_of_row(a.s, t);
    if (b >= a.s.seqs || h >= a.a.heads) return;
    const int kvh = h / (a.a.heads / a.c.heads);
    const int32_t pos = row_position(a.s, b, t);
    for (int d = lane; d < D; d += 64) q[w][d] = a.a.q[t * a.a.q_stride + (size_t)h * D + d];
    const int32_t end = min(pos + 1, a.s.max_len), begin = a.a.window ? max(0, pos - a.a.window + 1) : 0;
    float m = -1e30f, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int32_t j0 = begin; j0 < end; j0 += 64) {
        const int32_t j = j0 + lane;
        const int32_t page = j < end ? brik_page_of(a.s, b, j) : -1;
        const size_t vec = page < 0 ? 0 : brik_vector(a.s, a.c.heads, page, kvh, brik_slot(a.s, j));
        float x = -__builtin_inff();
        if (page >= 0) {
            x = 0.f;
            for (int d = 0; d < D; ++d)
                x = fmaf(q[w][d], cached<FMT>((const uint8_t*)a.c.k, a.c.k_scales, a.c.k_mins, vec, D, d), x);
            x *= a.a.scale;
            if (a.a.softcap > 0.f) x = a.a.softcap * tanhf(x / a.a.softcap);
        }
        float top = x;
        for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
        const float mn = fmaxf(m, top), alpha = expf(m - mn), e = page < 0 ? 0.f : expf(x - mn);
        float sum = e;
        for (int i = 1; i < 64; i <<= 1) sum += __shfl_xor(sum, i);
        l = l * alpha + sum;
        m = mn;
        p[w][lane] = e;
        at[w][lane] = page < 0 ? ~(size_t)0 : vec;
        __builtin_amdgcn_wave_barrier();
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (d >= D) break;
            float acc = o[i] * alpha;
            for (int k = 0; k < 64; ++k)
                if (at[w][k] != ~(size_t)0)
                    acc = fmaf(p[w][k], cached<FMT>((const uint8_t*)a.c.v, a.c.v_scales, a.c.v_mins, at[w][k], D, d), acc);
            o[i] = acc;
        }
        __builtin_amdgcn_wave_barrier();
    }
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < D) a.a.out[t * a.a.out_stride + (size_t)h * D + d] = l == 0.f ? 0.f : o[i] / l;
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void brik_attn_plain_q8(brik_attn_launch a) { plain_body<FMT_Q8>(a); }
extern "C" __global__ __launch_bounds__(256) void brik_attn_plain_q4(brik_attn_launch a) { plain_body<FMT_Q4>(a); }
