// Joins the partial results of split keys: out = sum_s f_s O_s / sum_s f_s l_s with f_s = exp2(M_s - max M), the slots in order
// (the same bits every time). A block per row and head; its threads are (quad of values) x (every n-th slot). Bound by latency:
// 4 us for 32 heads of one row by 32 slots, 6 us for 1024 rows and heads by the lengths of 32 sequences. Joining in the blocks
// that finish last instead cost more than this launch (a fence across the XCDs: 32 us).
#include "attn_common.h"

extern "C" __global__ __launch_bounds__(256) void brik_attn_join(brik_attn_launch a)
{
    __shared__ f32x4_t sums[256];
    const int D = a.c.head_dim, quads = D / 4, groups = 256 / quads;
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const size_t all = (size_t)a.s.rows * a.a.heads, row = (size_t)t * a.a.heads + h;
    // vector of slot s: the prefix's and static ones are `all` apart, a sequence's parts 16
    int slots = a.prefix_splits + a.own_splits;
    size_t own = 0;
    if (a.own_blocks) {
        const Share share(a);                                        // first: its loads and the search's go together
        int b = uniform(seq_of_row(a.s, t)), start;
        if (b >= a.s.seqs) return;                                   // of no sequence
        const Seq q = Share::find(a, b, 0, start);
        const int G = a.a.heads / a.c.heads, kvh = h / G;
        if (t < q.row || (t - q.row + 1) * G > 16) return;           // more rows than the call was said to have
        const int first = start / share.each, count = q.n ? (start + q.n - 1) / share.each - first + 1 : 0;
        if (count == 1 && a.prefix_splits == 0) return;              // written by its block
        slots = a.prefix_splits + count;
        own = a.prefix_splits * all + ((size_t)kvh * (a.own_blocks + a.s.seqs) + first + b) * 16 + (t - q.row) * G + (h - kvh * G);
    } else if (!brik_row_taken(a.s, t)) {
        return;
    }
    auto vec = [&](int s) { return a.own_blocks && s >= a.prefix_splits ? own + (size_t)(s - a.prefix_splits) * 16 : s * all + row; };
    // every wave: the reference exponent, then the weights (64 slots in a register, more are read twice)
    f32x2_t ml0 = {ATTN_NONE, 0.f};
    if (lane < slots) ml0 = *(const f32x2_t*)(a.ml + 2 * vec(lane));
    float M = ml0.x;
#pragma unroll 1
    for (int s = lane + 64; s < slots; s += 64) M = fmaxf(M, a.ml[2 * vec(s)]);
    M = half_max(M);
    float p, q;
    half_pair(M, p, q);
    M = fmaxf(p, q);
    const int g = tid / quads, d = 4 * (tid - g * quads);
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
#pragma unroll 1
    for (int s0 = 0; s0 < slots; s0 += 64) {                         // 64 slots at a time, one a lane
        float l = 0.f, f = -1.f;
        if (s0 + lane < slots) {
            const f32x2_t ml = s0 ? *(const f32x2_t*)(a.ml + 2 * vec(s0 + lane)) : ml0;
            l = ml.y;
            f = l == 0.f ? -1.f : __builtin_amdgcn_exp2f(ml.x - M);  // -1: nothing was written there
        }
        L += quarters_sum(sum16(l * f));
        const int n = min(64, slots - s0);
#pragma unroll 1
        // four loads at once, whatever their weights (decoding one sequence 13.8 -> 12.7 and 65.7 -> 63.5 us; a slot that was not written
        // is not added, one whose weight is 0 is: it may hold NaN); as often in every lane: weights come from other lanes
        for (int s1 = 0; s1 < n; s1 += 4 * groups) {
            f32x4_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = *(const f32x4_t*)(a.part + vec(s0 + min(s1 + i * groups + g, n - 1)) * D + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int s = s1 + i * groups + g;
                const float w = __shfl(f, min(s, 63));
                if (g < groups && s < n && !(w < 0.f)) v += x[i] * w;
            }
        }
    }
    sums[tid] = v;
    __syncthreads();
    if (g != 0) return;
    for (int k = 1; k < groups; ++k) v += sums[k * quads + tid];
    *(f32x4_t*)(a.a.out + t * a.a.out_stride + (size_t)h * D + d) = L == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : v / L;
}

// The same for up to 16 static slots: a group of D / 4 lanes per row and head, which loops over the slots by itself. (2048 rows
// of 32 heads by 2 slots, 170 MB: with the kernels before it 138 us, 200 by a block for each.)
extern "C" __global__ __launch_bounds__(256) void brik_attn_join_few(brik_attn_launch a)
{
    const int D = a.c.head_dim, quads = D / 4, g = threadIdx.x / quads, d = 4 * (threadIdx.x - g * quads);
    const int t = blockIdx.x, h = blockIdx.y * (256 / quads) + g, slots = a.prefix_splits + a.own_splits;
    if (g >= 256 / quads || h >= a.a.heads || !brik_row_taken(a.s, t)) return;
    const size_t all = (size_t)a.s.rows * a.a.heads, row = (size_t)t * a.a.heads + h;
    float M = ATTN_NONE;
#pragma unroll 4
    for (int s = 0; s < slots; ++s) M = fmaxf(M, a.ml[2 * (s * all + row)]);
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
#pragma unroll 1
    for (int s0 = 0; s0 < slots; s0 += 4) {
        f32x4_t x[4];
        f32x2_t ml[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const size_t at = min(s0 + i, slots - 1) * all + row;
            x[i] = *(const f32x4_t*)(a.part + at * D + d);
            ml[i] = *(const f32x2_t*)(a.ml + 2 * at);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + i >= slots || ml[i].y == 0.f) continue;        // nothing was written there
            const float f = __builtin_amdgcn_exp2f(ml[i].x - M);
            L += ml[i].y * f;
            v += x[i] * f;
        }
    }
    *(f32x4_t*)(a.a.out + t * a.a.out_stride + (size_t)h * D + d) = L == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : v / L;
}
