// Routing: the k best experts of every token and their weights, the assignments sorted by expert, the gradient of the logits.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  ids = k largest;  w_j = c s_j,  or c s_j / sum of the chosen
//
// A wave holds a token's logits, V neighbours a lane, and takes the largest k times: the maximum of order-preserving keys over
// the lanes, then the lowest lane that has it (its experts are the lowest), then the lowest of its V. Keys are the logits'
// own bits without a bias (s grows with l), else s + bias in 64 bits, high word first.
//
// Sorting is counting: every wave ranks 64 assignments at a time among those of the same expert by ballots over the bits of the
// expert's number, so the order is that of the assignments, whatever runs when. Chunks of tokens are counted as they are routed;
// a second launch adds up the counts of the chunks before its own and writes the rows. Few assignments are routed and sorted
// by one block.
#include "attn_common.h"
#include "moe_abi.h"

namespace {

constexpr int MOE_NT = 1024, MOE_NW = MOE_NT / 64;

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
    v = max16u(v);
    const auto q = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)q[0], (uint32_t)q[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (uint32_t)uniform((int)max((uint32_t)h[0], (uint32_t)h[1]));
}
__device__ __forceinline__ float wave_fmax(float v)
{
    v = BRIK_DPP_MAX(v, DPP_QUAD_1032);
    v = BRIK_DPP_MAX(v, DPP_QUAD_2301);
    v = BRIK_DPP_MAX(v, DPP_ROW_ROR4);
    v = BRIK_DPP_MAX(v, DPP_ROW_ROR8);
    return quarters_max(v);
}
__device__ __forceinline__ float wave_fsum(float v) { return quarters_sum(sum16(v)); }
__device__ __forceinline__ double wave_dsum(double v)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// A logit that counts: NaN as -infinity, -0 as 0 (equal, so a tie).
__device__ __forceinline__ float logit_of(float l) { return l == l ? l + 0.f : -__builtin_inff(); }

// Order-preserving bits; 0 for what is never chosen (-infinity and NaN).
__device__ __forceinline__ uint32_t key_of(float l) { return l == -__builtin_inff() ? 0u : order_key(l); }
__device__ __forceinline__ uint64_t key_of(double s)
{
    if (s != s || s == -__builtin_inf()) return 0;
    const uint64_t b = __builtin_bit_cast(uint64_t, s);
    return b >> 63 ? ~b : b | (1ull << 63);
}

__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }

// exp(min(l, 0) - m) / (1 + exp(-|l|)): the sigmoid of l times exp(-m), which stays in range where all of them are tiny.
__device__ __forceinline__ float sigmoid_part(float l, float m) { return expf(fminf(l, 0.f) - m) / (1.f + expf(-fabsf(l))); }

// One token by a wave: lane j < k gets the j-th id (-1: none) and its logit (-infinity).
template <int V, bool BIAS>
__device__ __forceinline__ void choose(const brik_route_launch& a, int t, float (&l)[V], int& id, float& mine)
{
    const int lane = threadIdx.x & 63, E = a.r.experts, e0 = lane * V;
    const float* const row = a.r.logits + t * a.r.logit_stride;
    uint32_t hi[V], lo[BIAS ? V : 1];
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = e0 + i < E ? logit_of(row[e0 + i]) : -__builtin_inff();
    if constexpr (BIAS) {
        double s[V], sum = 0, top = 0;
        const bool sig = a.r.flags & BRIK_ROUTE_SIGMOID;
        if (!sig) {
            float m = l[0];
#pragma unroll
            for (int i = 1; i < V; ++i) m = fmaxf(m, l[i]);
            top = wave_fmax(m);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s[i] = sig ? sigmoid64(l[i]) : exp(l[i] - top);
            sum += s[i];
        }
        if (!sig) sum = wave_dsum(sum);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool real = e0 + i < E && l[i] != -__builtin_inff();
            const uint64_t key = real ? key_of((sig ? s[i] : s[i] / sum) + (double)a.r.bias[e0 + i]) : 0;
            hi[i] = (uint32_t)(key >> 32);
            lo[i] = (uint32_t)key;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) hi[i] = key_of(l[i]);
    }
    id = -1;
    mine = -__builtin_inff();
    for (int j = 0; j < a.r.k; ++j) {
        uint32_t best = hi[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, hi[i]);
        const uint32_t top = wave_max_u32(best);
        if (top == 0) break;                                 // none left
        uint64_t have = __ballot(best == top);
        uint32_t low = 0;
        if constexpr (BIAS) {
            uint32_t b = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) b = max(b, hi[i] == top ? lo[i] : 0u);
            low = (have & (have - 1)) ? wave_max_u32(best == top ? b : 0u)
                                      : (uint32_t)__builtin_amdgcn_readlane((int)b, __ffsll((unsigned long long)have) - 1);
            have = __ballot(best == top && b == low);
        }
        const int owner = __ffsll((unsigned long long)have) - 1;
        int at = 0;
        float v = 0.f;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) {
            bool is = hi[i] == top;
            if constexpr (BIAS) is = is && lo[i] == low;
            if (is) {
                at = i;
                v = l[i];
            }
        }
        at = __builtin_amdgcn_readlane(at, owner);
        v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), owner));
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (lane == owner && i == at) hi[i] = 0;
        if (lane == j) {
            id = owner * V + at;
            mine = v;
        }
    }
}

// The weight of lane j's expert, before the scale; 0 where there is none.
template <int V>
__device__ __forceinline__ float weight_of(const brik_route_launch& a, const float (&l)[V], int id, float mine)
{
    const bool sig = a.r.flags & BRIK_ROUTE_SIGMOID, renorm = a.r.flags & BRIK_ROUTE_RENORM, have = id >= 0;
    if (sig) {
        const float m = renorm ? wave_fmax(fminf(mine, 0.f)) : 0.f;
        const float p = have ? sigmoid_part(mine, m) : 0.f;
        const float sum = renorm ? wave_fsum(p) : 1.f;       // (by all lanes)
        return have ? p / sum : 0.f;
    }
    float top = mine, sum;
    if (renorm) {
        top = wave_fmax(mine);
        sum = wave_fsum(have ? expf(mine - top) : 0.f);
    } else {
        top = l[0];
#pragma unroll
        for (int i = 1; i < V; ++i) top = fmaxf(top, l[i]);
        top = wave_fmax(top);
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) part += expf(l[i] - top);
        sum = wave_fsum(part);
    }
    return have ? expf(mine - top) / sum : 0.f;
}

// Lanes that hold the same id as this one, of the lanes that are `in`.
__device__ __forceinline__ uint64_t peers_of(int id, bool in, int bits)
{
    uint64_t m = __ballot(in);
    for (int b = 0; b < bits; ++b) {
        const bool set = (id >> b) & 1;
        const uint64_t s = __ballot(set);
        m &= set ? s : ~s;
    }
    return m;
}

// The rows of the assignments [a0, a1) of `n`, by a block of MOE_NT threads. With one chunk their counts are all there are;
// else `counts` holds those of every chunk.
__device__ __forceinline__ void sort_chunk(const int32_t* ids, int a0, int a1, int n, int E, const int32_t* counts, int chunks, int chunk,
                                           int32_t* row_off, int32_t* src, int32_t* slot)
{
    __shared__ int cnt[MOE_NW * BRIK_MOE_EXPERTS];
    __shared__ int all_part[MOE_NT], before_part[MOE_NT], wave_tot[MOE_NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    int bits = 0;
    while ((1 << bits) < E) ++bits;
    for (int i = tid; i < MOE_NW * E; i += MOE_NT) cnt[i] = 0;
    // the chunks' counts: thread by expert, groups of threads by chunk
    if (chunks > 1) {
        const int Eb = max(bits, 6), g = tid >> Eb, groups = MOE_NT >> Eb, e = tid & ((1 << Eb) - 1);
        int all = 0, before = 0;
        if (e < E) {
#pragma unroll 8
            for (int r = g; r < chunks; r += groups) {
                const int v = counts[r * E + e];
                all += v;
                before += r < chunk ? v : 0;
            }
        }
        all_part[tid] = all;
        before_part[tid] = before;
    }
    __syncthreads();
    const int per = ((a1 - a0 + MOE_NT - 1) / MOE_NT) * 64, w0 = a0 + wave * per, w1 = min(a1, w0 + per);
    int* const mine = cnt + wave * E;
    for (int b = w0; b < w1; b += 64) {
        const int i = b + lane, id = i < w1 ? ids[i] : -1;
        const bool in = (uint32_t)id < (uint32_t)E;
        const uint64_t peers = peers_of(id, in, bits);
        if (in && __ffsll((unsigned long long)peers) - 1 == lane) mine[id] += __popcll(peers);
    }
    __syncthreads();
    // base of every expert, and of every wave within it
    int all = 0, own = 0, before = 0;
    if (tid < E) {
        for (int w = 0; w < MOE_NW; ++w) {
            const int v = cnt[w * E + tid];
            cnt[w * E + tid] = own;
            own += v;
        }
        all = own;
        if (chunks > 1) {
            all = 0;
            for (int i = tid; i < MOE_NT; i += 1 << max(bits, 6)) {
                all += all_part[i];
                before += before_part[i];
            }
        }
    }
    const int upto = wave_scan(all);
    if (lane == 63) wave_tot[wave] = upto;
    __syncthreads();
    int base = upto - all, total = 0;
    for (int w = 0; w < MOE_NW; ++w) {
        base += w < wave ? wave_tot[w] : 0;
        total += wave_tot[w];
    }
    if (tid < E) {
        if (chunk == 0) row_off[tid] = base;
        for (int w = 0; w < MOE_NW; ++w) cnt[w * E + tid] += base + before;
    }
    if (chunk == 0 && tid == 0) row_off[E] = total;
    __syncthreads();
    for (int b = w0; b < w1; b += 64) {
        const int i = b + lane, id = i < w1 ? ids[i] : -1;
        const bool in = (uint32_t)id < (uint32_t)E;
        const uint64_t peers = peers_of(id, in, bits);
        const int rank = __popcll(peers & ((1ull << lane) - 1));
        const int row = in ? mine[id] + rank : -1;
        // (a wave's LDS operations complete in order; the fences bind the compiler)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        if (in && rank == 0) mine[id] += __popcll(peers);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        if (i < w1) slot[i] = row;
        if (in) src[row] = i;
        if (i < w1 && i >= total) src[i] = -1;
    }
    (void)n;
}

// `sorted`: one block, which then sorts. Else blocks count their chunks where the assignments are to be sorted.
template <int V, bool BIAS>
__device__ __forceinline__ void route_body(const brik_route_launch& a)
{
    __shared__ int count[BRIK_MOE_EXPERTS];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), k = a.r.k, E = a.r.experts;
    const int t0 = blockIdx.x * a.chunk, t1 = min(a.r.tokens, t0 + a.chunk);
    const bool counted = a.counts != nullptr;
    if (counted) {
        for (int i = threadIdx.x; i < E; i += blockDim.x) count[i] = 0;
        __syncthreads();
    }
    for (int t = t0 + wave; t < t1; t += MOE_NW) {
        float l[V], mine;
        int id;
        choose<V, BIAS>(a, t, l, id, mine);
        const float w = weight_of<V>(a, l, id, mine);
        if (lane < k) {
            a.r.ids[(size_t)t * k + lane] = id;
            a.r.weights[(size_t)t * k + lane] = id >= 0 ? a.r.scale * w : 0.f;
            if (counted && id >= 0) atomicAdd(&count[id], 1);
        }
    }
    if (counted) {
        __syncthreads();
        for (int i = threadIdx.x; i < E; i += blockDim.x) a.counts[blockIdx.x * E + i] = count[i];
    } else if (a.r.slot) {
        __threadfence_block();
        __syncthreads();
        sort_chunk(a.r.ids, 0, a.r.tokens * k, a.r.tokens * k, E, nullptr, 1, 0, a.r.row_off, a.r.src, a.r.slot);
    }
}

// dl of the formulas above; g_j = c dweights_j, G_e their sum over the places that chose e (a place has an expert of its own).
template <int V>
__device__ __forceinline__ void route_grad(const brik_route_launch& a, const float* dweights, float* dlogits, int t)
{
    const int lane = threadIdx.x & 63, E = a.r.experts, k = a.r.k, e0 = lane * V;
    const bool sig = a.r.flags & BRIK_ROUTE_SIGMOID, renorm = a.r.flags & BRIK_ROUTE_RENORM;
    const float* const row = a.r.logits + t * a.r.logit_stride;
    float l[V];
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = e0 + i < E ? logit_of(row[e0 + i]) : -__builtin_inff();
    int id = lane < k ? a.r.ids[(size_t)t * k + lane] : -1;
    if ((uint32_t)id >= (uint32_t)E) id = -1;
    const float mine = id >= 0 ? logit_of(row[id]) : -__builtin_inff();
    const float p = weight_of<V>(a, l, id, mine);
    float g = id >= 0 ? a.r.scale * dweights[(size_t)t * k + lane] : 0.f;
    // of this lane's expert: d, to be spread; `all`: taken off every expert's s (softmax over all of them)
    float d, all = 0.f;
    const float dot = !sig || renorm ? wave_fsum(id >= 0 ? p * g : 0.f) : 0.f;
    if (sig) {
        const float off = 1.f / (1.f + expf(mine));          // 1 - s
        d = renorm ? p * (g - dot) * off : p * off * g;
    } else {
        d = renorm ? p * (g - dot) : p * g;
        all = renorm ? 0.f : dot;
    }
    float out[V];
    if (!sig && !renorm) {
        float top = l[0], sum = 0.f;
#pragma unroll
        for (int i = 1; i < V; ++i) top = fmaxf(top, l[i]);
        top = wave_fmax(top);
#pragma unroll
        for (int i = 0; i < V; ++i) sum += out[i] = top == -__builtin_inff() ? 0.f : expf(l[i] - top);
        sum = wave_fsum(sum);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = sum == 0.f ? 0.f : -all * (out[i] / sum);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = 0.f;
    }
    for (int j = 0; j < k; ++j) {
        const int e = __builtin_amdgcn_readlane(id, j);
        const float v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, d), j));
        if (e < 0) continue;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e0 + i == e) out[i] += v;
    }
    float* const to = dlogits + (size_t)t * E;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (e0 + i < E) to[e0 + i] = out[i];
}

}  // namespace

#define BRIK_MOE_ROUTE(V)                                                                                                              \
    extern "C" __global__ __launch_bounds__(MOE_NT) void brik_route_##V(brik_route_launch a) { route_body<V, false>(a); }          \
    extern "C" __global__ __launch_bounds__(MOE_NT) void brik_route_bias_##V(brik_route_launch a) { route_body<V, true>(a); }      \
    extern "C" __global__ __launch_bounds__(256) void brik_route_grad_##V(brik_route_launch a, const float* dweights, float* dlogits) \
    {                                                                                                                                  \
        const int t = (int)blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);                                                            \
        if (t < a.r.tokens) route_grad<V>(a, dweights, dlogits, t);                                                                    \
    }
BRIK_MOE_ROUTE(1)
BRIK_MOE_ROUTE(2)
BRIK_MOE_ROUTE(4)
BRIK_MOE_ROUTE(8)
BRIK_MOE_ROUTE(16)

extern "C" __global__ __launch_bounds__(MOE_NT) void brik_route_count(brik_route_launch a)
{
    __shared__ int count[BRIK_MOE_EXPERTS];
    const int E = a.r.experts, per = a.chunk * a.r.k, n = a.r.tokens * a.r.k, a0 = blockIdx.x * per, a1 = min(n, a0 + per);
    for (int i = threadIdx.x; i < E; i += MOE_NT) count[i] = 0;
    __syncthreads();
    for (int i = a0 + (int)threadIdx.x; i < a1; i += MOE_NT) {
        const int id = a.r.ids[i];
        if ((uint32_t)id < (uint32_t)E) atomicAdd(&count[id], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < E; i += MOE_NT) a.counts[blockIdx.x * E + i] = count[i];
}

extern "C" __global__ __launch_bounds__(MOE_NT) void brik_route_sort(brik_route_launch a)
{
    const int per = a.chunk * a.r.k, n = a.r.tokens * a.r.k, a0 = blockIdx.x * per;
    sort_chunk(a.r.ids, a0, min(n, a0 + per), n, a.r.experts, a.counts, a.chunks, blockIdx.x, a.r.row_off, a.r.src, a.r.slot);
}
