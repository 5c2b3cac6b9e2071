// Routing: the k best experts of every token and their weights, the assignments sorted by expert, the gradient of the logits.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  ids = k largest;  w_j = c s_j,  or c s_j / sum of the chosen
//
// A team of 16 lanes holds a token's logits (64 lanes where there are more than 256 experts or k is over 16), V neighbours a lane, and
// takes the largest k times: the maximum of order-preserving keys over the lanes, then the lowest lane that has it (its experts are the
// lowest), then the lowest of its V. The owner notes it in LDS, so nothing is handed round. Keys are the logits' own bits without a
// bias (s grows with l), else s + bias: in f32 first, and where two of the keys in order lie within their error the token is taken
// again by a whole wave in 64 bits, high word first.
//
// Sorting is counting: every wave ranks 64 assignments at a time among those of the same expert by ballots over the bits of the
// expert's number, so the order is that of the assignments, whatever runs when. Chunks of tokens are counted as they are routed;
// a second launch adds up the counts of the chunks before its own and writes the rows. Few assignments are routed and sorted
// by one block.
//
// Bound by latency and vector instructions, not by bytes: 64 tokens of 64 experts, 8 each, 4.4 us, sorted 7.2; 16384 of them 4.9, sorted 11.8;
// 64 of 256 experts with a bias 11.7, 16384 of them 15.6 to 17 (73 % of the cycles issue vector instructions; the last waves are those of tokens taken
// again in 64 bits, one after the other, 3 to 4 us each), sorted 26 to 27. Assignments alone: 1024 sorted in 4.3 us by one block, 4096 in 7.8, 8192
// in 7.4 by two launches, 131072 in 8.6. The gradient of 4096 tokens of 64 experts 5 us. By whole waves with a bias, 16 experts a lane, 84 bytes a
// lane lie in scratch (1024 threads a block leave 128 registers).
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

// exp(x), off by (|x| + 2) 2^-24 of itself: a product's rounding and the exponential's. (The library's expf, written out for every value
// of a lane, is code that a block runs through once, waiting for it: 64 tokens of 256 experts 23 us with it.)
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * ATTN_LOG2E); }

// The V values of a lane from expert e0 on, -infinity behind the last. (All loads before the first use: with a bias read where it is
// added 64 tokens of 256 experts took 16 us.)
template <int V>
__device__ __forceinline__ void load_experts(const float* row, int E, int e0, bool by_four, float (&l)[V])
{
    if (V >= 4 && by_four) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            f32x4_t v = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
            const int e = e0 + 4 * q;
            if (e + 4 <= E) {
                v = *(const f32x4_t*)(row + e);
            } else {
                for (int i = 0; i < 3; ++i)
                    if (e + i < E) v[i] = row[e + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) l[(4 * q + i) % V] = v[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = e0 + i < E ? row[e0 + i] : -__builtin_inff();
}
template <int V>
__device__ __forceinline__ void load_logits(const brik_route_launch& a, int t, int e0, float (&l)[V])
{
    load_experts<V>(a.r.logits + t * a.r.logit_stride, a.r.experts, e0, ((a.r.logit_stride & 3) | ((uintptr_t)a.r.logits & 15)) == 0, l);
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = logit_of(l[i]);
}

__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }

// exp(min(l, 0) - m) / (1 + exp(-|l|)): the sigmoid of l times exp(-m), which stays in range where all of them are tiny.
__device__ __forceinline__ float sigmoid_part(float l, float m) { return exp_of(fminf(l, 0.f) - m) / (1.f + exp_of(-fabsf(l))); }

// Over the L lanes of a team (16: a row of lanes; 64).
template <int L>
__device__ __forceinline__ uint32_t team_max(uint32_t v) { return L == 16 ? max16u(v) : wave_max_u32(v); }
template <int L>
__device__ __forceinline__ float team_fmax(float v)
{
    v = BRIK_DPP_MAX(v, DPP_QUAD_1032);
    v = BRIK_DPP_MAX(v, DPP_QUAD_2301);
    v = BRIK_DPP_MAX(v, DPP_ROW_ROR4);
    v = BRIK_DPP_MAX(v, DPP_ROW_ROR8);
    return L == 16 ? v : quarters_max(v);
}
template <int L>
__device__ __forceinline__ float team_fsum(float v) { return L == 16 ? sum16(v) : quarters_sum(sum16(v)); }

// The largest of a token's logits, and of its softmax's terms the sum.
template <int L, int V>
__device__ __forceinline__ float top_of(const float (&l)[V])
{
    float top = l[0];
#pragma unroll
    for (int i = 1; i < V; ++i) top = fmaxf(top, l[i]);
    return team_fmax<L>(top);
}
template <int L, int V>
__device__ __forceinline__ float sum_of(const float (&l)[V], float top)
{
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) sum += exp_of(l[i] - top);
    return team_fsum<L>(sum);
}

// Notes of the chosen experts, by team of the block and place.
struct Chosen {
    int id;
    float l;
};

// The k best experts of token t into `out`, by a team of L lanes; -1 where none is left. Returns whether the order is in doubt: with a
// bias, where two keys that follow each other lie within the error of f32 ones. (Of a key half a step of itself and s's error, in 2^-24:
// of a sigmoid (|l| + 2) s (1 - s) < 0.8 by the exponential, 1 by the sum and 2 by the reciprocal; of a softmax at most 34 times its
// largest: (x + 2) exp(-x) < 2, sums of V and 6 steps, a quotient and a product.)
template <int L, int V, bool BIAS>
__device__ __forceinline__ bool choose(const brik_route_launch& a, const float (&l)[V], const float (&bias)[BIAS ? V : 1], Chosen* out)
{
    const int lane = threadIdx.x & 63, in = lane & (L - 1), e0 = in * V, k = a.r.k;
    uint32_t key[V];
    float off = 0.f;
    if constexpr (BIAS) {
        float s[V];
        const bool sig = a.r.flags & BRIK_ROUTE_SIGMOID;
        const float top = sig ? 0.f : top_of<L, V>(l), each = sig ? 1.f : 1.f / sum_of<L, V>(l, top);
        off = sig ? 0x1p-21f : 68 * 0x1p-24f * each;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s[i] = sig ? __builtin_amdgcn_rcpf(1.f + exp_of(-l[i])) : exp_of(l[i] - top) * each;
            key[i] = l[i] != -__builtin_inff() ? key_of(s[i] + bias[i] + 0.f) : 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = key_of(l[i]);
    }
    bool doubt = false;
    float before = 0.f;
    const int rounds = BIAS ? k + 1 : k;                      // (one more: what the last one is told from)
    for (int j = 0; j < rounds; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, key[i]);
        const uint32_t top = team_max<L>(best);
        if constexpr (BIAS) {
            const float now = __builtin_bit_cast(float, top >> 31 ? top ^ 0x80000000u : ~top);
            if (j > 0 && top != 0) doubt |= !(before - now > off + 0x1p-23f * fabsf(before));
            before = now;
            if (j == k) break;
        }
        uint64_t have = __ballot(best == top);
        if (L < 64) have &= ((1ull << (L & 63)) - 1) << (lane & ~(L - 1));
        const bool first = __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0)) == 0;
        if (best == top && first) {
            int at = 0;
            float v = l[0];
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (key[i] == top) {
                    at = i;
                    v = l[i];
                }
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = i == at ? 0u : key[i];
            out[j] = top ? Chosen{e0 + at, v} : Chosen{-1, -__builtin_inff()};
        }
    }
    return doubt;
}

// The same by a wave in 64 bits, with a bias.
template <int V>
__device__ __forceinline__ void choose64(const brik_route_launch& a, int t, Chosen* out)
{
    const int lane = threadIdx.x & 63, E = a.r.experts, e0 = lane * V;
    const bool sig = a.r.flags & BRIK_ROUTE_SIGMOID;
    float l[V];
    uint32_t hi[V], lo[V];
    double s[V], sum = 0;
    load_logits<V>(a, t, e0, l);
    float bias[V];
    load_experts<V>(a.r.bias, E, e0, ((uintptr_t)a.r.bias & 15) == 0, bias);
    const double top32 = sig ? 0.f : top_of<64, V>(l);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        s[i] = sig ? sigmoid64(l[i]) : exp(l[i] - top32);
        sum += s[i];
    }
    if (!sig) sum = wave_dsum(sum);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const uint64_t key = l[i] != -__builtin_inff() ? key_of((sig ? s[i] : s[i] / sum) + (double)bias[i]) : 0;
        hi[i] = (uint32_t)(key >> 32);
        lo[i] = (uint32_t)key;
    }
    for (int j = 0; j < a.r.k; ++j) {
        uint32_t best = hi[0], rest = 0;
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, hi[i]);
        const uint32_t top = wave_max_u32(best);
#pragma unroll
        for (int i = 0; i < V; ++i) rest = max(rest, hi[i] == top ? lo[i] : 0u);
        const uint32_t low = wave_max_u32(best == top ? rest : 0u);
        const uint64_t have = __ballot(best == top && rest == low);
        if (__ffsll((unsigned long long)have) - 1 == lane) {
            int at = 0;
            float v = l[0];
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (hi[i] == top && lo[i] == low) {
                    at = i;
                    v = l[i];
                }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                hi[i] = i == at ? 0u : hi[i];
                lo[i] = i == at ? 0u : lo[i];
            }
            out[j] = top ? Chosen{e0 + at, v} : Chosen{-1, -__builtin_inff()};
        }
    }
}

// The weight of lane j's expert of its team, before the scale; 0 where there is none.
template <int L, int V>
__device__ __forceinline__ float weight_of(const brik_route_launch& a, const float (&l)[V], int id, float mine)
{
    const bool sig = a.r.flags & BRIK_ROUTE_SIGMOID, renorm = a.r.flags & BRIK_ROUTE_RENORM, have = id >= 0;
    if (sig) {
        const float m = renorm ? team_fmax<L>(fminf(mine, 0.f)) : 0.f;
        const float p = have ? sigmoid_part(mine, m) : 0.f;
        const float sum = renorm ? team_fsum<L>(p) : 1.f;    // (by all lanes)
        return have ? p / sum : 0.f;
    }
    float top, sum;
    if (renorm) {
        top = team_fmax<L>(mine);
        sum = team_fsum<L>(have ? exp_of(mine - top) : 0.f);
    } else {
        top = top_of<L, V>(l);
        sum = sum_of<L, V>(l, top);
    }
    return have ? exp_of(mine - top) / sum : 0.f;
}

// Orders a wave's LDS writes before its own later reads (a wave's LDS operations complete in order: this binds the compiler).
__device__ __forceinline__ void wave_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
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

// The rows of the assignments [a0, a1), by a block of MOE_NT threads. With one chunk their counts are all there are;
// else `counts` holds those of every chunk.
__device__ __forceinline__ void sort_chunk(const int32_t* ids, int a0, int a1, int E, const int32_t* counts, int chunks, int chunk,
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
        wave_lds_order();
        if (in && rank == 0) mine[id] += __popcll(peers);
        wave_lds_order();
        if (i < w1) slot[i] = row;
        if (in) src[row] = i;
        if (i < w1 && i >= total) src[i] = -1;
    }
}

// Routes the chunk of the block. One chunk is then sorted here; of several, each block counts its own.
template <int L, int V, bool BIAS>
__device__ __forceinline__ void route_body(const brik_route_launch& a)
{
    constexpr int TEAMS = 64 / L, V64 = L == 64 ? V : (V + 3) / 4;
    __shared__ int count[BRIK_MOE_EXPERTS];
    __shared__ Chosen chosen[MOE_NW * TEAMS * (L == 64 ? BRIK_MOE_K : 16)];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), k = a.r.k, E = a.r.experts;
    const int team = lane / L, in = lane & (L - 1), e0 = in * V;
    const int t0 = blockIdx.x * a.chunk, t1 = min(a.r.tokens, t0 + a.chunk);
    const bool counted = a.counts != nullptr;
    if (counted) {
        for (int i = threadIdx.x; i < E; i += MOE_NT) count[i] = 0;
        __syncthreads();
    }
    float bias[BIAS ? V : 1];
    if constexpr (BIAS) load_experts<V>(a.r.bias, E, e0, ((uintptr_t)a.r.bias & 15) == 0, bias);
    Chosen* const notes = chosen + wave * TEAMS * k, *const mine = notes + team * k;
    for (int first = t0 + wave * TEAMS; first < t1; first += MOE_NW * TEAMS) {
        const int t = first + team;
        const bool real = t < t1;
        float l[V];
        load_logits<V>(a, min(t, t1 - 1), e0, l);
        wave_lds_order();
        const bool doubt = choose<L, V, BIAS>(a, l, bias, mine);
        wave_lds_order();
        if constexpr (BIAS) {
            uint64_t again = __ballot(doubt && real && in == 0);
            while (again) {
                const int from = __ffsll((unsigned long long)again) - 1, g = uniform(from / L);
                again &= again - 1;
                choose64<V64>(a, first + g, notes + g * k);
                wave_lds_order();
            }
        }
        const Chosen got = in < k ? mine[in] : Chosen{-1, -__builtin_inff()};
        const float w = weight_of<L, V>(a, l, got.id, got.l);
        if (real && in < k) {
            a.r.ids[(size_t)t * k + in] = got.id;
            a.r.weights[(size_t)t * k + in] = got.id >= 0 ? a.r.scale * w : 0.f;
            if (counted && got.id >= 0) atomicAdd(&count[got.id], 1);
        }
    }
    if (counted) {
        __syncthreads();
        for (int i = threadIdx.x; i < E; i += MOE_NT) a.counts[blockIdx.x * E + i] = count[i];
    } else if (a.r.slot) {
        __threadfence_block();
        __syncthreads();
        sort_chunk(a.r.ids, 0, a.r.tokens * k, E, nullptr, 1, 0, a.r.row_off, a.r.src, a.r.slot);
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
    load_logits<V>(a, t, e0, l);
    int id = lane < k ? a.r.ids[(size_t)t * k + lane] : -1;
    if ((uint32_t)id >= (uint32_t)E) id = -1;
    const float mine = id >= 0 ? logit_of(row[id]) : -__builtin_inff();
    const float p = weight_of<64, V>(a, l, id, mine);
    float g = id >= 0 ? a.r.scale * dweights[(size_t)t * k + lane] : 0.f;
    // of this lane's expert: d, to be spread; `all`: taken off every expert's s (softmax over all of them)
    float d, all = 0.f;
    const float dot = !sig || renorm ? team_fsum<64>(id >= 0 ? p * g : 0.f) : 0.f;
    if (sig) {
        const float off = 1.f / (1.f + exp_of(mine));          // 1 - s
        d = renorm ? p * (g - dot) * off : p * off * g;
    } else {
        d = renorm ? p * (g - dot) : p * g;
        all = renorm ? 0.f : dot;
    }
    float out[V];
    if (!sig && !renorm) {
        const float top = top_of<64, V>(l);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) sum += out[i] = top == -__builtin_inff() ? 0.f : exp_of(l[i] - top);
        sum = team_fsum<64>(sum);
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

#define BRIK_MOE_ROUTE(L, V)                                                                                                              \
    extern "C" __global__ __launch_bounds__(MOE_NT) void brik_route_##L##_##V(brik_route_launch a) { route_body<L, V, false>(a); }        \
    extern "C" __global__ __launch_bounds__(MOE_NT) void brik_route_bias_##L##_##V(brik_route_launch a) { route_body<L, V, true>(a); }
#define BRIK_MOE_ROUTE_GRAD(V)                                                                                                             \
    extern "C" __global__ __launch_bounds__(256) void brik_route_grad_##V(brik_route_launch a, const float* dweights, float* dlogits)     \
    {                                                                                                                                     \
        const int t = (int)blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);                                                               \
        if (t < a.r.tokens) route_grad<V>(a, dweights, dlogits, t);                                                                       \
    }
BRIK_MOE_ROUTE(16, 1)
BRIK_MOE_ROUTE(16, 2)
BRIK_MOE_ROUTE(16, 4)
BRIK_MOE_ROUTE(16, 8)
BRIK_MOE_ROUTE(16, 16)
BRIK_MOE_ROUTE(64, 1)
BRIK_MOE_ROUTE(64, 2)
BRIK_MOE_ROUTE(64, 4)
BRIK_MOE_ROUTE(64, 8)
BRIK_MOE_ROUTE(64, 16)
BRIK_MOE_ROUTE_GRAD(1)
BRIK_MOE_ROUTE_GRAD(2)
BRIK_MOE_ROUTE_GRAD(4)
BRIK_MOE_ROUTE_GRAD(8)
BRIK_MOE_ROUTE_GRAD(16)

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
    sort_chunk(a.r.ids, a0, min(n, a0 + per), a.r.experts, a.counts, a.chunks, blockIdx.x, a.r.row_off, a.r.src, a.r.slot);
}
