// Attention of up to 16 rows (query heads of a key / value head, times rows) over the quantized cache: decoding.
//
//   x_j = sum over groups g of s_jg (q . c_j)_g (+ m_jg sum(q)_g),   o = sum_j p_j v_j / sum_j p_j
//
// Four waves of a block take every fourth block of 32 keys; each is a pass over the keys of its own, with a running
// reference exponent M and sum, and they are joined at the end. The products run on the matrix cores in a form that
// keeps f32 accuracy: codes are small integers, exact in f16, and the other operand is split into two halves
// (22 bits). A group is 32 values, so one 16x16x32 product is one group of 16 keys and 16 rows:
//   scores: S^T = K Q^T, a product per group, its f32 result times the key's scale of the group (and, q4, the min times
//           the group's sum of q). A lane then holds 8 keys of one row: softmax needs no LDS.
//   output: O^T = V^T P'^T with P'_jg = p_j s_jg per group, split into halves in the registers where p lies. The order of
//           the keys within the product follows from that; V's transposed operand is read in it (ds_read_b64_tr_b8).
//   q4:     s n + m is taken as s (n - 8) + (m + 8 s), the second sum on the vector units.
// p s may be far from 1 (scales of any size), and a half holds 2^-24 to 65504. So M bounds x_j + e_j, e_j the exponent of the
// key's largest value scale, within 2^8; p is 2^7 times exp2(x - M) and P' stays below 2^15. Its second half ends at 2^-24, which
// is 2^-31 of the largest p_j 2^e_j: terms of groups whose scales lie far below the largest (of their key, or of one that
// weighs as much) are rounded to that, not to 2^-22 of themselves. A second pass by group where the sums are low keeps them
// too, but looking at the sums costs every call 1 to 5 %. Scores stay below 2^22, where M's last place is half a bit.
//
// Keys and values go through the wave's own LDS: whole 16-byte chunks of rows are loaded a block ahead into registers, and
// written rotated by row so that reading a column of chunks meets every bank once.
//
// Bound by the cache's bytes for one long q8 sequence (131072 tokens of 8 heads of 128: 285 MB in 58 us, 4.9 TB/s, then the join),
// by vector instructions for q4 (32 sequences of 1 to 8192: 177 MB in 66 us, two waves per SIMD), by latency for short ones
// (4095 tokens: 9 us, one block of 32 keys a wave). Two row tiles in a block, sharing the conversion of keys and values, need
// more registers than two waves per SIMD have (64 sequences behind a prefix of 8192: 80 us, 63 by 16 rows).
#include "attn_common.h"

namespace {

template <int FMT, int D>
struct FewTile {
    static constexpr int NG = D / 32;
    static constexpr int CH = (FMT == FMT_Q8 ? D : D / 2) / 16;          // 16-byte chunks of a row
    static constexpr int NI = (CH + 1) / 2;                              // loads of 64 chunks for 32 rows
    static constexpr int P2 = CH % 16 == 0 ? 4 : CH % 8 == 0 ? 3 : CH % 4 == 0 ? 2 : CH % 2 == 0 ? 1 : 0;
    static constexpr int SD = 16 * NG;                                   // dwords of the 32 keys' scales
    static constexpr int SI = (SD + 63) / 64;
    static constexpr int HP = FMT == FMT_Q4 ? 2 : 1;                     // planes of halves: scales, mins
    static constexpr int K = 0, V = 512 * CH, KS = 2 * V, VS = KS + 4 * SD, E = VS + 4 * SD, BAD = E + 128;
    static constexpr int KM = BAD + 128, VM = KM + (HP - 1) * 8 * SD, STAGE = VM + (HP - 1) * 8 * SD;     // mins: f32
    static constexpr int OS = D + 4;                                     // floats of a row of the joined output
    static constexpr int JOIN = 16 * OS * 4;
    static constexpr int BYTES = STAGE > JOIN ? STAGE : JOIN;
    // Where chunk c of a row lies: moved by a number of the row, so that rows whose chunks would share banks differ. By
    // exclusive or where the count of chunks is a power of two (one address and an instruction per chunk), else rotated.
    static constexpr bool XOR = CH == 1 << P2;
    static __device__ __forceinline__ int rot(int row) { return (row >> (4 - P2)) & ((1 << P2) - 1); }
    static __device__ __forceinline__ int chunk_at(int place, int row)        // which chunk lies at `place`
    {
        const int c = place - rot(row);
        return XOR ? place ^ rot(row) : c < 0 ? c + CH : c;
    }
    // byte of chunk `first + step` (step a compile-time number, its bits apart from first's) of the row; base: of (row, first)
    static __device__ __forceinline__ int base(int row, int first) { return XOR ? 16 * (row * CH + (first ^ rot(row))) : 16 * row * CH; }
    static __device__ __forceinline__ int at(int base, int row, int first, int step)
    {
        if constexpr (XOR) return base ^ (16 * step);
        const int c = first + step + rot(row);
        return base + 16 * (c >= CH ? c - CH : c);
    }
};

// A block of 32 keys in registers.
template <int FMT, int D>
struct FewLoad {
    using T = FewTile<FMT, D>;
    u32x4_t k[T::NI], v[T::NI];
    uint32_t ks[T::HP * T::SI], vs[T::HP * T::SI];
};

// Loads the 32 vectors from `v0` on, those of row r moved by `moved(r)` vectors: uniform base addresses and lane offsets that
// do not change from block to block.
template <int FMT, int D, class F>
__device__ __forceinline__ void few_fetch(FewLoad<FMT, D>& f, const brik_attn_launch& a, size_t v0, F moved)
{
    using T = FewTile<FMT, D>;
    const int lane = threadIdx.x & 63;
    const uint8_t* const kb = (const uint8_t*)a.c.k + v0 * (16 * T::CH);
    const uint8_t* const vb = (const uint8_t*)a.c.v + v0 * (16 * T::CH);
#pragma unroll
    for (int i = 0; i < T::NI; ++i) {
        const int c = 64 * i + lane, row = c / T::CH;
        if (T::CH % 2 && c >= 32 * T::CH) break;
        const int chunk = T::chunk_at(c - row * T::CH, row);
        const uint32_t off = 16u * (uint32_t)(row * T::CH + chunk);
        const size_t far = moved(row) * (16 * T::CH);
        f.k[i] = *(const u32x4_t*)(kb + far + off);
        f.v[i] = *(const u32x4_t*)(vb + far + off);
    }
    const size_t h0 = v0 * (2 * T::NG);                  // bytes
#pragma unroll
    for (int i = 0; i < T::SI; ++i) {
        const int d = 64 * i + lane;
        if (d < T::SD) {
            const uint32_t off = 4u * (uint32_t)d;
            const size_t far = moved(d < T::SD / 2 ? 0 : 16) * (2 * T::NG);
            f.ks[i] = *(const uint32_t*)((const uint8_t*)a.c.k_scales + h0 + far + off);
            f.vs[i] = *(const uint32_t*)((const uint8_t*)a.c.v_scales + h0 + far + off);
            if constexpr (FMT == FMT_Q4) {
                f.ks[T::SI + i] = *(const uint32_t*)((const uint8_t*)a.c.k_mins + h0 + far + off);
                f.vs[T::SI + i] = *(const uint32_t*)((const uint8_t*)a.c.v_mins + h0 + far + off);
            }
        }
    }
}

template <int FMT, int D>
__device__ __forceinline__ void few_load(FewLoad<FMT, D>& f, const brik_attn_launch& a, const Work& w, int t, const KeyPages& kp)
{
    const int slot = (32 * t) & ((1 << a.s.shift) - 1);
    // vectors of the first key and of the 17th (on page 0 where there is none: read and not used)
    const size_t v0 = (((size_t)max(kp.p[0], 0) * a.c.heads + w.head) << a.s.shift) + slot;
    if (a.s.shift > 4) {
        few_fetch<FMT, D>(f, a, v0, [](int) { return (size_t)0; });
    } else {
        const size_t v1 = ((size_t)max(kp.p[1], 0) * a.c.heads + w.head) << 4, jump = v1 - (v0 + 16);
        few_fetch<FMT, D>(f, a, v0, [=](int row) { return row < 16 ? (size_t)0 : jump; });
    }
}

// Orders a wave's LDS writes before its own later reads of what other lanes wrote (a wave's LDS operations complete in issue
// order, so this only binds the compiler).
__device__ __forceinline__ void wave_lds_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Bits 15 and 31: a half of w that is infinite or NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }

__device__ __forceinline__ f32x2_t centred_mins(uint32_t s, uint32_t m)
{
    f32x2_t r;
    r.x = fmaf(8.f, f16_bits_to_f32(s & 0xffffu), f16_bits_to_f32(m & 0xffffu));
    r.y = fmaf(8.f, f16_bits_to_f32(s >> 16), f16_bits_to_f32(m >> 16));
    return r;
}

// Into LDS. Returns whether some value scale or min is not finite: those are put in as 0, with a bit per key and group.
template <int FMT, int D>
__device__ __forceinline__ bool few_spread(const FewLoad<FMT, D>& f, unsigned char* lds)
{
    using T = FewTile<FMT, D>;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < T::NI; ++i) {
        if (T::CH % 2 && 64 * i + lane >= 32 * T::CH) break;
        *(u32x4_t*)(lds + T::K + 1024 * i + 16 * lane) = f.k[i];
        *(u32x4_t*)(lds + T::V + 1024 * i + 16 * lane) = f.v[i];
    }
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < T::SI; ++i) {
        const int d = 64 * i + lane;
        if (d < T::SD) {
            *(uint32_t*)(lds + T::KS + 4 * d) = f.ks[i];
            *(uint32_t*)(lds + T::VS + 4 * d) = f.vs[i];
            odd |= not_finite(f.vs[i]);
            if constexpr (FMT == FMT_Q4) {
                // a value is s n + m = s (n - 8) + (m + 8 s)
                *(f32x2_t*)(lds + T::KM + 8 * d) = centred_mins(f.ks[i], f.ks[T::SI + i]);
                *(f32x2_t*)(lds + T::VM + 8 * d) = centred_mins(f.vs[i], f.vs[T::SI + i]);
                odd |= not_finite(f.vs[T::SI + i]);
            }
        }
    }
    if (!__any(odd != 0)) return false;
    // rare: those groups become 0, noted by key
    if (lane < 32) *(uint32_t*)(lds + T::BAD + 4 * lane) = 0;
    wave_lds_fence();
#pragma unroll 1
    for (int e = lane; e < 2 * T::SD; e += 64) {
        uint16_t* const s = (uint16_t*)(lds + T::VS) + e;
        bool bad = (*s & 0x7c00u) == 0x7c00u;
        if constexpr (FMT == FMT_Q4) bad = bad || !(fabsf(((const float*)(lds + T::VM))[e]) <= 3.4028235e38f);
        if (bad) {
            *s = 0;
            if constexpr (FMT == FMT_Q4) ((float*)(lds + T::VM))[e] = 0.f;
            atomicOr((uint32_t*)(lds + T::BAD) + e / T::NG, 1u << (e % T::NG));
        }
    }
    return true;
}

typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;

// Half k of the halves that a lane read of 4 keys (NG each, in order).
template <int N>
__device__ __forceinline__ float half_of(const u32x2_t (&v)[N], int k)
{
    const uint32_t w = (k & 2) ? v[k >> 2].y : v[k >> 2].x;
    return f16_bits_to_f32((k & 1) ? w >> 16 : w & 0xffffu);
}

// One tile of 16 rows over its part of the keys.
template <int FMT, int D>
__device__ __forceinline__ void few_part(const brik_attn_launch& a, const Work& w, unsigned char* smem, float (&joinm)[4][16], float (&joinl)[4][16])
{
    using T = FewTile<FMT, D>;
    constexpr int NG = T::NG;
    constexpr bool Q4 = FMT == FMT_Q4;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
    unsigned char* const lds = smem + wave * T::BYTES;

    const Row row = find_row<16>(a, w, w.r0, m);
    int t0, t1;
    find_keys(w, wave_min(row.real ? row.lo : 0x7fffffff), wave_max(row.real ? row.hi : 0), 4, t0, t1);

    // first block's loads, then q while they are on the way
    FewLoad<FMT, D> next;
    PageWindow window(a, w);
    KeyPages kp = {{-1, -1}};
    int t = uniform(t0 + wave);
    if (t < t1) {
        kp = window.of(t);
        few_load(next, a, w, t, kp);
    }

    // q: this lane's values of its row, eight of each group, times a power of two that puts the row's largest below 2^15
    half8_t qh[NG], ql[NG];
    float qsum[NG], top = 0.f;
    {
        f32x4_t v[NG][2];
        const float* const src = a.a.q + (row.real ? row.t * a.a.q_stride + (size_t)row.h * D : 0) + 8 * q;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[g][i] = row.real ? *(const f32x4_t*)(src + 32 * g + 4 * i) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[g][i][e]));
            }
        top = quarters_max(top);
        const int up = top > 0.f && top < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float x[8], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_ldexpf(v[g][i >> 2][i & 3], up);
                sum += x[i];
            }
            // the order of the codes' conversion: words of four codes as 0, 2, 1, 3 (q8), eight nibbles as 0, 4, 1, 5, ... (q4)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int s = Q4 ? (i >> 1) + 4 * (i & 1) : (i & 4) + ((i & 1) << 1) + ((i >> 1) & 1);
                qh[g][i] = (_Float16)x[s];
                ql[g][i] = (_Float16)(x[s] - (float)qh[g][i]);
            }
            qsum[g] = Q4 ? quarters_sum(sum) : 0.f;
        }
        top = __builtin_amdgcn_ldexpf(a.a.scale, -up);
    }
    const bool cap = a.a.softcap > 0.f;
    const float xs = cap ? top / a.a.softcap : top * ATTN_LOG2E, ys = a.a.softcap * ATTN_LOG2E;

    // no mask inside [all_lo, all_hi)
    const int all_lo = wave_max(row.real ? row.lo : 0), all_hi = wave_min(row.hi);

    f32x4_t o[2 * NG];
    float om[NG], M = ATTN_NONE, l = 0.f;
    uint32_t bad = 0;                                    // groups of which this lane's row has seen a value that is not finite
#pragma unroll
    for (int n = 0; n < 2 * NG; ++n) o[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) om[g] = 0.f;

    // row of V that this lane's address names in a transposed read: keys 4 q .. 4 q + 3 of both 16-key halves
    const int vrow = ((lane & 15) >> 3) * 16 + 4 * q + (((lane & 15) >> 1) & 3), vbase = T::base(vrow, 0);
    const int kfirst = Q4 ? 0 : q >> 1, kbase = T::base(m, kfirst);

    // One block of keys, in LDS. general: some of its keys are not seen by some row, or some values are not finite (odd).
    auto block = [&](bool general, bool odd, int t, const bool (&have)[2]) {
        // e_j of the 32 keys
        {
            const uint16_t* const s = (const uint16_t*)(lds + T::VS) + (lane & 31) * NG;
            uint32_t top16 = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) top16 = max(top16, (uint32_t)s[g] & 0x7fffu);
            *(float*)(lds + T::E + 4 * (lane & 31)) = (float)((int)(top16 >> 10) - 14);
        }
        // scores: y[4 i + r] of key 16 i + 4 q + r
        float y[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x2_t s[NG];
            f32x4_t mn[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                s[g] = *(const u32x2_t*)(lds + T::KS + (16 * i + 4 * q) * 2 * NG + 8 * g);
                if constexpr (Q4) mn[g] = *(const f32x4_t*)(lds + T::KM + (16 * i + 4 * q) * 4 * NG + 16 * g);
            }
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                half8_t k;
                // (rows 16 apart are moved alike)
                const unsigned char* const src = lds + T::K + 256 * T::CH * i + T::at(kbase, m, kfirst, Q4 ? g : 2 * g);
                if constexpr (Q4) {
                    const uint32_t c = *(const uint32_t*)(src + 4 * q);
                    k = centred_q4(c, c >> 4, c >> 8, c >> 12);
                } else {
                    const u32x2_t c = *(const u32x2_t*)(src + 8 * (q & 1));
                    k = halves_q8(c.x, c.y);
                }
                floatx4_t acc = {0.f, 0.f, 0.f, 0.f};
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[g], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[g], acc, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = fmaf(half_of(s, r * NG + g), acc[r], x[r]);
                    if constexpr (Q4) x[r] = fmaf(mn[(r * NG + g) >> 2][(r * NG + g) & 3], qsum[g], x[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) y[4 * i + r] = x[r];
        }
        float mul = xs;                                  // scores are y * mul
        if (cap) {
            mul = 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = ys * attn_tanh(y[i] * xs);
        }
        if (general) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = 16 * (i >> 2) + 4 * q + (i & 3);
                const bool in = 32 * t + k >= row.lo && 32 * t + k < row.hi && have[i >> 2];
                y[i] = in ? y[i] * mul : -__builtin_inff();
                if (odd) bad |= in ? *(const uint32_t*)(lds + T::BAD + 4 * k) : 0u;
            }
            mul = 1.f;
        }
        wave_lds_fence();
        const f32x4_t e0 = *(const f32x4_t*)(lds + T::E + 16 * q), e1 = *(const f32x4_t*)(lds + T::E + 64 + 16 * q);
        float tm = ATTN_NONE;
#pragma unroll
        for (int i = 0; i < 4; ++i) tm = fmaxf(tm, fmaxf(fmaf(y[i], mul, e0[i]), fmaf(y[4 + i], mul, e1[i])));
        if (__any(tm > M + 8.f)) {
            const float Mn = fmaxf(M, quarters_max(tm)), f = __builtin_amdgcn_exp2f(M - Mn);
            M = Mn;
            l *= f;
#pragma unroll
            for (int n = 0; n < 2 * NG; ++n) o[n] *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) om[g] *= f;
        }
        float p[8];
        const float shift = 7.f - M;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(y[i], mul, shift));
            l += p[i];
        }
        u32x2_t s0[NG], s1[NG];
        f32x4_t m0[NG], m1[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            s0[g] = *(const u32x2_t*)(lds + T::VS + 4 * q * 2 * NG + 8 * g);
            s1[g] = *(const u32x2_t*)(lds + T::VS + (16 + 4 * q) * 2 * NG + 8 * g);
            if constexpr (Q4) {
                m0[g] = *(const f32x4_t*)(lds + T::VM + 4 * q * 4 * NG + 16 * g);
                m1[g] = *(const f32x4_t*)(lds + T::VM + (16 + 4 * q) * 4 * NG + 16 * g);
            }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            u32x4_t phw, plw;
            float ps[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ps[i] = fmaf(i < 4 ? half_of(s0, i * NG + g) : half_of(s1, (i - 4) * NG + g), p[i], 0.f);
                if constexpr (Q4)
                    om[g] = fmaf(p[i], i < 4 ? m0[(i * NG + g) >> 2][(i * NG + g) & 3] : m1[((i - 4) * NG + g) >> 2][((i - 4) * NG + g) & 3], om[g]);
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                // the order of V's conversion: keys 0, 2, 1, 3 of each half. (The product rounded to a half in one
                // instruction, and again for the rest of it, takes twice the time of these four.)
                const float u = ps[(i & 4) + ((i & 2) >> 1)], v = ps[(i & 4) + ((i & 2) >> 1) + 2];
                const half2_t h = halves(u, v);
                phw[i / 2] = __builtin_bit_cast(uint32_t, h);
                plw[i / 2] = __builtin_bit_cast(uint32_t, halves(residual<0>(h, u), residual<1>(h, v)));
            }
            const half8_t ph = __builtin_bit_cast(half8_t, phw), pl = __builtin_bit_cast(half8_t, plw);
            if constexpr (Q4) {
                const i32x2_t c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t*)(lds + T::V + T::at(vbase, vrow, 0, g) + 8 * (lane & 1)));
                const uint32_t c0 = (uint32_t)c.x, c1 = (uint32_t)c.y;
                const half8_t lo = centred_q4(c0, c0 >> 8, c1, c1 >> 8), hi = centred_q4(c0 >> 4, c0 >> 12, c1 >> 4, c1 >> 12);
                o[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, ph, o[2 * g], 0, 0, 0);
                o[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ph, o[2 * g + 1], 0, 0, 0);
                o[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pl, o[2 * g], 0, 0, 0);
                o[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pl, o[2 * g + 1], 0, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const i32x2_t c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t*)(lds + T::V + T::at(vbase, vrow, 0, 2 * g + j) + 8 * (lane & 1)));
                    const half8_t v = halves_q8((uint32_t)c.x, (uint32_t)c.y);
                    o[2 * g + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[2 * g + j], 0, 0, 0);
                    o[2 * g + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[2 * g + j], 0, 0, 0);
                }
            }
        }
    };

    for (; t < t1; t += 4) {
        const bool have[2] = {kp.p[0] >= 0, kp.p[1] >= 0};
        wave_lds_fence();
        const bool odd = few_spread(next, lds);
        if (t + 4 < t1) {
            kp = window.of(t + 4);
            few_load(next, a, w, t + 4, kp);
        }
        wave_lds_fence();
        const bool plain = 32 * t >= all_lo && 32 * t + 32 <= all_hi && have[0] && have[1] && !odd;
        block(!plain, odd, t, have);
    }

    // the four waves' results joined in LDS
    l = quarters_sum(l);
    bad |= (uint32_t)__shfl_xor((int)bad, 16);
    bad |= (uint32_t)__shfl_xor((int)bad, 32);
    if (q == 0) {
        joinm[wave][m] = M;
        joinl[wave][m] = row.real ? l : -1.f;
    }
    __syncthreads();
    float Mb = fmaxf(fmaxf(joinm[0][m], joinm[1][m]), fmaxf(joinm[2][m], joinm[3][m]));
    const float f = __builtin_amdgcn_exp2f(M - Mb);
    float* const mine = (float*)lds + m * T::OS;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        if ((bad >> g) & 1) o[2 * g] = o[2 * g + 1] = f32x4_t{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
        if constexpr (Q4) {
            const float add = quarters_sum(om[g]);
            // tile 2 g + j, row 4 q + r holds value 32 g + 2 (4 q + r) + j
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x4_t v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = (o[2 * g + (i & 1)][2 * h + (i >> 1)] + add) * f;
                *(f32x4_t*)(mine + 32 * g + 8 * q + 4 * h) = v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) *(f32x4_t*)(mine + 32 * g + 16 * j + 4 * q) = o[2 * g + j] * f;
        }
    }
    __syncthreads();
    const int G = a.a.heads / a.c.heads;
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
        const int r = i / (D / 4), d = 4 * (i - r * (D / 4));
        const int rel = (w.r0 + r) / G;
        if (rel >= w.count) continue;
        if (joinl[0][r] < 0.f) continue;                     // a row of no sequence
        const int tok = w.first + rel, h = w.head * G + w.r0 + r - rel * G;
        float Mr = joinm[0][r], L = 0.f;
#pragma unroll
        for (int k = 1; k < 4; ++k) Mr = fmaxf(Mr, joinm[k][r]);
#pragma unroll
        for (int k = 0; k < 4; ++k) L += joinl[k][r] * __builtin_amdgcn_exp2f(joinm[k][r] - Mr);
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) v += *(const f32x4_t*)((const float*)(smem + k * T::BYTES) + r * T::OS + d);
        if (w.whole) {
            *(f32x4_t*)(a.a.out + tok * a.a.out_stride + (size_t)h * D + d) = L == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : v / L;
        } else {
            const size_t at = part_at(a, w, r, tok, h);
            if (L != 0.f) *(f32x4_t*)(a.part + at * D + d) = v;
            if (d == 0) *(f32x2_t*)(a.ml + 2 * at) = f32x2_t{Mr, L};
        }
    }
}

template <int FMT, int D>
__device__ __forceinline__ void few_body(const brik_attn_launch& a)
{
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * FewTile<FMT, D>::BYTES];
    __shared__ float joinm[4][16], joinl[4][16];
    // One tile's keys, or parts of one sequence after the other.
    Work w;
    w.head = (a.first_block + (int)blockIdx.x) % a.c.heads;
    const int own = (a.first_block + (int)blockIdx.x) / a.c.heads - a.prefix_tiles * a.prefix_splits;
    const bool parts = a.own_blocks && own >= 0;
    int each = 0, g = 0, end = 0;
    if (parts) {
        const Share share(a);
        each = uniform(share.each);
        g = own * each;
        end = min(g + each, uniform(share.total));
        if (g >= end) return;
        w.prefix = false;
    } else if (!find_work<16>(a, w)) {
        return;
    }
    for (;;) {
        if (parts) next_part(a, each, own, end, g, w);
        few_part<FMT, D>(a, w, smem, joinm, joinl);
        if (!parts || g >= end) return;
        __syncthreads();
    }
}

}  // namespace

#define BRIK_ATTN_FEW(D)                                                                                                             \
    extern "C" __global__ __launch_bounds__(256, D <= 64 ? 3 : D <= 128 ? 2 : 1) void brik_attn_few_q8_##D(brik_attn_launch a) { few_body<FMT_Q8, D>(a); }             \
    extern "C" __global__ __launch_bounds__(256, D <= 64 ? 3 : D <= 128 ? 2 : 1) void brik_attn_few_q4_##D(brik_attn_launch a) { few_body<FMT_Q4, D>(a); }
BRIK_ATTN_FEW(64)
BRIK_ATTN_FEW(96)
BRIK_ATTN_FEW(128)
BRIK_ATTN_FEW(192)
BRIK_ATTN_FEW(256)
