// Attention of many rows over the quantized cache: prefill, and the rows of all sequences over a shared prefix.
//
// 128 or 256 rows a block, 32 a wave (a row: a query head of the key / value head, of a token); 32 keys a step, in LDS for all of
// its waves, two buffers. As in attn_few.hip the products keep f32 accuracy on the f16 matrix cores, here with
// 32x32x16 products and the conversion done once per block:
//   scores: S^T = K Q^T; codes exact in f16 (q4: less 8), q as two halves; per group one f32 result, times the key's scale.
//           q4: the mins' part, sum over groups of (m + 8 s)_jg sum(q)_g, is a product of its own: both as two halves.
//   output: O^T = V^T P^T with V dequantized to two halves, times 2^-e_j (e_j: exponent of the key's largest scale, so
//           that its halves are well inside their range, exact to 2^-25, which groups far below the key's largest feel),
//           P''_j = p_j 2^e_j as two halves, and the three products that are above 2^-22. With the scales in V instead of in
//           P the split of P is done once instead of per group.
// A lane holds 16 keys of one row of S^T, which is the layout that the second product wants of P; V's columns come
// from its rows in LDS by transposed reads (ds_read_b64_tr_b16).
//
// Blocks of keys that all rows of a wave see, whose e_j lie within 2^10 and whose scales are finite, take the short
// path (one bound for the block instead of one per key); others mask, bound each key by itself, and give NaN to the
// rows that see a token with an infinite or NaN scale (its values are 0 in LDS, so that other rows are not touched).
//
// Bound by the five products of halves that two f32 products take, and the conversion and softmax between them (4096 rows of
// 32 heads over 8 of 128, q8: 377 to 393 us, 0.36 PFLOP/s of the formula, 0.9 of products; without the output's products 122
// less, the scores' 83, the conversion 31). 256 rows a block against 128: 423 and 451 us at that stage. Waves 4 to 7
// converting after the products instead of before, to run beside the others' products: 408 against 389.
#include "attn_common.h"

namespace {

// NW: waves of a block, 32 rows each.
template <int FMT, int D, int NW>
struct TileCfg {
    static constexpr bool Q4 = FMT == FMT_Q4;
    static constexpr int NG = D / 32, U = D / 8;                       // groups, 8-value chunks of a row
    static constexpr int MM = Q4 ? (NG + 3) / 4 : 0;                   // products of the mins' part
    // In LDS, K as fragments: chunk u of key k (16 bytes as halves) at u KB + 16 k, so that a chunk's keys are read, and a
    // key's chunks are written, without meeting a bank twice; V's rows RB bytes apart, so that four rows read together
    // (64 bytes each) meet all banks.
    static constexpr int KB = 32 * 16 + 16, RB = 2 * D + (2 * D % 128 ? 0 : 64);
    static constexpr int KC = 0, VH = U * KB, VL = VH + 32 * RB, KS = VL + 32 * RB, G = KS + 64 * NG, BAD = G + 128, KM = BAD + 128;
    static constexpr int BUF = KM + 1024 * MM;
    // chunks that a thread brings in: 4 D of keys, then 4 D of values, NT at a time (kinds the same for a wave)
    static constexpr int NT = 64 * NW, ITEMS = (8 * D + NT - 1) / NT;
    static constexpr int V0 = 4 * D / NT, VITEMS = ITEMS - V0;         // from item V0 on they may be values
    static constexpr bool EVEN = 4 * D % NT == 0;
    static __device__ __forceinline__ bool value(int i) { return EVEN ? i >= V0 : (int)threadIdx.x + NT * i >= 4 * D; }
    static __device__ __forceinline__ bool live(int i) { return (i + 1) * NT <= 8 * D || (int)threadIdx.x + NT * i < 8 * D; }
    // A key's chunks lie in 8, 16 or 32 consecutive lanes: a thread loads its own group's scale and the key's maximum is a
    // cross-lane one. Otherwise every thread loads all scales of its key.
    static constexpr bool ROWS = U == 8 || U == 16 || U == 32;
    static constexpr int SW = (NG + 1) / 2, VS = ROWS ? 1 : SW;        // dwords of a key's scales (NG odd: padded)
};

// A block of 32 keys on its way: raw codes and scales in registers.
template <int FMT, int D, int NW>
struct TileLoad {
    using T = TileCfg<FMT, D, NW>;
    uint32_t code[T::ITEMS][FMT == FMT_Q8 ? 2 : 1];
    uint32_t vs[T::VITEMS][T::VS], vm[T::VITEMS][FMT == FMT_Q4 ? T::VS : 1];   // of the items that are values
    uint32_t ks[T::SW], km[FMT == FMT_Q4 ? T::SW : 1];                           // threads 0..31: of key threadIdx.x
};

// NG halves from p (2-byte aligned where NG is odd).
template <int NG>
__device__ __forceinline__ void load_halves(uint32_t (&v)[(NG + 1) / 2], const uint16_t* p)
{
    if constexpr (NG % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NG / 2; ++i) v[i] = ((const uint32_t*)p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < NG / 2; ++i) v[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        v[NG / 2] = p[NG - 1];
    }
}

template <int N>
__device__ __forceinline__ uint32_t half_bits(const uint32_t (&v)[N], int g)
{
    return g & 1 ? v[g >> 1] >> 16 : v[g >> 1] & 0xffffu;
}

template <int FMT, int D, int NW>
__device__ __forceinline__ void tile_load(TileLoad<FMT, D, NW>& f, const brik_attn_launch& a, const Work& w, int t, const KeyPages& kp)
{
    using T = TileCfg<FMT, D, NW>;
    constexpr int RC = FMT == FMT_Q8 ? D : D / 2;                      // bytes of a row of codes
    const int tid = threadIdx.x, slot = (32 * t) & ((1 << a.s.shift) - 1);
    const size_t v0 = (((size_t)max(kp.p[0], 0) * a.c.heads + w.head) << a.s.shift) + slot;
    // vectors from v0 to the 17th key's, less the 16 between them where they follow on
    const size_t jump = a.s.shift > 4 ? 0 : (((size_t)max(kp.p[1], 0) * a.c.heads + w.head) << 4) - (v0 + 16);
    const uint8_t* const kb = (const uint8_t*)a.c.k + v0 * RC;
    const uint8_t* const vb = (const uint8_t*)a.c.v + v0 * RC;
#pragma unroll
    for (int i = 0; i < T::ITEMS; ++i) {
        if (!T::live(i)) break;
        const int it = tid + T::NT * i;
        const bool value = T::value(i);
        const int j = value ? it - 4 * D : it, key = j / T::U, u = j - key * T::U;
        const size_t far = key < 16 ? 0 : jump;
        const uint8_t* const p = (value ? vb : kb) + far * RC + (uint32_t)(key * RC + u * (RC / T::U));
        if constexpr (FMT == FMT_Q8) {
            const u32x2_t c = *(const u32x2_t*)p;
            f.code[i][0] = c.x;
            f.code[i][1] = c.y;
        } else {
            f.code[i][0] = *(const uint32_t*)p;
        }
        if (value) {
            const int n = i < T::V0 ? 0 : i - T::V0;
            const size_t at = (v0 + far + key) * T::NG;
            if constexpr (T::ROWS) {
                f.vs[n][0] = a.c.v_scales[at + (u >> 2)];
                if constexpr (FMT == FMT_Q4) f.vm[n][0] = a.c.v_mins[at + (u >> 2)];
            } else {
                load_halves<T::NG>(f.vs[n], a.c.v_scales + at);
                if constexpr (FMT == FMT_Q4) load_halves<T::NG>(f.vm[n], a.c.v_mins + at);
            }
        }
    }
    if (tid < 32) {
        const size_t v = v0 + (tid < 16 ? 0 : jump) + tid;
        load_halves<T::NG>(f.ks, a.c.k_scales + v * T::NG);
        if constexpr (FMT == FMT_Q4) load_halves<T::NG>(f.km, a.c.k_mins + v * T::NG);
    }
}

// Maximum / union over the groups of a key whose U chunks lie in U consecutive lanes, four chunks a group.
template <int U, class F>
__device__ __forceinline__ uint32_t key_fold(uint32_t v, F f)
{
    if constexpr (U == 8) return f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, DPP_ROW_HALF_MIRROR, 0xF, 0xF, false));
    v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, DPP_ROW_ROR4, 0xF, 0xF, false));
    v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, DPP_ROW_ROR8, 0xF, 0xF, false));
    if constexpr (U == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        const uint32_t a = r[0], b = r[1];
        v = f(a, b);
    }
    return v;
}
template <int U>
__device__ __forceinline__ uint32_t key_max(uint32_t v) { return key_fold<U>(v, [](uint32_t a, uint32_t b) { return max(a, b); }); }
template <int U>
__device__ __forceinline__ uint32_t key_or(uint32_t v) { return key_fold<U>(v, [](uint32_t a, uint32_t b) { return a | b; }); }

template <int FMT, int D, int NW>
__device__ __forceinline__ void tile_spread(const TileLoad<FMT, D, NW>& f, unsigned char* buf)
{
    using T = TileCfg<FMT, D, NW>;
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < T::ITEMS; ++i) {
        if (!T::live(i)) break;
        const int it = tid + T::NT * i;
        const bool value = T::value(i);
        const int j = value ? it - 4 * D : it, key = j / T::U, u = j - key * T::U;
        if (!value) {
            half8_t k;
            if constexpr (T::Q4) k = centred_q4(f.code[i][0], f.code[i][0] >> 4, f.code[i][0] >> 8, f.code[i][0] >> 12);
            else k = halves_q8(f.code[i][0], f.code[i][1]);
            *(half8_t*)(buf + T::KC + u * T::KB + 16 * key) = k;
            continue;
        }
        const auto& vs = f.vs[i < T::V0 ? 0 : i - T::V0];
        const auto& vm = f.vm[i < T::V0 ? 0 : i - T::V0];
        // the key's exponent, and which of its groups are not finite
        const int g = u >> 2;
        uint32_t top = 0, bad = 0, sb = 0, mb = 0;
        auto take = [&](uint32_t sbits, uint32_t mbits, int group) {
            const uint32_t s = sbits & 0x7fffu, m = mbits & 0x7fffu;
            const bool odd = s >= 0x7c00u || m >= 0x7c00u;
            bad |= (uint32_t)odd << group;
            const uint32_t n = T::Q4 ? max(s, m < (4u << 10) ? 0u : m - (4u << 10)) : s;          // |s n + m| < 2^8 both ways
            top = max(top, odd ? 0u : n);
        };
        if constexpr (T::ROWS) {
            sb = vs[0];
            mb = T::Q4 ? vm[0] : 0;
            take(sb, mb, g);
            top = key_max<T::U>(top);
            bad = key_or<T::U>(bad);
        } else {
#pragma unroll
            for (int k = 0; k < T::NG; ++k) {
                const uint32_t s = half_bits(vs, k), m = T::Q4 ? half_bits(vm, k) : 0;
                take(s, m, k);
                sb = g == k ? s : sb;
                mb = g == k ? m : mb;
            }
        }
        const int e = (int)(top >> 10) - 14;
        const bool ok = !((bad >> g) & 1);
        const float s = ok ? __builtin_amdgcn_ldexpf(f16_bits_to_f32(sb), -e) : 0.f;
        float v[8];
        if constexpr (T::Q4) {
            const float m = ok ? __builtin_amdgcn_ldexpf(f16_bits_to_f32(mb), -e) : 0.f;
            const uint32_t lo = f.code[i][0] & 0x0f0f0f0fu, hi = (f.code[i][0] >> 4) & 0x0f0f0f0fu;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = fmaf((float)((lo >> (8 * k)) & 0xffu), s, m);
                v[2 * k + 1] = fmaf((float)((hi >> (8 * k)) & 0xffu), s, m);
            }
        } else {
            const uint32_t c[2] = {f.code[i][0] ^ 0x80808080u, f.code[i][1] ^ 0x80808080u};
            const float m = -128.f * s;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = fmaf((float)((c[k >> 2] >> (8 * (k & 3))) & 0xffu), s, m);
        }
        u32x4_t vh, vl;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const half2_t h = halves(v[2 * k], v[2 * k + 1]);
            vh[k] = __builtin_bit_cast(uint32_t, h);
            vl[k] = __builtin_bit_cast(uint32_t, halves(residual<0>(h, v[2 * k]), residual<1>(h, v[2 * k + 1])));
        }
        const int at = key * T::RB + 16 * u;
        *(u32x4_t*)(buf + T::VH + at) = vh;
        *(u32x4_t*)(buf + T::VL + at) = vl;
        if (u == 0) {
            *(float*)(buf + T::G + 4 * key) = __builtin_amdgcn_ldexpf(1.f, e);
            *(uint32_t*)(buf + T::BAD + 4 * key) = bad;
        }
    }
    if (tid < 32) {
#pragma unroll
        for (int g = 0; g < T::NG; ++g) *(uint16_t*)(buf + T::KS + 64 * g + 2 * tid) = (uint16_t)half_bits(f.ks, g);
        if constexpr (T::Q4) {
            // sixteenths of m + 8 s as two halves, the second times 2^11: [high 4 | low 4] and [high 4 | 0] of four groups
#pragma unroll
            for (int k = 0; k < T::MM; ++k) {
                half8_t x, y;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int g = 4 * k + i;
                    float m = 0.f;
                    if (g < T::NG) m = fmaf(8.f, f16_bits_to_f32(half_bits(f.ks, g)), f16_bits_to_f32(half_bits(f.km, g))) * 0.0625f;
                    x[i] = y[i] = (_Float16)m;
                    x[4 + i] = (_Float16)((m - (float)x[i]) * 2048.f);
                    y[4 + i] = (_Float16)0.f;
                }
                *(half8_t*)(buf + T::KM + 1024 * k + 16 * tid) = x;
                *(half8_t*)(buf + T::KM + 1024 * k + 512 + 16 * tid) = y;
            }
        }
    }
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

// Eight keys of a value column: two transposed reads, 8 rows apart.
template <int RB>
__device__ __forceinline__ half8_t v_frag(const unsigned char* p)
{
    const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)p);
    const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p + 8 * RB));
    return __builtin_bit_cast(half8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <int FMT, int D, int NW>
__device__ __forceinline__ void tile_body(const brik_attn_launch& a)
{
    using T = TileCfg<FMT, D, NW>;
    constexpr int NG = T::NG;
    constexpr bool Q4 = T::Q4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * T::BUF];
    __shared__ int range[2 * NW];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 31, h = lane >> 5;

    Work w;
    if (!find_work<32 * NW>(a, w)) return;
    const Row row = find_row<32>(a, w, w.r0 + 32 * wave, m);
    // keys that any row of the wave sees, [any_lo, any_hi), and that all see
    const int any_lo = wave_min(row.real ? row.lo : 0x7fffffff), any_hi = wave_max(row.real ? row.hi : 0);
    const int all_lo = wave_max(row.real ? row.lo : 0), all_hi = wave_min(row.hi);
    if (lane == 0) {
        range[wave] = any_lo;
        range[NW + wave] = any_hi;
    }
    __syncthreads();
    int t0, t1;
    int lo = range[0], hi = range[NW];
#pragma unroll
    for (int i = 1; i < NW; ++i) {
        lo = min(lo, range[i]);
        hi = max(hi, range[NW + i]);
    }
    find_keys(w, uniform(lo), uniform(hi), 4, t0, t1);

    TileLoad<FMT, D, NW> next;
    PageWindow window(a, w);
    KeyPages kp = {{-1, -1}}, kn = {{-1, -1}};       // of this block of keys and the next
    if (t0 < t1) {
        kp = window.of(t0);
        tile_load(next, a, w, t0, kp);
    }

    // q: eight values of each half group, times a power of two that puts the row's largest below 2^6; a negative scale
    // goes to q
    half8_t qh[2 * NG], ql[2 * NG], qs[Q4 ? T::MM : 1];
    float xs, top = 0.f;
    {
        f32x4_t v[2 * NG][2];
        const float* const src = a.a.q + (row.real ? row.t * a.a.q_stride + (size_t)row.h * D : 0) + 8 * h;
#pragma unroll
        for (int c = 0; c < 2 * NG; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[c][i] = row.real ? *(const f32x4_t*)(src + 16 * c + 4 * i) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[c][i][e]));
            }
        float o, n;
        half_pair(top, o, n);
        top = fmaxf(o, n);
        const int up = top > 0.f && top < __builtin_inff() ? 6 - __builtin_amdgcn_frexp_expf(top) : 0;
        const float sign = a.a.scale < 0.f ? -1.f : 1.f;
        float sum[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) sum[g] = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * NG; ++c) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_ldexpf(v[c][i >> 2][i & 3] * sign, up);
                sum[c >> 1] += x[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int s = Q4 ? (i >> 1) + 4 * (i & 1) : (i & 4) + ((i & 1) << 1) + ((i >> 1) & 1);
                qh[c][i] = (_Float16)x[s];
                ql[c][i] = (_Float16)(x[s] - (float)qh[c][i]);
            }
        }
        if constexpr (Q4) {
#pragma unroll
            for (int k = 0; k < T::MM; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float s = 0.f;
                    if (4 * k + i < NG) {
                        half_pair(sum[4 * k + i], o, n);
                        s = (o + n) * 16.f;
                    }
                    const _Float16 hi = (_Float16)s, lo = (_Float16)(s - (float)hi);
                    qs[k][i] = h ? lo : hi;
                    qs[k][4 + i] = h ? (_Float16)0.f : (_Float16)((float)hi * 0x1p-11f);
                }
        }
        xs = __builtin_amdgcn_ldexpf(fabsf(a.a.scale), -up);
    }
    const bool cap = a.a.softcap > 0.f;
    xs = cap ? xs / a.a.softcap : xs * ATTN_LOG2E;
    const float ys = a.a.softcap * ATTN_LOG2E;

    floatx16_t o[NG];
    float M = ATTN_NONE, l = 0.f;
    uint32_t bad = 0;                           // groups of which this lane's row has seen a scale that is not finite
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[g][r] = 0.f;

    // this lane's address in a fragment of K, and in a transposed read of V (four rows of 16 values by 16 lanes)
    const int kat = T::KC + h * T::KB + 16 * m, vat = T::VH + (4 * h + ((lane & 15) >> 2)) * T::RB + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

    // x[r]: scores (without xs) of key 8 (r / 4) + 4 h + r % 4
    auto block = [&](bool general, const unsigned char* buf, int t, const bool (&have)[2], float gmax) {
        floatx16_t x;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 0.f;
        if constexpr (Q4) {
#pragma unroll
            for (int k = 0; k < T::MM; ++k)
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8_t*)(buf + T::KM + 1024 * k + 16 * lane), qs[k], x, 0, 0, 0);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            floatx16_t acc;
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
            for (int c = 2 * g; c < 2 * g + 2; ++c) {
                const half8_t k = *(const half8_t*)(buf + kat + 2 * c * T::KB);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[c], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[c], acc, 0, 0, 0);
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const u32x2_t s = *(const u32x2_t*)(buf + T::KS + 64 * g + 16 * b + 8 * h);
                x[4 * b] = fmaf(f16_bits_to_f32(s.x & 0xffffu), acc[4 * b], x[4 * b]);
                x[4 * b + 1] = fmaf(f16_bits_to_f32(s.x >> 16), acc[4 * b + 1], x[4 * b + 1]);
                x[4 * b + 2] = fmaf(f16_bits_to_f32(s.y & 0xffffu), acc[4 * b + 2], x[4 * b + 2]);
                x[4 * b + 3] = fmaf(f16_bits_to_f32(s.y >> 16), acc[4 * b + 3], x[4 * b + 3]);
            }
        }
        float mul = xs, tm;
        if (general) {
            tm = ATTN_NONE;
            mul = 1.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int k = 8 * (r >> 2) + 4 * h + (r & 3);
                const bool in = 32 * t + k >= row.lo && 32 * t + k < row.hi && have[r >> 3];
                float y = x[r] * xs;
                if (cap) y = ys * attn_tanh(y);
                x[r] = in ? y : -__builtin_inff();
                tm = fmaxf(tm, x[r] + (float)__builtin_amdgcn_frexp_expf(*(const float*)(buf + T::G + 4 * k)));
                bad |= in ? *(const uint32_t*)(buf + T::BAD + 4 * k) : 0u;
            }
        } else {
            float top = fmaxf(x[0], x[1]);
#pragma unroll
            for (int r = 2; r < 16; ++r) top = fmaxf(top, x[r]);
            tm = fmaf(top, xs, gmax);
        }
        if (__any(tm > M + 8.f)) {
            float u, v;
            half_pair(tm, u, v);
            const float Mn = fmaxf(M, fmaxf(u, v)), f = __builtin_amdgcn_exp2f(M - Mn);
            M = Mn;
            l *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[g][r] *= f;
        }
        const float shift = 7.f - M;
        half8_t ph[2], pl[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4_t hw, lw;
            f32x4_t gk[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) gk[i] = *(const f32x4_t*)(buf + T::G + 32 * (2 * s + i) + 16 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float p[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int r = 8 * s + 2 * i + k;
                    p[k] = __builtin_amdgcn_exp2f(fmaf(x[r], mul, shift));
                    l += p[k];
                    p[k] *= gk[i >> 1][2 * (i & 1) + k];
                }
                const half2_t v = halves(p[0], p[1]);
                hw[i] = __builtin_bit_cast(uint32_t, v);
                lw[i] = __builtin_bit_cast(uint32_t, halves(residual<0>(v, p[0]), residual<1>(v, p[1])));
            }
            ph[s] = __builtin_bit_cast(half8_t, hw);
            pl[s] = __builtin_bit_cast(half8_t, lw);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const unsigned char* const p = buf + vat + 64 * g;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const half8_t vh = v_frag<T::RB>(p + 16 * s * T::RB), vl = v_frag<T::RB>(p + (T::VL - T::VH) + 16 * s * T::RB);
                o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[s], o[g], 0, 0, 0);
                o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[s], o[g], 0, 0, 0);
                o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[s], o[g], 0, 0, 0);
            }
        }
    };

    if (t0 < t1) {
        tile_spread(next, smem);
        if (t0 + 1 < t1) {
            kn = window.of(t0 + 1);
            tile_load(next, a, w, t0 + 1, kn);
        }
    }
    for (int t = t0; t < t1; ++t) {
        const unsigned char* const buf = smem + ((t - t0) & 1) * T::BUF;
        const bool have[2] = {kp.p[0] >= 0, kp.p[1] >= 0};
        __syncthreads();                        // this block of keys is written, the other buffer no longer read
        kp = kn;
        if (t + 1 < t1) {
            tile_spread(next, smem + ((t + 1 - t0) & 1) * T::BUF);
            if (t + 2 < t1) {
                kn = window.of(t + 2);
                tile_load(next, a, w, t + 2, kn);
            }
        }
        if (32 * t >= any_hi || 32 * t + 32 <= any_lo) continue;
        const float e = (float)__builtin_amdgcn_frexp_expf(*(const float*)(buf + T::G + 4 * m));
        const bool odd = *(const uint32_t*)(buf + T::BAD + 4 * m) != 0;
        const float emin = -half_max(-e), emax = half_max(e);
        const bool plain = 32 * t >= all_lo && 32 * t + 32 <= all_hi && have[0] && have[1] && !cap && !__any(odd || emax - emin > 10.f);
        block(!plain, buf, t, have, emax);
    }

    bad |= (uint32_t)__shfl_xor((int)bad, 32);
    if (!row.real) return;
    float u, v;
    half_pair(l, u, v);
    const float L = u + v;
    const bool whole = w.whole;
    const size_t at = part_at(a, w, 0, row.t, row.h);
    float* const dst = (whole ? a.a.out + row.t * a.a.out_stride + (size_t)row.h * D : a.part + at * D) + 4 * h;
    if (!whole && h == 0) {
        a.ml[2 * at] = M;
        a.ml[2 * at + 1] = L;
    }
    const float f = whole ? (L == 0.f ? 0.f : 1.f / L) : 1.f;      // a row that saw no key has sums of 0
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4_t x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (bad >> g) & 1 ? __builtin_nanf("") : o[g][4 * b + i] * f;
            *(f32x4_t*)(dst + 32 * g + 8 * b) = x;
        }
}

}  // namespace

#define BRIK_ATTN_TILE(D, NW)                                                                                            \
    extern "C" __global__ __launch_bounds__(64 * NW, D <= 128 ? 2 : 1) void brik_attn_tile##NW##_q8_##D(brik_attn_launch a) \
    {                                                                                                                     \
        tile_body<FMT_Q8, D, NW>(a);                                                                                      \
    }                                                                                                                     \
    extern "C" __global__ __launch_bounds__(64 * NW, D <= 128 ? 2 : 1) void brik_attn_tile##NW##_q4_##D(brik_attn_launch a) \
    {                                                                                                                     \
        tile_body<FMT_Q4, D, NW>(a);                                                                                      \
    }
BRIK_ATTN_TILE(64, 4)
BRIK_ATTN_TILE(96, 4)
BRIK_ATTN_TILE(128, 4)
BRIK_ATTN_TILE(192, 4)
BRIK_ATTN_TILE(256, 4)
BRIK_ATTN_TILE(64, 8)
BRIK_ATTN_TILE(96, 8)
BRIK_ATTN_TILE(128, 8)
