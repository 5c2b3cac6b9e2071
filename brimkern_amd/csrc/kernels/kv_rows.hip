// The rows of a step on their way into attention: head norms and rotation of q and k, keys and values quantized into
// the cache, and cached tokens read back (the reference's rope / quantize_kv, src/lib/webgpu/shaders.ts:1361, 1673).
//
//   y = x / sqrt(sum(x^2) / D + eps) * g,   (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = p * inv_freq[i]
//
// Everything up to the one rounding to f32 is in 64 bits: a code of the cache is the rounding of y / scale, so
// with f32 sums the order of a sum, or whether the rotation is fused with the write, would move codes by one.
//
// A team of TL lanes (head_dim / 4, rounded up to a power of two) holds one head of one row, four values a lane, so a
// quantization group is 8 neighbouring lanes; sums over a head and the scales of a group are cross-lane reductions, and
// no value passes through LDS. A block works on one row: its cosines and sines are computed once in LDS and serve
// all its heads. Long prompts are bound by memory where rows are normed and rotated (2048 rows of 40 heads of 128: 84 MB in 21 us,
// 4.0 TB/s) and read back (4096 tokens of 16 heads 10 us), by vector instructions where they are written (the same tokens as q8
// 14 us, 90 % of the issue cycles), single rows by the latency of the 64-bit arithmetic (4 us).
#include "attn_common.h"
#include "encode.h"

namespace {

// cos and sin of an angle in radians, |a| < 2^31: a - n pi/2 by two fused multiply-adds with pi/2 in two parts (n has
// up to 31 bits, so the first difference is exact to 2^-53 and the second part's error is below 2^-75), then the
// Taylor series on [-pi/4, pi/4], whose first terms left out are below 2^-63.
__device__ __forceinline__ void cos_sin(double a, double& c, double& s)
{
    const double n = rint(a * 0x1.45f306dc9c883p-1);                          // 2 / pi
    double r = fma(n, -0x1.921fb54442d18p+0, a);                              // pi / 2
    r = fma(n, -0x1.1a62633145c07p-54, r);
    const double z = r * r;
    double p = 1.0 / 355687428096000.0;                                       // 1 / 17!
    p = fma(p, z, -1.0 / 1307674368000.0);
    p = fma(p, z, 1.0 / 6227020800.0);
    p = fma(p, z, -1.0 / 39916800.0);
    p = fma(p, z, 1.0 / 362880.0);
    p = fma(p, z, -1.0 / 5040.0);
    p = fma(p, z, 1.0 / 120.0);
    p = fma(p, z, -1.0 / 6.0);
    const double sr = fma(p * z, r, r);
    double q = -1.0 / 6402373705728000.0;                                     // -1 / 18!
    q = fma(q, z, 1.0 / 20922789888000.0);
    q = fma(q, z, -1.0 / 87178291200.0);
    q = fma(q, z, 1.0 / 479001600.0);
    q = fma(q, z, -1.0 / 3628800.0);
    q = fma(q, z, 1.0 / 40320.0);
    q = fma(q, z, -1.0 / 720.0);
    q = fma(q, z, 1.0 / 24.0);
    q = fma(q, z, -0.5);
    const double cr = fma(q, z, 1.0);
    const int k = (int)(long long)n & 3;
    const double cc = k & 1 ? sr : cr, ss = k & 1 ? cr : sr;
    c = k == 1 || k == 2 ? -cc : cc;
    s = k & 2 ? -ss : ss;
}

// Sum over a team of TL lanes.
template <int TL>
__device__ __forceinline__ double team_sum(double v)
{
#pragma unroll
    for (int m = 1; m < TL; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// Minimum over aligned groups of 8 lanes.
__device__ __forceinline__ float min8(float v) { return -max8(-v); }

// x (four values of a head, this lane's) into group codes at `vec` of the planes. Every lane of the group takes part.
template <int FMT>
__device__ __forceinline__ void put(f32x4_t x, const brik_kv_cache& c, bool value, size_t vec, int lane, bool live)
{
    const int D = c.head_dim;
    uint8_t* const code = (uint8_t*)(value ? c.v : c.k);
    const size_t grp = vec * (size_t)(D / BRIK_GROUP) + (lane >> 3);
    const float e[4] = {x.x, x.y, x.z, x.w};
    bool unsure;
    if constexpr (FMT == FMT_Q8) {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(__builtin_canonicalizef(e[i])));
        amax = max8(amax);
        const uint32_t sh = f16_encode(or_tiny((double)amax / 127.0));
        const double s = or_tiny((double)f16_decode(sh));
        const FastConst fk = fast_const(s, 0.0, unsure);
        uint32_t word = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            word |= ((uint32_t)code_fast<-127, 127>(e[i], fk.r, fk.c, fk.er, fk.h0, unsure) & 0xffu) << (8 * i);
        if (unsure) {
            word = 0u;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) word |= ((uint32_t)code_exact((double)x[i], s, -127.0, 127.0) & 0xffu) << (8 * i);
        }
        if (!live) return;
        *(uint32_t*)(code + vec * D + 4 * lane) = word;
        if ((lane & 7) == 0) (value ? c.v_scales : c.k_scales)[grp] = (uint16_t)sh;
    } else {
        float mn = __builtin_inff(), mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = __builtin_canonicalizef(e[i]);
            mn = fminf(mn, v);
            mx = fmaxf(mx, v);
        }
        mn = min8(mn);
        mx = max8(mx);
        if (mn == 0.f) {
            // the encoder keeps the first of equal values, +0 or -0: the first zero of the group in order
            uint32_t first = 0xffffffffu;
#pragma unroll
            for (int i = 3; i >= 0; --i)
                if (e[i] == 0.f) first = (uint32_t)(((lane & 7) * 4 + i) * 2) | (__builtin_bit_cast(uint32_t, e[i]) >> 31);
            first = min(first, (uint32_t)__builtin_amdgcn_mov_dpp((int)first, DPP_QUAD_1032, 0xF, 0xF, false));
            first = min(first, (uint32_t)__builtin_amdgcn_mov_dpp((int)first, DPP_QUAD_2301, 0xF, 0xF, false));
            first = min(first, (uint32_t)__builtin_amdgcn_mov_dpp((int)first, DPP_ROW_HALF_MIRROR, 0xF, 0xF, false));
            mn = first & 1 ? -0.f : 0.f;
        }
        const uint32_t sh = f16_encode(or_tiny(((double)mx - (double)mn) / 15.0)), mh = f16_encode((double)mn);
        const double s = or_tiny((double)f16_decode(sh)), m = (double)f16_decode(mh);
        const FastConst fk = fast_const(s, m, unsure);
        uint32_t half = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) half |= (uint32_t)code_fast<0, 15>(e[i], fk.r, fk.c, fk.er, fk.h0, unsure) << (4 * i);
        if (unsure) {
            half = 0u;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) half |= (uint32_t)code_exact((double)x[i] - m, s, 0.0, 15.0) << (4 * i);
        }
        if (!live) return;
        *(uint16_t*)(code + vec * (D / 2) + 2 * lane) = (uint16_t)half;
        if ((lane & 7) == 0) {
            (value ? c.v_scales : c.k_scales)[grp] = (uint16_t)sh;
            (value ? c.v_mins : c.k_mins)[grp] = (uint16_t)mh;
        }
    }
}

__device__ __forceinline__ f32x4_t load4(const float* p) { return *(const f32x4_t*)p; }

// FMT 0: no cache (norm and rotation only).
template <int TL, int FMT>
__device__ __forceinline__ void rows_body(const brik_rows_launch& a)
{
    __shared__ __attribute__((aligned(16))) double cs[2 * 128];
    const brik_qkv_rows& r = a.r;
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid % TL, D = r.head_dim, half = r.rot_dim / 2;
    const bool turn = r.inv_freq != nullptr, inter = r.flags & BRIK_QKV_INTERLEAVED;
    const int units = a.nq + a.nk + a.nv, e0 = 4 * lane;
    const bool in = e0 < D;
    const int u0 = blockIdx.y * (256 / TL) + tid / TL;
    // the first head's load is on its way before the row's sequence, page and angles are known (2 % of 84 MB, 0.1 us of one row)
    const float* const q0 = r.q + t * r.q_stride;
    const float* const k0 = r.k + t * r.k_stride - (size_t)a.nq * D;
    const float* const v0 = r.v + t * r.v_stride - (size_t)(a.nq + a.nk) * D;
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
    if (in && u0 < units) x = load4((u0 < a.nq ? q0 : u0 < a.nq + a.nk ? k0 : v0) + (size_t)u0 * D + e0);
    int b = 0;
    int32_t pos = 0, page = -1;
    if (FMT || (turn && !r.positions)) {
        b = seq_of_row(a.s, t);
        if (b >= a.s.seqs) return;                       // of no sequence
        pos = row_position(a.s, b, t);
    } else if (!brik_row_taken(a.s, t)) {
        return;
    }
    if (FMT && pos >= a.s.prefix_len) page = brik_page_of(a.s, b, pos);
    if (turn) {
        const double at = (double)(r.positions ? r.positions[t] : pos);
        for (int i = tid; i < half; i += 256) {
            double c, s;
            cos_sin(at * (double)r.inv_freq[i], c, s);
            cs[2 * i] = c;
            cs[2 * i + 1] = s;
        }
        __syncthreads();
    }
    for (int u = u0; u < units; u += gridDim.y * (256 / TL)) {
        const bool isq = u < a.nq, isk = !isq && u < a.nq + a.nk;
        const int h = isq ? u : isk ? u - a.nq : u - a.nq - a.nk;
        const float* const src = (isq ? q0 : isk ? k0 : v0) + (size_t)u * D;
        if (in && u != u0) x = load4(src + e0);
        if (isq || isk) {
            const float* const w = isq ? r.q_norm : r.k_norm;
            const bool rot = turn && e0 < r.rot_dim;
            // the other value of each pair: in this lane, or half the rotated values away
            const int pe = e0 < half ? e0 + half : e0 - half;
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
            if (rot && !inter) o = load4(src + pe);
            double y[4], z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                y[i] = (double)x[i];
                z[i] = (double)o[i];
            }
            if (w) {
                const double ss = team_sum<TL>(y[0] * y[0] + y[1] * y[1] + (y[2] * y[2] + y[3] * y[3]));
                const double inv = 1.0 / sqrt(ss / (double)D + (double)r.eps);
                const double one = r.flags & BRIK_QKV_GAIN_ONE_PLUS ? 1.0 : 0.0;
                if (in) {
                    const f32x4_t g = load4(w + e0);
                    f32x4_t go = g;
                    if (rot && !inter) go = load4(w + pe);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[i] *= inv * ((double)g[i] + one);
                        z[i] *= inv * ((double)go[i] + one);
                    }
                }
            }
            if (rot) {
                if (inter) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const double c = cs[e0 + 2 * j], s = cs[e0 + 2 * j + 1], p = y[2 * j], q = y[2 * j + 1];
                        y[2 * j] = p * c - q * s;
                        y[2 * j + 1] = q * c + p * s;
                    }
                } else {
                    const bool first = e0 < half;
                    const int i0 = first ? e0 : e0 - half;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const double c = cs[2 * (i0 + i)], s = cs[2 * (i0 + i) + 1];
                        y[i] = fma(first ? -z[i] : z[i], s, y[i] * c);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (float)y[i];
            float* const dst = isq ? r.q_out + t * r.q_out_stride : r.k_out ? r.k_out + t * r.k_out_stride : nullptr;
            if (dst && in) *(f32x4_t*)(dst + (size_t)h * D + e0) = x;
        }
        if constexpr (FMT != 0) {
            if (!isq && page >= 0)
                put<FMT>(x, a.c, !isk, brik_vector(a.s, a.c.heads, page, h, brik_slot(a.s, pos)), lane, in);
        }
    }
}

// One head of one cached token per team of head_dim / 4 lanes, four values a lane: 16-byte stores of consecutive values,
// which are four fifths of the bytes and more.
template <int FMT>
__device__ __forceinline__ void read_body(const brik_read_launch& a)
{
    const brik_kv_cache& c = a.c;
    const int t = blockIdx.x, D = c.head_dim, quads = D / 4, G = D / BRIK_GROUP;
    const int b = seq_of_row(a.s, t);
    if (b >= a.s.seqs) return;
    const int32_t pos = row_position(a.s, b, t), page = brik_page_of(a.s, b, pos);
    const size_t first = page < 0 ? 0 : brik_vector(a.s, c.heads, page, 0, brik_slot(a.s, pos));
    const int each = c.heads * quads, n = (a.k ? each : 0) + (a.v ? each : 0);
    for (int i = blockIdx.y * 256 + threadIdx.x; i < n; i += gridDim.y * 256) {
        const bool value = !a.k || i >= each;
        const int j = value && a.k ? i - each : i, h = j / quads, q = j - h * quads;
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
        if (page >= 0) {
            const size_t vec = first + ((size_t)h << a.s.shift), grp = vec * G + (q >> 3);
            const uint8_t* const code = (const uint8_t*)(value ? c.v : c.k);
            const float s = f16_bits_to_f32((value ? c.v_scales : c.k_scales)[grp]);
            if constexpr (FMT == FMT_Q8) {
                const uint32_t w = *(const uint32_t*)(code + vec * D + 4 * q);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (float)(int8_t)byte_of(w, e) * s;
            } else {
                const uint32_t w = *(const uint16_t*)(code + vec * (D / 2) + 2 * q);
                const float m = f16_bits_to_f32((value ? c.v_mins : c.k_mins)[grp]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf((float)((w >> (4 * e)) & 15u), s, m);
            }
        }
        *(f32x4_t*)((value ? a.v : a.k) + ((size_t)t * c.heads + h) * D + 4 * q) = x;
    }
}

}  // namespace

#define BRIK_ROWS(TL)                                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void brik_rows_rope_##TL(brik_rows_launch a) { rows_body<TL, 0>(a); }      \
    extern "C" __global__ __launch_bounds__(256) void brik_rows_q8_##TL(brik_rows_launch a) { rows_body<TL, FMT_Q8>(a); }   \
    extern "C" __global__ __launch_bounds__(256) void brik_rows_q4_##TL(brik_rows_launch a) { rows_body<TL, FMT_Q4>(a); }
BRIK_ROWS(8)
BRIK_ROWS(16)
BRIK_ROWS(32)
BRIK_ROWS(64)

extern "C" __global__ __launch_bounds__(256) void brik_kv_read_q8(brik_read_launch a) { read_body<FMT_Q8>(a); }
extern "C" __global__ __launch_bounds__(256) void brik_kv_read_q4(brik_read_launch a) { read_body<FMT_Q4>(a); }
