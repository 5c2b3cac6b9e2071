// The arithmetic of the .brik encoders (quantizeQ8 / Q4 / Q3 and f32ToF16Bits: src/lib/brik/q8web.ts:28-50,
// q4web.ts:28-53, q3web.ts:34-60, f16.ts:8-22), shared by the tensor encoders (quantize.hip) and the cache writes
// (kv_rows.hip), so that both give the same bytes for the same values.
#pragma once
#include "common.h"

namespace {

// f32ToF16Bits: the value rounded to f32, then sign | exponent | 10-bit mantissa rounded half up on
// the first dropped bit; exponents below the normal range give +-0, above it +-65504 (0x7bff), and a
// mantissa carry out of exponent 30 gives the infinity bits, as the reference's conversion does.
// Branch-free: the rounded mantissa is added to the shifted exponent, so a carry out of the mantissa
// (r = 0x400) increments the exponent and clears the mantissa bits.
__device__ __forceinline__ uint32_t f16_encode(double v)
{
    const uint32_t x = __builtin_bit_cast(uint32_t, (float)v);
    const uint32_t sign = (x >> 16) & 0x8000u;
    const int exp = (int)((x >> 23) & 0xffu) - 127 + 15;
    const uint32_t mant = x & 0x7fffffu;
    const uint32_t body = ((uint32_t)exp << 10) + (mant >> 13) + ((mant >> 12) & 1u);
    return sign | (exp <= 0 ? 0u : exp >= 31 ? 0x7bffu : body);
}

// f16BitsToF32 for the bits f16_encode produces (no subnormals, no NaN; the infinity bits decode to
// infinity): the exact value, through the hardware conversion (every f16 value is an f32 value).
__device__ __forceinline__ float f16_decode(uint32_t h)
{
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// JavaScript's `v || 1e-8` for a number: 0 and NaN are falsy.
__device__ __forceinline__ double or_tiny(double v) { return (v == 0.0 || v != v) ? 1e-8 : v; }

// Math.round: the nearest integer, ties toward +infinity (exact for every double: v - floor(v) is
// exact below 2^52 and v is integral above). NaN stays NaN.
__device__ __forceinline__ double js_round(double v)
{
    const double f = floor(v);
    return v - f >= 0.5 ? f + 1.0 : f;
}

// The integer a clamped code becomes when stored into a typed array (NaN -> 0).
__device__ __forceinline__ int code_of(double q, double lo, double hi)
{
    if (q != q) return 0;
    q = q < lo ? lo : q > hi ? hi : q;
    return (int)q;
}

// The code of one value exactly as the reference computes it: Math.round(d / s) with the f64
// division, clamped to [lo, hi].
__device__ __forceinline__ int code_exact(double d, double s, double lo, double hi)
{
    return code_of(js_round(d / s), lo, hi);
}

// v_cvt_i32_f32: the integer part, saturating, with NaN -> 0 (the hardware conversion; a C cast of
// NaN would be undefined).
__device__ __forceinline__ int cvt_i32(float v)
{
    int r;
    asm("v_cvt_i32_f32 %0, %1" : "=v"(r) : "v"(v));
    return r;
}

// The same code in f32, without a division. Per group: r = 1 / s to within 2^-23 relative (v_rcp_f32),
// c = 1/2 - m r (two f32 roundings). Per value, u = x r + c with one rounding: against the exact
// U = (x - m) / s + 1/2, |u - U| <= 5 * 2^-24 (|x| + |m|) / s + 2^-24 (the r error on both products,
// the roundings of m r, of c and of u, and |U| <= (|x| + |m|) / s + 1/2). JavaScript's f64 quotient,
// rounded half up, is floor of a value within 2^-52 (|x| + |m|) / s + 2^-53 of U. The margin
// e = (|x| + |m|) r 2^-20, about 16 * 2^-24 (|x| + |m|) / s, covers both whenever u lies near an
// integer (then |x - m| / s >= 1/2, so the absolute terms are at most 4 * 2^-24 (|x| + |m|) / s);
// far from one, when (|x| + |m|) / s < 1/11, u is within 0.1 of 1/2. So when u is farther than e
// from every integer, floor(u) is JavaScript's Math.round. Otherwise `unsure` is set and the caller
// redoes the group with code_exact (rare for weights: exact ties, values within about 2^-20 of one,
// or groups far from zero relative to their spread).
// NaN gives 0 and infinities saturate before the clamp, as the reference's stores and clamp do. For
// lo = 0 the truncating conversion gives the clamped floor (they differ only below 0), so no floor
// is taken. Per group: `c`, `er` = r 2^-20 and `h0` = 1/2 - |m| er; then 1/2 - e = h0 - |x| er.
template <int LO, int HI>
__device__ __forceinline__ int code_fast(float x, float r, float c, float er, float h0, bool& unsure)
{
    const float u = fmaf(x, r, c);
    const float h = fmaf(-fabsf(x), er, h0);
    int q;
    if constexpr (LO == 0) {
        unsure |= fabsf(__builtin_amdgcn_fractf(u) - 0.5f) >= h;
        q = cvt_i32(u);
    } else {
        const float fu = floorf(u);
        unsure |= fabsf((u - fu) - 0.5f) >= h;
        q = cvt_i32(fu);
    }
    return q < LO ? LO : q > HI ? HI : q;
}

// The per-group constants of code_fast for scale s and min m. A non-finite c (m infinite) marks the
// group unsure.
struct FastConst {
    float r, c, er, h0;
};
__device__ __forceinline__ FastConst fast_const(double s, double m, bool& unsure)
{
    FastConst k;
    const float mf = (float)m;
    k.r = __builtin_amdgcn_rcpf((float)s);
    k.c = 0.5f - mf * k.r;
    k.er = k.r * 0x1p-20f;
    k.h0 = 0.5f - fabsf(mf) * k.er;
    unsure = !(fabsf(k.c) <= 3.4028235e38f);
    return k;
}

}  // namespace
