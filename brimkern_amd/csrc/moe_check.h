// The argument checks of a mixture-of-experts layer's entry points and of the 8-bit products, apart from any context: each
// returns BRIK_OK or the code of the refusal, with its reason in `why`.
#pragma once
#include "attn_check.h"
#include "kernels/moe_abi.h"

namespace brik_check {

inline int places(Why& w, const char* who, int tokens, int k)
{
    if (tokens < 0 || k < 0) return no(w, BRIK_EINVAL, "%s: negative size tokens=%d k=%d", who, tokens, k);
    if (tokens >= 1 << 24) return no(w, BRIK_EINVAL, "%s: %d tokens exceed 2^24 - 1 in one call", who, tokens);
    if (k > BRIK_MOE_K) return no(w, BRIK_EINVAL, "%s: k=%d exceeds %d", who, k, BRIK_MOE_K);
    if ((long long)tokens * k > (1ll << 30)) return no(w, BRIK_EINVAL, "%s: tokens * k = %lld exceeds 2^30", who, (long long)tokens * k);
    return BRIK_OK;
}

inline int experts(Why& w, const char* who, int E)
{
    if (E < 0 || E > BRIK_MOE_EXPERTS) return no(w, BRIK_EINVAL, "%s: %d experts (0 to %d)", who, E, BRIK_MOE_EXPERTS);
    return BRIK_OK;
}

inline int sorted(Why& w, const char* who, const int32_t* row_off, const int32_t* src, const int32_t* slot, bool any)
{
    if (!row_off || (any && (!src || !slot))) return no(w, BRIK_EINVAL, "%s: row_off, src or slot is null", who);
    if (off(row_off, 4) || off(src, 4) || off(slot, 4)) return no(w, BRIK_EALIGN, "%s: row_off, src and slot must be 4-byte aligned", who);
    return BRIK_OK;
}

// `r` comes back with its stride filled in. grad: ids are read, weights and the sorted arrays not looked at.
inline int route(Why& w, const char* who, brik_moe_route_args& r, bool grad)
{
    BRIK_CHECK(places(w, who, r.tokens, r.k));
    BRIK_CHECK(experts(w, who, r.experts));
    if (r.k > r.experts) return no(w, BRIK_EINVAL, "%s: k=%d of %d experts", who, r.k, r.experts);
    if (r.flags & ~(BRIK_ROUTE_SIGMOID | BRIK_ROUTE_RENORM)) return no(w, BRIK_EINVAL, "%s: unknown flags 0x%x", who, (unsigned)r.flags);
    if (r.reserved) return no(w, BRIK_EINVAL, "%s: reserved must be 0", who);
    if (!std::isfinite(r.scale)) return no(w, BRIK_EINVAL, "%s: scale %g", who, (double)r.scale);
    if (r.logit_stride == 0) r.logit_stride = r.experts;
    if (r.logit_stride < r.experts)
        return no(w, BRIK_EINVAL, "%s: logit_stride %lld is less than %d experts", who, (long long)r.logit_stride, r.experts);
    const bool any = (long long)r.tokens * r.k > 0;
    if (!grad && (r.row_off || r.src || r.slot)) BRIK_CHECK(sorted(w, who, r.row_off, r.src, r.slot, any));
    if (grad ? r.tokens > 0 && r.experts > 0 && !r.logits : any && !r.logits) return no(w, BRIK_EINVAL, "%s: logits is null", who);
    if (any && (!r.ids || (!grad && !r.weights))) return no(w, BRIK_EINVAL, "%s: ids or weights is null", who);
    if (off(r.logits, 4) || off(r.bias, 4) || off(r.ids, 4) || off(r.weights, 4))
        return no(w, BRIK_EALIGN, "%s: logits, bias, ids and weights must be 4-byte aligned", who);
    return BRIK_OK;
}

// Rows of `width` values to and from the experts.
inline int spread(Why& w, const char* who, int tokens, int k, int width, const int32_t* slot, const float* weights)
{
    BRIK_CHECK(places(w, who, tokens, k));
    if (width < 0 || width % 4) return no(w, BRIK_EINVAL, "%s: width %d is not a multiple of 4", who, width);
    if ((long long)tokens * k > 0 && !slot) return no(w, BRIK_EINVAL, "%s: slot is null", who);
    if (off(slot, 4) || off(weights, 4)) return no(w, BRIK_EALIGN, "%s: slot and weights must be 4-byte aligned", who);
    return BRIK_OK;
}

inline int rows16(Why& w, const char* who, const char* name, const void* p, bool needed)
{
    if (needed && !p) return no(w, BRIK_EINVAL, "%s: %s is null", who, name);
    if (off(p, 16)) return no(w, BRIK_EALIGN, "%s: %s must be 16-byte aligned", who, name);
    return BRIK_OK;
}

inline int quantize_i8(Why& w, const char* who, brik_quant_launch& a, int flags)
{
    if (a.M < 0 || a.K < 0) return no(w, BRIK_EINVAL, "%s: negative shape M=%d K=%d", who, a.M, a.K);
    if (a.K % 32) return no(w, BRIK_EINVAL, "%s: K=%d is not a multiple of 32", who, a.K);
    if (a.M >= 1 << 22) return no(w, BRIK_EINVAL, "%s: %d rows exceed 2^22 - 1 in one call", who, a.M);
    if (flags & ~BRIK_JOB_ACT_GELU) return no(w, BRIK_EINVAL, "%s: unknown flags 0x%x", who, (unsigned)flags);
    BRIK_CHECK(stride(w, who, "x", a.x_stride, a.K));
    BRIK_CHECK(stride(w, who, "gate", a.gate_stride, a.K));
    if (a.M == 0) return BRIK_OK;
    BRIK_CHECK(rows16(w, who, "x", a.x, a.K > 0));
    BRIK_CHECK(rows16(w, who, "gate", a.gate, false));
    BRIK_CHECK(rows16(w, who, "codes", a.codes, a.K > 0));
    if (!a.scales) return no(w, BRIK_EINVAL, "%s: scales is null", who);
    if (off(a.scales, 4)) return no(w, BRIK_EALIGN, "%s: scales must be 4-byte aligned", who);
    return BRIK_OK;
}

// M, K and N of the launch, and its pointers; by experts E of them (0: dense).
inline int product_i8(Why& w, const char* who, const brik_i8_launch& a, bool moe)
{
    if (a.M < 0 || a.K < 0 || a.N < 0) return no(w, BRIK_EINVAL, "%s: negative shape M=%d K=%d N=%d", who, a.M, a.K, a.N);
    if (a.M > 1 << 30) return no(w, BRIK_EINVAL, "%s: %d rows exceed 2^30 in one call", who, a.M);
    if (a.K % 32 || a.K > BRIK_I8_K) return no(w, BRIK_EINVAL, "%s: K=%d is not a multiple of 32 up to %d", who, a.K, BRIK_I8_K);
    if (moe) {
        if (a.E < 0 || a.E > 65536) return no(w, BRIK_EINVAL, "%s: %d experts (0 to 65536)", who, a.E);
        if (a.src && a.k < 1) return no(w, BRIK_EINVAL, "%s: src with k=%d", who, a.k);
        if (a.src && (long long)a.x_rows * a.K >= (1ll << 32))
            return no(w, BRIK_EINVAL, "%s: x of %d rows of %d values found by src exceeds 2^32", who, a.x_rows, a.K);
        if (a.x_rows < 0 || (!a.src && a.x_rows < a.M)) return no(w, BRIK_EINVAL, "%s: x of %d rows for %d", who, a.x_rows, a.M);
    }
    if ((long long)a.N * a.K >= (1ll << 32)) return no(w, BRIK_EINVAL, "%s: N*K = %lld exceeds the 2^32 per-tensor limit", who, (long long)a.N * a.K);
    if (a.N >= 1 << 22) return no(w, BRIK_EINVAL, "%s: N=%d exceeds 2^22 - 1 channels", who, a.N);
    if (a.M == 0 || a.N == 0 || (moe && a.E == 0)) return BRIK_OK;
    if (!a.y) return no(w, BRIK_EINVAL, "%s: y is null", who);
    if (off(a.y, 4) || off(a.res, 4)) return no(w, BRIK_EALIGN, "%s: y and res must be 4-byte aligned", who);
    if (moe && !a.row_off) return no(w, BRIK_EINVAL, "%s: row_off is null", who);
    if (moe && (off(a.row_off, 4) || off(a.src, 4))) return no(w, BRIK_EALIGN, "%s: row_off and src must be 4-byte aligned", who);
    if (a.K > 0) {
        BRIK_CHECK(rows16(w, who, "x", a.x, !moe || a.x_rows > 0));
        BRIK_CHECK(rows16(w, who, "w", a.w, true));
    }
    if ((!a.xs && (!moe || a.x_rows > 0)) || !a.ws) return no(w, BRIK_EINVAL, "%s: null scales", who);
    if (off(a.xs, 4) || off(a.ws, 4)) return no(w, BRIK_EALIGN, "%s: scales must be 4-byte aligned", who);
    return BRIK_OK;
}

}  // namespace brik_check
