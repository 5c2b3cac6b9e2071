// The argument checks of the attention side's entry points, apart from any context: each returns BRIK_OK or the code of
// the refusal, with its reason in `why`.
#pragma once
#include "kernels/attn_abi.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace brik_check {

struct Why {
    char text[256] = {0};
};

inline int no(Why& w, int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(w.text, sizeof w.text, fmt, ap);
    va_end(ap);
    return code;
}

inline bool off(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

inline int cache(Why& w, const char* who, const brik_kv_cache* c)
{
    if (!c) return no(w, BRIK_EINVAL, "%s: cache is null", who);
    if (c->fmt != BRIK_FMT_Q8 && c->fmt != BRIK_FMT_Q4) return no(w, BRIK_EINVAL, "%s: cache format %d (8 or 4)", who, c->fmt);
    if (c->reserved) return no(w, BRIK_EINVAL, "%s: cache.reserved must be 0", who);
    if (c->heads < 1 || c->pages < 1) return no(w, BRIK_EINVAL, "%s: cache of %d pages, %d heads", who, c->pages, c->heads);
    if (c->head_dim < 32 || c->head_dim > 256 || c->head_dim % 32)
        return no(w, BRIK_EINVAL, "%s: head_dim %d is not a multiple of 32 up to 256", who, c->head_dim);
    if (c->page < 16 || c->page > 65536 || (c->page & (c->page - 1)))
        return no(w, BRIK_EINVAL, "%s: page %d is not a power of two from 16 to 65536", who, c->page);
    // a page's heads are addressed by 64-bit offsets, a vector within them by 32-bit ones
    if ((long long)c->heads * c->page * c->head_dim >= (1ll << 31))
        return no(w, BRIK_EINVAL, "%s: heads * page * head_dim = %lld values per page exceed 2^31", who,
                  (long long)c->heads * c->page * c->head_dim);
    const bool q4 = c->fmt == BRIK_FMT_Q4;
    if (!c->k || !c->v || !c->k_scales || !c->v_scales || (q4 && (!c->k_mins || !c->v_mins)))
        return no(w, BRIK_EINVAL, "%s: null cache plane", who);
    if (off(c->k, 16) || off(c->v, 16) || off(c->k_scales, 16) || off(c->v_scales, 16) ||
        (q4 && (off(c->k_mins, 16) || off(c->v_mins, 16))))
        return no(w, BRIK_EALIGN, "%s: cache planes must be 16-byte aligned", who);
    return BRIK_OK;
}

// tokens: the call looks tokens up (lengths and tables needed); lens: it needs their positions.
inline int batch(Why& w, const char* who, const brik_kv_batch* b, bool tokens, bool lens)
{
    if (!b) return no(w, BRIK_EINVAL, "%s: batch is null", who);
    if (b->seqs < 0 || b->rows < 0 || b->table_cols < 0 || b->max_len < 0 || b->max_rows < 0 || b->prefix_len < 0)
        return no(w, BRIK_EINVAL, "%s: negative size in the batch", who);
    if (b->rows > (1 << 24) - 1) return no(w, BRIK_EINVAL, "%s: %d rows exceed 2^24 - 1 in one call", who, b->rows);
    if (b->rows == 0) return BRIK_OK;
    if (off(b->row_off, 4)) return no(w, BRIK_EALIGN, "%s: row_off must be 4-byte aligned", who);
    if (!tokens && !lens) return BRIK_OK;
    if (b->seqs == 0) return no(w, BRIK_EINVAL, "%s: %d rows of no sequences", who, b->rows);
    if (!b->row_off && b->rows % b->seqs)
        return no(w, BRIK_EINVAL, "%s: %d rows do not divide over %d sequences and row_off is null", who, b->rows, b->seqs);
    if (!b->kv_len) return no(w, BRIK_EINVAL, "%s: kv_len is null", who);
    if (off(b->kv_len, 4) || off(b->table, 4) || off(b->prefix_table, 4))
        return no(w, BRIK_EALIGN, "%s: kv_len and the tables must be 4-byte aligned", who);
    if (!tokens) return BRIK_OK;
    if (b->table_cols > 0 && !b->table) return no(w, BRIK_EINVAL, "%s: table is null", who);
    if (b->prefix_len > 0 && !b->prefix_table) return no(w, BRIK_EINVAL, "%s: prefix_table is null", who);
    if (b->max_rows > 0 && !b->row_off && b->rows / b->seqs > b->max_rows)
        return no(w, BRIK_EINVAL, "%s: %d rows a sequence, max_rows %d", who, b->rows / b->seqs, b->max_rows);
    return BRIK_OK;
}

// A row stride in values; fills in the packed one.
inline int stride(Why& w, const char* who, const char* name, int64_t& s, int64_t packed)
{
    if (s == 0) s = packed;
    if (s < packed || s % 4)
        return no(w, BRIK_EINVAL, "%s: %s_stride %lld (a multiple of 4, at least %lld)", who, name, (long long)s, (long long)packed);
    return BRIK_OK;
}

#define BRIK_CHECK(call)             \
    do {                             \
        const int r_ = (call);       \
        if (r_ != BRIK_OK) return r_; \
    } while (0)

// Whether rows of aw values, as apart, and of bw values, bs apart, share memory. Of the same stride they may lie side by side in the
// rows of one buffer; of others only their ranges are compared.
inline bool overlap(const float* a, int64_t as, int64_t aw, const float* b, int64_t bs, int64_t bw, int rows)
{
    if (rows <= 0) return false;
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    const uintptr_t a1 = a0 + 4 * (uintptr_t)((rows - 1) * as + aw), b1 = b0 + 4 * (uintptr_t)((rows - 1) * bs + bw);
    if (!(a0 < b1 && b0 < a1)) return false;
    if (as != bs || a0 % 4 != b0 % 4) return true;
    const int64_t apart = ((int64_t)(b0 - a0) / 4 % as + as) % as;       // b's first column, counted from a's
    return apart < aw || apart + bw > as;
}

// write: into a cache (else only norm and rotation). `r` comes back with its strides filled in.
inline int rows(Why& w, const char* who, const brik_kv_cache* c, const brik_kv_batch* b, brik_qkv_rows& r, bool write)
{
    const int D = r.head_dim;
    if (D < 32 || D > 256 || D % 32) return no(w, BRIK_EINVAL, "%s: head_dim %d is not a multiple of 32 up to 256", who, D);
    if (r.flags & ~(BRIK_QKV_GAIN_ONE_PLUS | BRIK_QKV_INTERLEAVED)) return no(w, BRIK_EINVAL, "%s: unknown flags 0x%x", who, (unsigned)r.flags);
    if (r.heads < 0 || r.kv_heads < 0 || r.heads > 65536 || r.kv_heads > 65536)
        return no(w, BRIK_EINVAL, "%s: heads %d, kv_heads %d", who, r.heads, r.kv_heads);
    if (write && (D != c->head_dim || r.kv_heads != c->heads))
        return no(w, BRIK_EINVAL, "%s: rows of %d heads of %d, a cache of %d heads of %d", who, r.kv_heads, D, c->heads, c->head_dim);
    if (write && (!r.k || !r.v)) return no(w, BRIK_EINVAL, "%s: k or v is null", who);
    if (r.q && (!r.q_out || r.heads < 1)) return no(w, BRIK_EINVAL, "%s: q without q_out or heads", who);
    if (!write && ((r.k && !r.k_out) || (r.k && r.kv_heads < 1))) return no(w, BRIK_EINVAL, "%s: k without k_out or kv_heads", who);
    if (off(r.q, 16) || off(r.k, 16) || off(r.v, 16) || off(r.q_out, 16) || off(r.k_out, 16) || off(r.q_norm, 16) || off(r.k_norm, 16))
        return no(w, BRIK_EALIGN, "%s: q, k, v, their outputs and the norm weights must be 16-byte aligned", who);
    if (r.inv_freq) {
        if (r.rot_dim < 8 || r.rot_dim > D || r.rot_dim % 8)
            return no(w, BRIK_EINVAL, "%s: rot_dim %d (a multiple of 8 up to head_dim %d)", who, r.rot_dim, D);
        if (off(r.inv_freq, 4) || off(r.positions, 4)) return no(w, BRIK_EALIGN, "%s: inv_freq and positions must be 4-byte aligned", who);
    }
    if (!(r.eps >= 0) || !std::isfinite(r.eps)) return no(w, BRIK_EINVAL, "%s: eps %g", who, (double)r.eps);
    const int64_t qw = (int64_t)r.heads * D, kw = (int64_t)r.kv_heads * D;
    BRIK_CHECK(stride(w, who, "q", r.q_stride, qw));
    BRIK_CHECK(stride(w, who, "k", r.k_stride, kw));
    BRIK_CHECK(stride(w, who, "v", r.v_stride, kw));
    BRIK_CHECK(stride(w, who, "q_out", r.q_out_stride, qw));
    BRIK_CHECK(stride(w, who, "k_out", r.k_out_stride, kw));
    if ((r.q && r.q_out == r.q && r.q_out_stride != r.q_stride) || (r.k && r.k_out == r.k && r.k_out_stride != r.k_stride))
        return no(w, BRIK_EINVAL, "%s: an output in place needs its input's stride", who);
    (void)b;
    return BRIK_OK;
}

inline bool attn_dim(int D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }

inline int attn(Why& w, const char* who, const brik_kv_cache* c, const brik_kv_batch* b, brik_attn_args& a)
{
    if (!attn_dim(c->head_dim)) return no(w, BRIK_EINVAL, "%s: head_dim %d (64, 96, 128, 192 or 256)", who, c->head_dim);
    if (a.heads < 1 || a.heads > 65535 || a.heads % c->heads)
        return no(w, BRIK_EINVAL, "%s: %d query heads over %d key / value heads", who, a.heads, c->heads);
    if (a.window < 0) return no(w, BRIK_EINVAL, "%s: window %d", who, a.window);
    if (!std::isfinite(a.scale) || !(a.softcap >= 0) || !std::isfinite(a.softcap))
        return no(w, BRIK_EINVAL, "%s: scale %g, softcap %g", who, (double)a.scale, (double)a.softcap);
    const int64_t width = (int64_t)a.heads * c->head_dim;
    BRIK_CHECK(stride(w, who, "q", a.q_stride, width));
    BRIK_CHECK(stride(w, who, "out", a.out_stride, width));
    if (b->rows == 0) return BRIK_OK;
    if ((long long)b->rows * a.heads >= (1ll << 27))
        return no(w, BRIK_EINVAL, "%s: %d rows of %d heads exceed 2^27 in one call", who, b->rows, a.heads);
    if (!a.q || !a.out) return no(w, BRIK_EINVAL, "%s: q or out is null", who);
    if (off(a.q, 16) || off(a.out, 16)) return no(w, BRIK_EALIGN, "%s: q and out must be 16-byte aligned", who);
    if (overlap(a.q, a.q_stride, width, a.out, a.out_stride, width, b->rows)) return no(w, BRIK_EINVAL, "%s: out overlaps q", who);
    return BRIK_OK;
}

// The step of a checked batch (and cache, where there is one).
inline brik_step step(const brik_kv_batch& b, const brik_kv_cache* c)
{
    brik_step s{};
    s.row_off = b.row_off;
    s.kv_len = b.kv_len;
    s.table = b.table;
    s.prefix_table = b.prefix_table;
    s.seqs = b.seqs;
    s.rows = b.rows;
    s.table_cols = b.table_cols;
    s.max_len = b.max_len;
    s.prefix_len = b.prefix_len;
    s.per_seq = b.row_off || b.seqs == 0 ? 0 : b.rows / b.seqs;
    s.pages = c ? c->pages : 0;
    s.shift = c ? brik_log2(c->page) : 0;
    return s;
}

}  // namespace brik_check
