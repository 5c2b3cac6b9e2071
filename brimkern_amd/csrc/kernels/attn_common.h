// What the attention kernels share: the rows of a tile, which keys they see, the split of the keys, half pairs.
#pragma once
#include "attn_abi.h"
#include "common.h"

namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr float ATTN_LOG2E = 1.44269504088896340736f;
constexpr float ATTN_NONE = -1e30f;      // reference exponent of a row that has seen no key

// v of the lower and of the upper lane of this lane's pair (l, l ^ 32; quarter_pair: l, l ^ 16): both lanes get the same two
// values. (The elements are copied out first: a bit cast of a vector's element reads element 0.)
__device__ __forceinline__ void half_pair(float v, float& a, float& b)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t lo = r[0], hi = r[1];
    a = __builtin_bit_cast(float, lo);
    b = __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ void quarter_pair(float v, float& a, float& b)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t lo = r[0], hi = r[1];
    a = __builtin_bit_cast(float, lo);
    b = __builtin_bit_cast(float, hi);
}
// Maximum / sum over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quarters_max(float v)
{
    float a, b;
    quarter_pair(v, a, b);
    half_pair(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float quarters_sum(float v)
{
    float a, b;
    quarter_pair(v, a, b);
    half_pair(a + b, a, b);
    return a + b;
}

// Maximum over the 32 lanes of a half wave.
__device__ __forceinline__ float half_max(float v)
{
    v = BRIK_DPP_MAX(v, DPP_QUAD_1032);
    v = BRIK_DPP_MAX(v, DPP_QUAD_2301);
    v = BRIK_DPP_MAX(v, DPP_ROW_ROR4);
    v = BRIK_DPP_MAX(v, DPP_ROW_ROR8);
    float a, b;
    quarter_pair(v, a, b);
    return fmaxf(a, b);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Min / max over the 64 lanes (uniform result).
__device__ __forceinline__ int wave_min(int v)
{
    v = min(v, __builtin_amdgcn_mov_dpp(v, DPP_QUAD_1032, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_mov_dpp(v, DPP_QUAD_2301, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_mov_dpp(v, DPP_ROW_ROR4, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_mov_dpp(v, DPP_ROW_ROR8, 0xF, 0xF, false));
    const auto q = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = min((int)q[0], (int)q[1]);
    const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    return uniform(min((int)h[0], (int)h[1]));
}
__device__ __forceinline__ int wave_max(int v) { return -wave_min(-v); }

// Sum of v over the lanes up to this one: within rows of 16 by shifts, then the sums of the rows before.
__device__ __forceinline__ int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);       // row_shr 1, 2, 4, 8; zeros come in
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    const int row = (threadIdx.x & 63) >> 4;
    const int a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31), c = __builtin_amdgcn_readlane(v, 47);
    return v + (row > 0 ? a : 0) + (row > 1 ? b : 0) + (row > 2 ? c : 0);
}
__device__ __forceinline__ int wave_sum(int v)
{
    v += __builtin_amdgcn_mov_dpp(v, DPP_QUAD_1032, 0xF, 0xF, false);
    v += __builtin_amdgcn_mov_dpp(v, DPP_QUAD_2301, 0xF, 0xF, false);
    v += __builtin_amdgcn_mov_dpp(v, DPP_ROW_ROR4, 0xF, 0xF, false);
    v += __builtin_amdgcn_mov_dpp(v, DPP_ROW_ROR8, 0xF, 0xF, false);
    const auto q = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = (int)(q[0] + q[1]);
    const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    return uniform((int)(h[0] + h[1]));
}

// The sequence of row t, or seqs where the row belongs to none (behind the last sequence, or before row_off[0]): how many of
// row_off[1..seqs] are at most t, where any of row_off[0..seqs) is. One load round trip per 64 sequences.
__device__ __forceinline__ int seq_of_row(const brik_step& s, int t)
{
    if (!s.row_off) return t / s.per_seq;
    const int lane = threadIdx.x & 63;
    int count = 0;
    uint64_t begun = 0;
    for (int base = 0; base < s.seqs; base += 64) {
        const int i = base + lane;
        const int32_t first = i < s.seqs ? s.row_off[i] : 0x7fffffff, end = i < s.seqs ? s.row_off[i + 1] : 0x7fffffff;
        begun |= __ballot(first <= t);
        count += __popcll(__ballot(end <= t));
    }
    return begun ? count : s.seqs;
}

// For a row per lane, whose rows are t0 + (0 .. count - 1) over the wave: the last sequence that begins at most at the row, or -1.
// Every candidate row is compared with 64 sequences at a time, so no lane follows a chain of dependent loads.
__device__ __forceinline__ int seq_of_lane(const brik_step& s, int t, int t0, int count)
{
    if (!s.row_off) return t / s.per_seq;
    const int lane = threadIdx.x & 63;
    int mine = -1;
    for (int base = 0; base < s.seqs; base += 64) {
        const int i = base + lane;
        const int32_t first = i < s.seqs ? s.row_off[i] : 0x7fffffff;
        for (int k = 0; k < count; ++k) {
            const int c = __popcll(__ballot(first <= t0 + k));
            if (t == t0 + k) mine += c;
        }
    }
    return mine;
}

// The position of row t of sequence b.
__device__ __forceinline__ int32_t row_position(const brik_step& s, int b, int t)
{
    const int32_t end = s.row_off ? s.row_off[b + 1] : (b + 1) * s.per_seq;
    return s.kv_len[b] - end + t;
}

// Tile `tile` of the sequences' row tiles (BM rows of rows * G each), in order: its sequence and its place in it.
// b == seqs: there is no such tile.
__device__ __forceinline__ void find_tile(const brik_step& s, int tile, int G, int BM, int& b, int& j)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < s.seqs; base += 64) {
        const int i = base + lane;
        int32_t first, n = 0;
        if (i < s.seqs) brik_rows_of(s, i, first, n);
        const int tiles = (int)(((long long)n * G + BM - 1) / BM);
        const int sum = wave_scan(tiles);
        const uint64_t past = __ballot(before + sum > tile);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            b = uniform(base + l);
            j = uniform(tile - before - (__shfl(sum, l) - __shfl(tiles, l)));
            return;
        }
        before += __shfl(sum, 63);
    }
    b = s.seqs;
    j = 0;
}

// One block's work: which rows, which keys.
struct Work {
    int head;                  // key / value head
    int slot;                  // of the partial results, or block of the sequences' blocks
    bool prefix;               // keys of the prefix, rows of all sequences
    int b;                     // sequence (own keys)
    int first, count;          // its rows
    int r0;                    // first of the tile's rows, counted over count * G
    int split, splits;
    int t0, t1;                // blocks of 32 keys, where they are shared out (else t1 == 0: by split and splits)
    int pos;                   // position of the first row (own keys)
    bool whole;                // nothing to join: the block writes the output
};

// The first key that the window of a row at `pos` shows, counted from token `first` on. (In 64 bits: a window of 2^31 - 1 and a
// position before `first` leave 32.)
__device__ __forceinline__ int first_seen(const brik_attn_launch& a, int32_t pos, int32_t first)
{
    return a.a.window ? (int)max(0ll, (long long)pos - a.a.window + 1 - first) : 0;
}

// A sequence's rows, and the blocks of 32 of its own keys that they see (first, count).
struct Seq {
    int32_t row, rows, pos;      // first row, how many, the first row's position
    int first, n;
};
__device__ __forceinline__ Seq find_seq(const brik_attn_launch& a, int b)
{
    Seq q;
    brik_rows_of(a.s, b, q.row, q.rows);
    const int32_t end_row = a.s.row_off ? a.s.row_off[b + 1] : (b + 1) * a.s.per_seq;
    q.pos = a.s.kv_len[b] - end_row + q.row;
    const int32_t before = a.s.prefix_len;
    const int32_t end = (int32_t)min((long long)a.s.max_len - before, min((long long)a.s.table_cols << a.s.shift, 0x7fffffc0ll));
    const int hi = min(q.pos + q.rows - before, end), lo = first_seen(a, q.pos, before);
    q.first = lo >> 5;
    q.n = q.rows > 0 && lo < hi ? ((hi + 31) >> 5) - q.first : 0;
    return q;
}

// The own keys of all sequences in a row, in blocks of 32, are shared out evenly: `each` blocks of keys for every block of the
// grid (four at least, one per wave), which may end one sequence and begin the next. Its part of sequence b is number
// block + b of the partial results: a sequence's parts follow each other, and no two parts share a number. Every wave reads
// all lengths, 64 at a time, one a lane.
struct Share {
    int each, total;
    __device__ __forceinline__ explicit Share(const brik_attn_launch& a)
    {
        total = 0;
        for (int base = 0; base < a.s.seqs; base += 64) total += wave_sum(lane_seq(a, base).n);
        each = max(4, (total + a.own_blocks - 1) / a.own_blocks);
    }
    __device__ __forceinline__ static Seq lane_seq(const brik_attn_launch& a, int base)
    {
        Seq q;
        q.n = q.rows = q.row = q.pos = q.first = 0;
        const int b = base + (int)(threadIdx.x & 63);
        if (b < a.s.seqs) q = find_seq(a, b);
        return q;
    }
    // Sequence b, all of it uniform, and the key blocks before it. b < 0: of the sequence that key block g < total belongs to.
    __device__ __forceinline__ static Seq find(const brik_attn_launch& a, int& b, int g, int& start)
    {
        int before = 0;
        for (int base = 0;; base += 64) {
            const Seq q = lane_seq(a, base);
            const int sum = wave_scan(q.n);
            int l = b - base;
            if (b < 0) {
                const uint64_t past = __ballot(before + sum > g);
                l = past ? __ffsll((unsigned long long)past) - 1 : 64;
            }
            if (l < 64) {
                b = base + l;
                Seq r;
                r.row = __builtin_amdgcn_readlane(q.row, l);
                r.rows = __builtin_amdgcn_readlane(q.rows, l);
                r.pos = __builtin_amdgcn_readlane(q.pos, l);
                r.first = __builtin_amdgcn_readlane(q.first, l);
                r.n = __builtin_amdgcn_readlane(q.n, l);
                start = before + __builtin_amdgcn_readlane(sum, l) - r.n;
                return r;
            }
            before += __builtin_amdgcn_readlane(sum, 63);
        }
    }
};

// The grid: heads fastest, then the splits, then the row tiles; the prefix's blocks before the own keys'.
template <int BM>
__device__ __forceinline__ bool find_work(const brik_attn_launch& a, Work& w)
{
    const int KV = a.c.heads, G = a.a.heads / KV;
    int id = a.first_block + blockIdx.x;
    w.head = id % KV;
    id /= KV;
    const int pre = a.prefix_tiles * a.prefix_splits;
    w.t0 = w.t1 = 0;
    w.whole = a.whole;
    w.prefix = id < pre;
    if (w.prefix) {
        w.splits = a.prefix_splits;
        w.split = id % w.splits;
        w.slot = w.split;
        w.b = 0;
        w.first = 0;
        w.count = a.s.rows;
        w.r0 = id / w.splits * BM;
        return true;
    }
    id -= pre;
    w.splits = a.own_splits;
    w.split = id % w.splits;
    w.slot = a.prefix_splits + w.split;
    int tile = id / w.splits, j;
    if (a.tiles_per_seq) {
        w.b = tile / a.tiles_per_seq;
        j = tile - w.b * a.tiles_per_seq;
    } else {
        find_tile(a.s, tile, G, BM, w.b, j);
        if (w.b >= a.s.seqs) return false;
    }
    brik_rows_of(a.s, w.b, w.first, w.count);
    w.pos = row_position(a.s, w.b, w.first);
    // the last tiles see the most keys: they come first. Of a sequence with more rows than the call was said to have, the first
    // ones are done.
    int tiles = (int)(((long long)w.count * G + BM - 1) / BM);
    if (a.tiles_per_seq) tiles = min(tiles, a.tiles_per_seq);
    if (j >= tiles) return false;
    w.r0 = (tiles - 1 - j) * BM;
    return true;
}

// The parts of a block of the shared-out keys: w is set to the part that begins at key block g (of all sequences' in a row), g
// to the end of that part.
__device__ __forceinline__ void next_part(const brik_attn_launch& a, int each, int block, int end, int& g, Work& w)
{
    int start;
    w.b = -1;
    const Seq q = Share::find(a, w.b, g, start);
    w.first = q.row;
    w.count = q.rows;
    w.pos = q.pos;
    w.r0 = 0;
    w.slot = block + w.b;
    w.t0 = q.first + (g - start);
    g = min(end, start + q.n);
    w.t1 = q.first + (g - start);
    w.whole = a.prefix_splits == 0 && start / each == (start + q.n - 1) / each;
}

// A row of a tile (this lane's): its token and head, and the keys it sees, [lo, hi) in the section's own numbering
// (prefix tokens, or own tokens behind the prefix). A row past the tile's end sees everything and is not stored.
struct Row {
    int t, h;
    bool real;
    int lo, hi;
};

// Row m of the ROWS rows from r0 on, counted over count * G.
template <int ROWS>
__device__ __forceinline__ Row find_row(const brik_attn_launch& a, const Work& w, int r0, int m)
{
    const int G = a.a.heads / a.c.heads;
    Row r;
    const int i = r0 + m, rel = i / G;
    r.real = rel < w.count;
    r.t = w.first + rel;
    r.h = w.head * G + i - rel * G;
    r.lo = 0;
    r.hi = 0x7fffffff;
    int32_t pos = w.pos + rel;
    if (w.prefix) {
        const int t0 = uniform(r0 / G), last = min((r0 + ROWS - 1) / G, a.s.rows - 1), b = seq_of_lane(a.s, r.t, t0, uniform(last) - t0 + 1);
        if (!r.real || b < 0) {
            r.real = false;
            return r;
        }
        const int32_t end = a.s.row_off ? a.s.row_off[b + 1] : (b + 1) * a.s.per_seq;
        pos = a.s.kv_len[b] - end + r.t;
        r.real = r.t < end;                                  // else behind the last sequence
    }
    if (!r.real) return r;
    const int32_t first = w.prefix ? 0 : a.s.prefix_len;
    const int32_t end = w.prefix ? min(a.s.prefix_len, a.s.max_len)
                                 : (int32_t)min((long long)a.s.max_len - first, min((long long)a.s.table_cols << a.s.shift, 0x7fffffc0ll));
    r.hi = max(0, min(pos + 1 - first, end));
    r.lo = first_seen(a, pos, first);
    return r;
}

// Where row m of the tile (token t, head h) keeps its partial result.
__device__ __forceinline__ size_t part_at(const brik_attn_launch& a, const Work& w, int m, int t, int h)
{
    const size_t all = (size_t)a.s.rows * a.a.heads;
    if (a.own_blocks && !w.prefix) return a.prefix_splits * all + ((size_t)w.head * (a.own_blocks + a.s.seqs) + w.slot) * 16 + m;
    return w.slot * all + (size_t)t * a.a.heads + h;
}

// The key blocks [t0, t1) of 32 keys that this split works on: those of the keys [lo, hi) that any row sees, divided over
// the splits in whole multiples of `least`.
__device__ __forceinline__ void find_keys(const Work& w, int lo, int hi, int least, int& t0, int& t1)
{
    t0 = w.t0;
    t1 = w.t1;
    if (t1 || lo >= hi) return;
    const int first = lo >> 5, n = ((hi + 31) >> 5) - first;
    const int each = (n + least * w.splits - 1) / (least * w.splits) * least;
    t0 = first + min(n, w.split * each);
    t1 = first + min(n, (w.split + 1) * each);
}

// The pages of keys 32 t .. 32 t + 31: of the first and of the last 16 (the same page unless a page holds 16 tokens), -1
// where they do not exist.
struct KeyPages {
    int32_t p[2];
};

// A window of 64 columns of the section's table, one a lane: looking a page up reads a register. (Loaded one by one, every
// look-up waited for all the loads before it, the keys of the next block among them.)
struct PageWindow {
    const int32_t* tab;
    int cols, pages, shift, base;
    int32_t id;                // of column base + lane

    __device__ __forceinline__ PageWindow(const brik_attn_launch& a, const Work& w)
    {
        tab = w.prefix ? a.s.prefix_table : a.s.table + (size_t)w.b * a.s.table_cols;
        cols = w.prefix ? (a.s.prefix_len + (1 << a.s.shift) - 1) >> a.s.shift : a.s.table_cols;
        pages = a.s.pages;
        shift = a.s.shift;
        base = -64;
        id = -1;
    }
    __device__ __forceinline__ int32_t page(int c)
    {
        if ((uint32_t)(c - base) >= 64u) {
            base = c;
            const int mine = c + (int)(threadIdx.x & 63);
            const int32_t v = mine < cols ? tab[mine] : -1;
            id = (uint32_t)v < (uint32_t)pages ? v : -1;
        }
        return __builtin_amdgcn_readlane(id, c - base);
    }
    __device__ __forceinline__ KeyPages of(int t)
    {
        KeyPages k;
        k.p[0] = page((32 * t) >> shift);
        k.p[1] = shift > 4 ? k.p[0] : page(2 * t + 1);
        return k;
    }
};

// Eight int8 codes as f16, the bytes of each word in the order 0, 2, 1, 3: 1024 + (c + 128) has the code's bits in its low
// byte, and the subtraction is exact.
__device__ __forceinline__ half8_t halves_q8(uint32_t w0, uint32_t w1)
{
    const half2_t off = {(_Float16)-1152.f, (_Float16)-1152.f};
    half8_t r;
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    const uint32_t u[4] = {__builtin_amdgcn_perm(0x64646464u, w0, 0x04020400u), __builtin_amdgcn_perm(0x64646464u, w0, 0x04030401u),
                           __builtin_amdgcn_perm(0x64646464u, w1, 0x04020400u), __builtin_amdgcn_perm(0x64646464u, w1, 0x04030401u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2_t h = __builtin_bit_cast(half2_t, u[i]) + off;
        r[2 * i] = h.x;
        r[2 * i + 1] = h.y;
    }
    return r;
}

// Codes in the low nibbles of each 16 bits as f16 less 8. The products of values have to be of both signs: the matrix
// cores' sums cut the bits that do not fit, and over sums of nearly equal terms that shows (32 sequences of up to 8192: 2.6e-6 of the
// output's norm with codes from 0, 3.9e-7 so).
__device__ __forceinline__ half8_t centred_q4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    const half2_t off = {(_Float16)-1032.f, (_Float16)-1032.f};
    const uint32_t u[4] = {a, b, c, d};
    // in a vector register, so that the mask and the bits of 1024 go into one instruction (two constants do not)
    uint32_t thousand = 0x64006400u;
    asm("" : "+v"(thousand));
    half8_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2_t h = __builtin_bit_cast(half2_t, (u[i] & 0x000f000fu) | thousand) + off;
        r[2 * i] = h.x;
        r[2 * i + 1] = h.y;
    }
    return r;
}

// Both values as halves, to nearest (one instruction).
__device__ __forceinline__ half2_t halves(float a, float b)
{
    const f32x2_t v = {a, b};
    return __builtin_convertvector(v, half2_t);
}

// v less half I of h, exact (one mixed-precision instruction; the compiler would convert and subtract).
template <int I>
__device__ __forceinline__ float residual(half2_t h, float v)
{
    float r;
    if constexpr (I == 0) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v));
    return r;
}

// tanh in f32: the exponential, and near 0, where that cancels, the odd series (next term below 2^-26 of the value).
__device__ __forceinline__ float attn_tanh(float u)
{
    const float z = u * u;
    const float s = u * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    const float e = __builtin_amdgcn_exp2f(u * (2.f * ATTN_LOG2E));
    const float t = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
    return fabsf(u) < 0.25f ? s : t;
}

}  // namespace
