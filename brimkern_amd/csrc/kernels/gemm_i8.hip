// y[M, N] = x[M, K] . w[N, K]^T of 8-bit integers, a scale for every row of each, dense or by experts.
//
//   y_mn = (sum_k x_mk w_nk) ws_n xs_m (+ res_mn), the sum exact in int32
//
// Integer sums have no order and every rounding after them is one of its own, so K may be split over waves and blocks freely: results are
// the same bits, whichever kernel computes them. Two kernels:
//   few rows (decoding, experts of few tokens): bound by the bytes of w and by latency. A block has 16 channels; its 4 to 16 waves split
//     K, and a wave loads all of its part of w at once, into registers, and multiplies it with 16 or 32 rows of x after the other. 1 row of
//     2560 x 9728 7.7 us (3.2 TB/s, a launch among them), of 9728 x 2560 8.9; 24 rows of 4096 x 2561 7.6.
//   tiles (prompts): bound by the matrix cores. Both operands go through LDS, 128 of K a step, double-buffered, the loads of the next
//     step (256 x 256) or of the next two in registers meanwhile. 8192^3 492 us, 2.2 POP/s (the card's library 2.1; the clock falls
//     under this load); 8192 x 9728 x 2560 218 (library 202); 512 x 2560 x 9728 21 to 22 with w in the last-level cache, 26 from memory (library
//     38), where loads through the vector-memory path, some 22 clocks a KiB, take as long as the products, so tiles of 256 x 128, which load least,
//     are fastest. By experts, 64 of them, 8 a token: 256 tokens by 2048 x 1536 51 (201 MB of w, 4.2 TB/s), 4096 by 768 x 2048 145 (268 MB of y,
//     2.7 TB/s in all: a tile has 6 steps between its loads' start and its stores), 8192 by 2048 x 1536 318 (1.3 POP/s: the experts' last tiles are
//     part filled, and brik_i8_moe_256x256 has two registers more than there are, so its loop reads 12 bytes a lane from scratch).
#include "attn_common.h"
#include "moe_abi.h"

namespace {

typedef int i32x16_t __attribute__((ext_vector_type(16)));
struct Yes {
    static constexpr bool value = true;
};
struct No {
    static constexpr bool value = false;
};

// Orders LDS accesses of the block; global loads stay in flight.
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A product and what is added to it, a rounding of its own whatever kernel computes it (elsewhere the build lets products and sums fuse).
__device__ __forceinline__ float plus(float y, float res)
{
#pragma clang fp contract(off)
    return y + res;
}

// What a block multiplies: rows [m0, m1) of y, and the weight of their expert.
struct I8Rows {
    int m0, m1;
    const int8_t* w;
    const float* ws;
};

// Row tile `tile` of BM rows of the experts' rows, in order of the experts. Every wave reads all offsets, 64 at a time. False: there
// is no such tile. Offsets that decrease are empty experts, rows past M are cut off.
__device__ __forceinline__ bool expert_tile(const brik_i8_launch& a, int tile, int BM, I8Rows& r)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.E; base += 64) {
        const int e = base + lane;
        int first = 0, end = 0;
        if (e < a.E) {
            first = max(a.row_off[e], 0);
            end = min(a.row_off[e + 1], a.M);
        }
        const int tiles = end > first ? (end - first + BM - 1) / BM : 0;
        const int sum = wave_scan(tiles);
        const uint64_t past = __ballot(before + sum > tile);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            const int j = tile - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
            const int e1 = uniform(base + l);
            r.m0 = uniform(__builtin_amdgcn_readlane(first, l) + j * BM);
            r.m1 = uniform(min(__builtin_amdgcn_readlane(end, l), r.m0 + BM));
            r.w = a.w + (size_t)e1 * a.N * a.K;
            r.ws = a.ws + (size_t)e1 * a.N;
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// The row of x that row m of y is made of; -1: none.
__device__ __forceinline__ int x_row(const brik_i8_launch& a, int m)
{
    if (!a.src) return m;
    const int v = a.src[m];
    const int row = v >= 0 ? v / a.k : -1;
    return row < a.x_rows ? row : -1;
}

// ---- few rows ------------------------------------------------------------------------------------

constexpr int FEW_S = 8;         // 64-byte steps of K that a wave holds at once

// MB: 16 rows each at a time, by NW waves.
template <int MB, int NW>
__device__ __forceinline__ void i8_few(const brik_i8_launch& a)
{
    constexpr int C = 16, R = 16 * MB, LD = C + 1;
    __shared__ int red[R * LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), i16 = lane & 15, q = lane >> 4;
    int id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int ct = id % a.col_tiles, e = id / a.col_tiles;
    I8Rows r{0, a.M, a.w, a.ws};
    if (a.E) {
        r.m0 = max(a.row_off[e], 0);
        r.m1 = min(a.row_off[e + 1], a.M);
        if (r.m0 >= r.m1) return;
        r.w += (size_t)e * a.N * a.K;
        r.ws += (size_t)e * a.N;
    }
    const int n0 = ct * C, K = a.K;
    const int steps = (K + 63) >> 6, s0 = split * a.steps, s1 = min(steps, s0 + a.steps);
    const int pieces = (s1 - s0 + NW * FEW_S - 1) / (NW * FEW_S), per = (s1 - s0 + NW * pieces - 1) / (NW * pieces);
    const int8_t* const wr = r.w + (size_t)min(n0 + i16, a.N - 1) * K;
    i32x4_t w[FEW_S];
    for (int m = r.m0; m < r.m1; m += R) {
        const int8_t* xr[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const int mine = m + 16 * b + i16, row = mine < r.m1 ? x_row(a, mine) : -1;
            xr[b] = row < 0 ? nullptr : a.x + (size_t)row * K;
        }
        i32x4_t acc[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[b] = i32x4_t{0, 0, 0, 0};
        for (int p = 0; p < pieces; ++p) {
            const int first = s0 + (p * NW + wave) * per, count = min(per, s1 - first);
            if (pieces > 1 || m == r.m0) {
#pragma unroll
                for (int s = 0; s < FEW_S; ++s)
                    if (s < count) w[s] = *(const i32x4_t*)(wr + min(64 * (first + s) + 16 * q, K - 16));
            }
#pragma unroll
            for (int s = 0; s < FEW_S; ++s)
                if (s < count) {
                    const int k = 64 * (first + s) + 16 * q;
                    i32x4_t x[MB];
#pragma unroll
                    for (int b = 0; b < MB; ++b) {
                        x[b] = i32x4_t{0, 0, 0, 0};
                        if (xr[b] && k < K) x[b] = *(const i32x4_t*)(xr[b] + k);
                    }
#pragma unroll
                    for (int b = 0; b < MB; ++b) acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s], x[b], acc[b], 0, 0, 0);
                }
        }
        for (int i = tid; i < R * LD; i += 64 * NW) red[i] = 0;
        __syncthreads();
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int v = 0; v < 4; ++v) atomicAdd(&red[(16 * b + i16) * LD + 4 * q + v], acc[b][v]);
        __syncthreads();
        for (int i = tid; i < R * C; i += 64 * NW) {
            const int t = i / C, c = i - t * C, row = m + t, n = n0 + c;
            if (row >= r.m1 || n >= a.N) continue;
            const int sum = red[t * LD + c];
            const size_t at = (size_t)row * a.N + n;
            if (a.part) {
                a.part[(size_t)split * a.M * a.N + at] = sum;
                continue;
            }
            const int from = x_row(a, row);
            if (from < 0) continue;
            const float y = (float)sum * r.ws[n] * a.xs[from];
            a.y[at] = a.res ? plus(y, a.res[at]) : y;
        }
        __syncthreads();
    }
}

// ---- tiles -----------------------------------------------------------------------------------------

// WR x WC waves, each WA x WB blocks of 32 x 32; BK of K a step, double-buffered.
template <int WR_, int WC_, int WA_, int WB_, int AHEAD_, int FD_>
struct I8Tile {
    static constexpr int WR = WR_, WC = WC_, WA = WA_, WB = WB_, BK = 128, AHEAD = AHEAD_, FD = FD_;
    static constexpr int NT = 64 * WR * WC, BM = 32 * WR * WA, BN = 32 * WC * WB;
    static constexpr int CH = BK / 16, ROWS = NT / CH;           // 16-byte chunks of a row, rows that the block loads at once
    static constexpr int CX = BM / ROWS, CW = BN / ROWS;         // chunks of a thread and step
    static constexpr int BUF = (BM + BN) * BK, H = BK / 32;
    static_assert(BM % ROWS == 0 && BN % ROWS == 0 && ROWS % 32 == 0, "whole chunks");
    // Chunk c of row r lies at c ^ turn(r): a column of chunks is read in groups of the rows 4 a .. 4 a + 3 and 4 (a ^ 5) .. 4 (a ^ 5) + 3,
    // which then meet every bank once (no conflicts counted).
    static __device__ __forceinline__ int turn(int r) { return (r & 7) ^ ((r >> 3) & 1); }
};

// Loads past `bytes` give zeros.
__device__ __forceinline__ brsrc_t rest_of(const void* p, size_t bytes) { return make_rsrc(p, (uint32_t)min(bytes, (size_t)0xffffffffu)); }

// A row of accumulators, read out of the accumulation registers here and not before (the compiler would read all of them at the
// first use of any, and has no room for them).
template <class T>
__device__ __forceinline__ void in_vector_registers(i32x16_t (&acc)[T::WB])
{
#pragma unroll
    for (int j = 0; j < T::WB; ++j) asm volatile("" : "+v"(acc[j]));
}

// A wave's part of the tile into y: row v of register r, column block j. Offsets from the tile's first value, past any buffer for
// what is no value of y (no store waits for another, as it would behind branches). WHOLE: every value of the tile is one of y.
template <class T, bool RES, bool WHOLE>
__device__ __forceinline__ void i8_write(i32x16_t (&acc)[T::WA][T::WB], brsrc_t y, brsrc_t res, const float (&ws)[T::WB], const float* scale,
                                         const int* ok, uint32_t at0, uint32_t pitch, int left)
{
    // the values to add, 16 rows ahead of their use (res may be y, so no load passes a store by itself)
    float add[2][RES ? 8 : 1][T::WB];
    auto offset = [&](uint32_t row, bool is, int j) {
        return WHOLE || (is && 32 * j < left) ? at0 + row * pitch + 128 * j : 0xffffffffu;
    };
    auto read = [&](int part) {
#pragma unroll
        for (int v = 0; v < 8; ++v) {
            const int row = 16 * part + 8 * (v >> 2) + (v & 3);
#pragma unroll
            for (int j = 0; j < T::WB; ++j)
                add[part & 1][v][j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(res, offset(row, ok[row], j), 0, 0));
        }
    };
    if constexpr (RES) read(0);
#pragma unroll
    for (int part = 0; part < 2 * T::WA; ++part) {
        if constexpr (RES) {
            if (part + 1 < 2 * T::WA) read(part + 1);
        }
        if (part % 2 == 0) in_vector_registers<T>(acc[part / 2]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const f32x4_t xs = *(const f32x4_t*)(scale + 16 * part + 8 * q);
            const i32x4_t is = *(const i32x4_t*)(ok + 16 * part + 8 * q);
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int j = 0; j < T::WB; ++j) {
                    float val = (float)acc[part / 2][j][8 * (part & 1) + 4 * q + v] * ws[j] * xs[v];
                    if constexpr (RES) val = plus(val, add[part & 1][4 * q + v][j]);
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, val), y, offset(16 * part + 8 * q + v, is[v], j), 0, 0);
                }
        }
    }
}

// MOE: by experts, the rows of x perhaps found by src; else dense, with values to add or K split.
template <class T, bool MOE>
__device__ __forceinline__ void i8_tile(const brik_i8_launch& a)
{
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * T::BUF];
    __shared__ __attribute__((aligned(16))) float row_scale[T::BM];
    __shared__ __attribute__((aligned(16))) int row_ok[T::BM];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), wr = wave / T::WC, wc = wave % T::WC;
    // blocks of one XCD (every eighth) take neighbouring tiles, 8 row tiles by as many columns as fit
    const int tiles = a.row_tiles * a.col_tiles * a.splits, xcd = blockIdx.x & 7, each = tiles >> 3, more = tiles & 7;
    int id = xcd * each + min(xcd, more) + ((int)blockIdx.x >> 3);
    const int split = id % a.splits;
    id /= a.splits;
    const int group = 8 * a.col_tiles, g = id / group, rows = min(8, a.row_tiles - 8 * g), in = id - g * group;
    const int rt = 8 * g + in % rows, ct = in / rows;
    I8Rows r{rt * T::BM, min(a.M, (rt + 1) * T::BM), a.w, a.ws};
    if (MOE && !expert_tile(a, rt, T::BM, r)) return;
    const int n0 = ct * T::BN, K = a.K;
    const int k0 = split * a.steps * 64, k1 = min(K, k0 + a.steps * 64);

    // the scales of the tile's rows, and whether they are rows
    for (int i = tid; i < T::BM; i += T::NT) {
        const int from = r.m0 + i < r.m1 ? MOE ? x_row(a, r.m0 + i) : r.m0 + i : -1;
        row_ok[i] = from >= 0;
        row_scale[i] = from >= 0 ? a.xs[from] : 0.f;
    }
    // D layout of a 32 x 32 tile: lane holds column lane & 31, register 4 q + v row 8 q + 4 (lane >> 5) + v. The columns' scales are
    // there before the first chunk is.
    const int lrow = lane & 31, rel = 32 * wr * T::WA + 4 * (lane >> 5), n1 = n0 + 32 * wc * T::WB + lrow;
    const size_t first = (size_t)r.m0 * a.N + n0;
    float ws[T::WB];
#pragma unroll
    for (int j = 0; j < T::WB; ++j) ws[j] = r.ws[min(n1 + 32 * j, a.N - 1)];
    // A chunk past K is zeros: its offset is past any buffer. (Rows past the tile's are other rows or zeros, and not used.)
    const int part = tid % T::CH, trow = tid / T::CH;
    uint32_t xo[T::CX], wo[T::CW];
    const brsrc_t rx = MOE && a.src ? rest_of(a.x, (size_t)a.x_rows * K) : rest_of(a.x + (size_t)r.m0 * K, (size_t)(a.M - r.m0) * K);
    const brsrc_t rw = rest_of(r.w + (size_t)n0 * K, (size_t)(a.N - n0) * K);
    int k = k0 + 16 * part;
#pragma unroll
    for (int i = 0; i < T::CX; ++i) {
        const int m = i * T::ROWS + trow;
        const int row = MOE && a.src ? max(x_row(a, min(r.m0 + m, r.m1 - 1)), 0) : m;
        xo[i] = (uint32_t)row * (uint32_t)K;
    }
#pragma unroll
    for (int i = 0; i < T::CW; ++i) wo[i] = (uint32_t)(i * T::ROWS + trow) * (uint32_t)K;

    // chunk i of the thread: of x, then of w
    constexpr int C = T::CX + T::CW;
    i32x4_t chunk[T::AHEAD][C];
    auto load = [&](int i, int set) {
        const bool of_x = i < T::CX;
        chunk[set][i] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                               of_x ? rx : rw, k < k1 ? (of_x ? xo[of_x ? i : 0] : wo[of_x ? 0 : i - T::CX]) + k : 0xffffffffu, 0, 0));
    };
    const int put = trow * T::BK + 16 * (part ^ T::turn(trow));
    // (rows of w follow those of x)
    auto store = [&](int i, int buf, int set) { *(i32x4_t*)(smem + buf * T::BUF + put + i * T::NT * 16) = chunk[set][i]; };
    const int get = lrow * T::BK + 16 * ((lane >> 5) ^ T::turn(lrow));
    const int xget = get + wr * T::WA * 32 * T::BK, wget = get + T::BM * T::BK + wc * T::WB * 32 * T::BK;
    constexpr int NF = T::FD == 1 ? 2 : 4;                       // sets of operands
    static_assert(T::H % NF == 0 && T::FD < T::H, "parts");
    i32x4_t fx[NF][T::WA], fw[NF][T::WB];
    // operand i (of w, then of x) of part h, 32 of K, of a buffer
    auto fetch = [&](int i, int buf, int h) {
        const unsigned char* const from = smem + buf * T::BUF;
        if (i < T::WB) fw[h % NF][i < T::WB ? i : 0] = *(const i32x4_t*)(from + (wget ^ (32 * h)) + i * 32 * T::BK);
        else fx[h % NF][i < T::WB ? 0 : i - T::WB] = *(const i32x4_t*)(from + (xget ^ (32 * h)) + (i - T::WB) * 32 * T::BK);
    };
    i32x16_t acc[T::WA][T::WB];
#pragma unroll
    for (int i = 0; i < T::WA; ++i)
#pragma unroll
        for (int j = 0; j < T::WB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;

#pragma unroll
    for (int i = 0; i < C; ++i) load(i, T::AHEAD - 1);
    k += T::BK;
    if constexpr (T::AHEAD == 2) {
#pragma unroll
        for (int i = 0; i < C; ++i) load(i, 0);
        k += T::BK;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
        store(i, 0, T::AHEAD - 1);
        load(i, T::AHEAD - 1);
    }
    k += T::BK;
    lds_barrier();
#pragma unroll
    for (int h = 0; h < T::FD; ++h)
#pragma unroll
        for (int i = 0; i < T::WA + T::WB; ++i) fetch(i, 0, h);
    // A step: parts of 32 of K. Between the products of a part go the next part's operands from LDS and, in the middle parts, the next
    // step's chunks into the other buffer, whose last readers are past the barrier, each followed by the load of the step after.
    // The barrier before the last part ends both: the next step's first operands come from the other buffer. The order is written
    // out and held (left to itself the compiler moves the products together and waits for every operand where it is used).
    constexpr int P = T::WA * T::WB, OPS = T::WA + T::WB, MID = T::H - T::FD, SLOTS = MID * P;
    auto step = [&](int buf, int set) {
#pragma unroll
        for (int h = 0; h < T::H; ++h) {
            const bool other = h >= MID;                         // operands of the next step from here on
            if (h == MID) {
                k += T::BK;
                lds_barrier();
            }
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const int i = p / T::WB, j = p % T::WB;
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[h % NF][i], fw[h % NF][j], acc[i][j], 0, 0, 0);
#pragma unroll
                for (int o = p * OPS / P; o < (p + 1) * OPS / P; ++o) fetch(o, other ? buf ^ 1 : buf, other ? h - MID : h + T::FD);
                if (!other) {
#pragma unroll
                    for (int o = (h * P + p) * C / SLOTS; o < (h * P + p + 1) * C / SLOTS; ++o) {
                        store(o, buf ^ 1, set);
                        load(o, set);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    int at = k0;
    if constexpr (T::AHEAD == 2) {
        for (; at + T::BK < k1; at += 2 * T::BK) {
            step(0, 0);
            step(1, 1);
        }
        if (at < k1) step(0, 0);
    } else {
        for (int buf = 0; at < k1; at += T::BK, buf ^= 1) step(buf, 0);
    }

    const uint32_t pitch = 4u * (uint32_t)a.N, at0 = (uint32_t)rel * pitch + 4u * (uint32_t)(n1 - n0);
    if (!MOE && a.part) {
        const brsrc_t to = rest_of(a.part + (size_t)split * a.M * a.N + first, 4 * ((size_t)a.M * a.N - first));
#pragma unroll
        for (int i = 0; i < T::WA; ++i) {
            in_vector_registers<T>(acc[i]);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int row = 32 * i + 8 * (v >> 2) + (v & 3);
#pragma unroll
                for (int j = 0; j < T::WB; ++j)
                    __builtin_amdgcn_raw_buffer_store_b32((uint32_t)acc[i][j][v], to,
                                                          r.m0 + rel + row < r.m1 && n1 + 32 * j < a.N ? at0 + row * pitch + 128 * j : 0xffffffffu, 0, 0);
            }
        }
        return;
    }
    const brsrc_t y = rest_of(a.y + first, 4 * ((size_t)a.M * a.N - first));
    const bool whole = !(MOE && a.src) && r.m0 + T::BM <= r.m1 && n0 + T::BN <= a.N;
    auto write = [&](auto added, brsrc_t res) {
        if (whole) i8_write<T, decltype(added)::value, true>(acc, y, res, ws, row_scale + rel, row_ok + rel, at0, pitch, a.N - n1);
        else i8_write<T, decltype(added)::value, false>(acc, y, res, ws, row_scale + rel, row_ok + rel, at0, pitch, a.N - n1);
    };
    if (!MOE && a.res) write(Yes(), rest_of(a.res + first, 4 * ((size_t)a.M * a.N - first)));
    else write(No(), y);
}

}  // namespace

#define BRIK_I8_FEW(MB, NW) \
    extern "C" __global__ __launch_bounds__(64 * NW) void brik_i8_few_##MB##_##NW(brik_i8_launch a) { i8_few<MB, NW>(a); }
BRIK_I8_FEW(1, 4)
BRIK_I8_FEW(1, 8)
BRIK_I8_FEW(2, 8)
BRIK_I8_FEW(1, 16)
BRIK_I8_FEW(2, 16)

#define BRIK_I8_TILE(NAME, WR, WC, WA, WB, AHEAD, FD, OCC)                                                    \
    extern "C" __global__ __launch_bounds__(64 * WR * WC, OCC) void brik_i8_tile_##NAME(brik_i8_launch a)     \
    {                                                                                                         \
        i8_tile<I8Tile<WR, WC, WA, WB, AHEAD, FD>, false>(a);                                                 \
    }
#define BRIK_I8_MOE(NAME, WR, WC, WA, WB, AHEAD, FD, OCC)                                                     \
    extern "C" __global__ __launch_bounds__(64 * WR * WC, OCC) void brik_i8_moe_##NAME(brik_i8_launch a)      \
    {                                                                                                         \
        i8_tile<I8Tile<WR, WC, WA, WB, AHEAD, FD>, true>(a);                                                  \
    }
BRIK_I8_TILE(256x256, 2, 2, 4, 4, 1, 1, 1)
BRIK_I8_TILE(256x128, 2, 2, 4, 2, 2, 2, 1)
BRIK_I8_TILE(128x128, 2, 2, 2, 2, 2, 2, 2)
BRIK_I8_TILE(64x128, 2, 2, 1, 2, 2, 2, 2)
BRIK_I8_MOE(256x256, 2, 2, 4, 4, 1, 1, 1)
BRIK_I8_MOE(128x128, 2, 2, 2, 2, 2, 2, 2)
BRIK_I8_MOE(64x128, 2, 2, 1, 2, 2, 2, 3)

// The splits' sums and the scaling: a thread takes one value of y at a time.
extern "C" __global__ __launch_bounds__(256) void brik_i8_join(brik_i8_launch a)
{
    const size_t all = (size_t)a.M * a.N;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        int sum = 0;
        for (int s = 0; s < a.splits; ++s) sum += a.part[s * all + i];
        const size_t m = i / a.N, n = i - m * a.N;
        const float y = (float)sum * a.ws[n] * a.xs[m];
        a.y[i] = a.res ? plus(y, a.res[i]) : y;
    }
}
