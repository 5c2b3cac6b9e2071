// y[M, N] = x[M, K] . w[N, K]^T of 8-bit integers, a scale for every row of each, dense or by experts.
//
//   y_mn = (sum_k x_mk w_nk) ws_n xs_m (+ res_mn), the sum exact in int32
//
// Integer sums have no order, so K may be split over waves and blocks freely: results are the same bits. Two kernels:
//   few rows (decoding, experts of few tokens): bound by the bytes of w. A block has 16 or 32 channels; its waves split K, and a
//     wave loads all of its part of w at once, into registers, and multiplies it with 16 rows of x after the other.
//   tiles (prompts): bound by the matrix cores. Both operands go through LDS, 64 of K a step, double-buffered, the next step's
//     loads in registers meanwhile.
#include "attn_common.h"
#include "moe_abi.h"

namespace {

typedef int i32x16_t __attribute__((ext_vector_type(16)));

// Orders LDS accesses of the block; global loads stay in flight.
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
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
            r.m0 = __builtin_amdgcn_readlane(first, l) + j * BM;
            r.m1 = min(__builtin_amdgcn_readlane(end, l), r.m0 + BM);
            r.w = a.w + (size_t)(base + l) * a.N * a.K;
            r.ws = a.ws + (size_t)(base + l) * a.N;
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

// MB: 16 rows each at a time, CB: 16 channels each, NW waves.
template <int MB, int CB, int NW>
__device__ __forceinline__ void i8_few(const brik_i8_launch& a)
{
    constexpr int C = 16 * CB, R = 16 * MB, LD = C + 1;
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
    const int per = min(FEW_S, (s1 - s0 + NW - 1) / NW), pieces = (s1 - s0 + NW * per - 1) / (NW * per);
    const int8_t* wr[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) wr[c] = r.w + (size_t)min(n0 + 16 * c + i16, a.N - 1) * K;
    i32x4_t w[CB][FEW_S];
    for (int m = r.m0; m < r.m1; m += R) {
        const int8_t* xr[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const int mine = m + 16 * b + i16, row = mine < r.m1 ? x_row(a, mine) : -1;
            xr[b] = row < 0 ? nullptr : a.x + (size_t)row * K;
        }
        i32x4_t acc[MB][CB];
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int c = 0; c < CB; ++c) acc[b][c] = i32x4_t{0, 0, 0, 0};
        for (int p = 0; p < pieces; ++p) {
            const int first = s0 + (p * NW + wave) * per, count = min(per, s1 - first);
            if (pieces > 1 || m == r.m0) {
#pragma unroll
                for (int s = 0; s < FEW_S; ++s)
                    if (s < count) {
                        const int k = min(64 * (first + s) + 16 * q, K - 16);
#pragma unroll
                        for (int c = 0; c < CB; ++c) w[c][s] = *(const i32x4_t*)(wr[c] + k);
                    }
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
                    for (int b = 0; b < MB; ++b)
#pragma unroll
                        for (int c = 0; c < CB; ++c) acc[b][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[c][s], x[b], acc[b][c], 0, 0, 0);
                }
        }
        for (int i = tid; i < R * LD; i += 64 * NW) red[i] = 0;
        __syncthreads();
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int c = 0; c < CB; ++c)
#pragma unroll
                for (int v = 0; v < 4; ++v) atomicAdd(&red[(16 * b + i16) * LD + 16 * c + 4 * q + v], acc[b][c][v]);
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
            a.y[at] = a.res ? y + a.res[at] : y;
        }
        __syncthreads();
    }
}

// ---- tiles -----------------------------------------------------------------------------------------

// WR x WC waves, each WA x WB blocks of 32 x 32.
template <int WR_, int WC_, int WA_, int WB_>
struct I8Tile {
    static constexpr int WR = WR_, WC = WC_, WA = WA_, WB = WB_;
    static constexpr int NT = 64 * WR * WC, BM = 32 * WR * WA, BN = 32 * WC * WB;
    static constexpr int CX = BM * 4 / NT, CW = BN * 4 / NT;     // 16-byte chunks of a thread and step
    static constexpr int BUF = (BM + BN) * 64;
    static_assert(BM * 4 % NT == 0 && BN * 4 % NT == 0, "whole chunks");
};

// Chunk c of row r lies at c ^ turn(r): 8 rows of a column of chunks meet every bank of 128 bytes once, 16 rows of 256 bytes.
__device__ __forceinline__ int turn(int r) { return ((r >> 1) ^ (r >> 3)) & 3; }

template <class T>
__device__ __forceinline__ void i8_tile(const brik_i8_launch& a)
{
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * T::BUF];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), wr = wave / T::WC, wc = wave % T::WC;
    // blocks of one XCD (every eighth) take neighbouring tiles, 8 row tiles by as many columns as fit
    const int tiles = a.row_tiles * a.col_tiles * a.splits, xcd = blockIdx.x & 7, each = tiles >> 3, more = tiles & 7;
    int id = xcd * each + min(xcd, more) + ((int)blockIdx.x >> 3);
    const int split = id % a.splits;
    id /= a.splits;
    const int group = 8 * a.col_tiles, g = id / group, rows = min(8, a.row_tiles - 8 * g), in = id - g * group;
    const int rt = 8 * g + in % rows, ct = in / rows;
    I8Rows r{rt * T::BM, min(a.M, (rt + 1) * T::BM), a.w, a.ws};
    if (a.E && !expert_tile(a, rt, T::BM, r)) return;
    const int n0 = ct * T::BN, K = a.K;
    const int steps = (K + 63) >> 6, s0 = split * a.steps, s1 = min(steps, s0 + a.steps);

    const int part = tid & 3, trow = tid >> 2;
    const int8_t *xp[T::CX], *wp[T::CW];
#pragma unroll
    for (int i = 0; i < T::CX; ++i) {
        const int row = x_row(a, min(r.m0 + i * (T::NT / 4) + trow, r.m1 - 1));
        xp[i] = a.x + (size_t)max(row, 0) * K + 16 * part;
    }
#pragma unroll
    for (int i = 0; i < T::CW; ++i) wp[i] = r.w + (size_t)min(n0 + i * (T::NT / 4) + trow, a.N - 1) * K + 16 * part;

    i32x4_t gx[T::CX], gw[T::CW];
    auto load = [&](int s) {
        const int k = 64 * s;
        if (k + 64 <= K) {
#pragma unroll
            for (int i = 0; i < T::CX; ++i) gx[i] = *(const i32x4_t*)(xp[i] + k);
#pragma unroll
            for (int i = 0; i < T::CW; ++i) gw[i] = *(const i32x4_t*)(wp[i] + k);
        } else {
            // half a step: zeros of x behind the row's end (of w whatever lies there in the row)
            const bool inside = part < 2;
            const int at = inside ? k : k - 32;
#pragma unroll
            for (int i = 0; i < T::CX; ++i) {
                const i32x4_t v = *(const i32x4_t*)(xp[i] + at);
                gx[i] = inside ? v : i32x4_t{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < T::CW; ++i) gw[i] = *(const i32x4_t*)(wp[i] + at);
        }
    };
    const int put = trow * 64 + 16 * (part ^ turn(trow));
    auto store = [&](int buf) {
        unsigned char* const to = smem + buf * T::BUF + put;
#pragma unroll
        for (int i = 0; i < T::CX; ++i) *(i32x4_t*)(to + i * T::NT * 16) = gx[i];
#pragma unroll
        for (int i = 0; i < T::CW; ++i) *(i32x4_t*)(to + T::BM * 64 + i * T::NT * 16) = gw[i];
    };
    const int lrow = lane & 31, get = lrow * 64 + 16 * ((lane >> 5) ^ turn(lrow));
    const int xget = get + wr * T::WA * 2048, wget = get + T::BM * 64 + wc * T::WB * 2048;
    i32x4_t fx[2][T::WA], fw[2][T::WB];
    auto fetch = [&](int buf, int h) {
        const unsigned char* const from = smem + buf * T::BUF;
#pragma unroll
        for (int i = 0; i < T::WA; ++i) fx[h][i] = *(const i32x4_t*)(from + (xget ^ (32 * h)) + i * 2048);
#pragma unroll
        for (int j = 0; j < T::WB; ++j) fw[h][j] = *(const i32x4_t*)(from + (wget ^ (32 * h)) + j * 2048);
    };
    i32x16_t acc[T::WA][T::WB];
#pragma unroll
    for (int i = 0; i < T::WA; ++i)
#pragma unroll
        for (int j = 0; j < T::WB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
    auto multiply = [&](int h) {
#pragma unroll
        for (int i = 0; i < T::WA; ++i)
#pragma unroll
            for (int j = 0; j < T::WB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[h][i], fw[h][j], acc[i][j], 0, 0, 0);
    };

    if (s0 < s1) {
        load(s0);
        store(0);
        if (s0 + 1 < s1) load(s0 + 1);
        lds_barrier();
        fetch(0, 0);
        for (int s = s0; s < s1; ++s) {
            const int buf = (s - s0) & 1;
            fetch(buf, 1);
            multiply(0);
            // (the other buffer's last reads were waited for before the last barrier)
            if (s + 1 < s1) store(buf ^ 1);
            if (s + 2 < s1) load(s + 2);
            lds_barrier();
            if (s + 1 < s1) fetch(buf ^ 1, 0);
            multiply(1);
        }
    }

    const int h = lane >> 5;
#pragma unroll
    for (int i = 0; i < T::WA; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int m = r.m0 + 32 * (wr * T::WA + i) + 8 * (v >> 2) + 4 * h + (v & 3);
            if (m >= r.m1) continue;
            const int from = x_row(a, m);
            const float xs = from < 0 || a.part ? 0.f : a.xs[from];
#pragma unroll
            for (int j = 0; j < T::WB; ++j) {
                const int n = n0 + 32 * (wc * T::WB + j) + lrow;
                if (n >= a.N) continue;
                const size_t at = (size_t)m * a.N + n;
                if (a.part) {
                    a.part[(size_t)split * a.M * a.N + at] = acc[i][j][v];
                } else if (from >= 0) {
                    const float y = (float)acc[i][j][v] * r.ws[n] * xs;
                    a.y[at] = a.res ? y + a.res[at] : y;
                }
            }
        }
}

}  // namespace

#define BRIK_I8_FEW(MB, CB, NW) \
    extern "C" __global__ __launch_bounds__(64 * NW) void brik_i8_few_##MB##_##CB##_##NW(brik_i8_launch a) { i8_few<MB, CB, NW>(a); }
BRIK_I8_FEW(1, 1, 8)
BRIK_I8_FEW(2, 1, 8)
BRIK_I8_FEW(4, 1, 8)
BRIK_I8_FEW(1, 2, 8)
BRIK_I8_FEW(2, 2, 8)
BRIK_I8_FEW(4, 2, 8)

#define BRIK_I8_TILE(WR, WC, WA, WB, OCC) \
    extern "C" __global__ __launch_bounds__(64 * WR * WC, OCC) void brik_i8_tile_##WR##WC##_##WA##x##WB(brik_i8_launch a) { i8_tile<I8Tile<WR, WC, WA, WB>>(a); }
BRIK_I8_TILE(2, 2, 4, 4, 1)
BRIK_I8_TILE(2, 2, 4, 2, 2)
BRIK_I8_TILE(2, 2, 2, 2, 2)
BRIK_I8_TILE(2, 2, 1, 2, 3)

// The splits' sums and the scaling: a thread per four neighbours of y.
extern "C" __global__ __launch_bounds__(256) void brik_i8_join(brik_i8_launch a)
{
    const size_t all = (size_t)a.M * a.N;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        int sum = 0;
        for (int s = 0; s < a.splits; ++s) sum += a.part[s * all + i];
        const size_t m = i / a.N, n = i - m * a.N;
        const float y = (float)sum * a.ws[n] * a.xs[m];
        a.y[i] = a.res ? y + a.res[i] : y;
    }
}
