// moe_mm_rows.hip — grouped products with few rows an expert (tokens of sequences that answer): bound by reading the
// weights, which go straight from memory to the matrix cores' registers, once for up to 16 rows.
#include "moe_tiles.hpp"

namespace pfmoe {
namespace {

constexpr int kWaves = 4;
// 16-byte pieces of a row that a lane takes at a time; four lanes share a row.  With two, rows of few bytes still give every
// wave several turns, and more waves fit: 8-bit integers, 16 tokens, 8 of 64 experts, 2048 -> 2 x 1024, in 42 us and not 51, 64
// tokens of 128, 4096 -> 2 x 512, in 89 and not 103, with one 101.  (The others' order of summation stays as it was.)
template <int FORM> constexpr int kPiecesOf = FORM == kI8 ? 2 : 4;

// A workgroup computes 16 columns (and the 16 of the gate) of up to 16 rows.  Its waves share k out in blocks of
// kPieces pieces a lane, the next block's weights on their way while one is multiplied, and add their sums in LDS in a
// fixed order.  Lane l has row l % 16 of both operands and the k that group g = l / 16 takes: of 16-bit elements the
// pieces g, 4 + g, ... of a block, of 4-bit ones 4 g to 4 g + 3, whose four scales are then one word.
//
// Measured with the weights not in cache: one token, 8 of 64 experts, 2048 -> 2 x 1024, 67 MB, in 12.9 us; 67 tokens, 537
// MB in 107 to 109 us, 5.0 TB/s (a stream that only reads: 6.2, with non-temporal loads 7.0).  With the gate a wave has twice the loads on their way, and two waves a SIMD
// with their registers do better than three with a spill (118 us); without it two to four are alike.
template <typename T, int FORM, int ACT, bool ALIGNED>
__global__ __launch_bounds__(kWaves * kWave, FORM == kI8 || (ALIGNED && !ACT) ? 4 : 2) void k_mm_rows(const Args a)
{
    constexpr bool FP4 = FORM == kMx4;
    constexpr int kPieces = kPiecesOf<FORM>;
    constexpr int NB = ACT ? 2 : 1;
    typedef typename sums_of<FORM>::type SUM;
    typedef typename std::conditional<FORM == kI8, int, float>::type Sum;
    __shared__ Sum sums[kWaves][NB][256];
    const int lane = threadIdx.x & (kWave - 1), wave = wave_id(), g = lane >> 4, r = lane & 15;
    const int nt = (a.n + 15) / 16;
    Tile t;
    if (!find_tile<16>(a, nt, a.first + blockIdx.x, t)) return;
    const int m0 = t.m * 16, count = t.end - t.begin, blocks32 = a.k / 32;

    // The weights' addresses need the expert alone: their first loads go out before the rows are looked up.
    const char *x, *w[NB];
    const unsigned char *xs, *ws[FP4 ? NB : 1];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const long long row = min(t.n * 16 + r, a.n - 1) + (long long)b * a.n;
        w[b] = a.q + a.q_expert * t.e + a.ld_q * row;
        if constexpr (FP4) ws[b] = a.q_scales + blocks32 * ((long long)NB * a.n * t.e + row);
    }

    const int pieces = ALIGNED ? a.k / kPerPiece<FORM> : (a.k + 7) / 8;
    const int blocks = (pieces + 4 * kPieces - 1) / (4 * kPieces);
    typedef typename std::conditional<ALIGNED, i32x4, Words>::type Piece;
    const bool any = a.k > 0;
    const uintptr_t x_end = any ? end_of(a.p, a.ld_p * (a.p_rows - 1LL) + 2LL * a.k) : 0;
    const uintptr_t w_end = any ? end_of(a.q + a.q_expert * t.e, a.q_expert) : 0;
    const auto whole = [&](int b) { return (b + 1) * 32 * kPieces <= a.k; };   // whether rows have all of block b
    const auto load = [&](const char *row, int b, Piece (&v)[kPieces], uintptr_t end) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const int at = b * 4 * kPieces + (FP4 ? kPieces * g + u : 4 * u + g);
            if constexpr (ALIGNED) {
                v[u] = i32x4{0, 0, 0, 0};
                if (at < pieces) v[u] = *(const i32x4 *)(row + 16LL * at);
            } else {
                const uintptr_t p = word_of((uintptr_t)row + 16LL * at);
                if (whole(b)) v[u].load(p, p + 8 * Words::shift_of((uintptr_t)row));
                else v[u].load_until(p, end);
            }
        }
    };
    const auto settled = [&](const Piece &v, const char *row, int b, int u) {
        if constexpr (ALIGNED) {
            return v;
        } else {
            const i32x4 r = v.shifted(Words::shift_of((uintptr_t)row));
            return whole(b) ? r : Words::kept(r, a.k - (b * 4 * kPieces + 4 * u + g) * 8);
        }
    };
    const auto load_scales = [&](const unsigned char *row, int b) {
        const int at = b * 4 * kPieces + kPieces * g;
        unsigned v = 0x7f7f7f7fu;   // 1 where the codes are zeros behind the row's end
        if (at + 4 <= blocks32) {
            __builtin_memcpy(&v, row + at, 4);
        } else {
            for (int i = 0; at + i < blocks32; ++i) v = (v & ~(0xffu << 8 * i)) | (unsigned)row[at + i] << 8 * i;
        }
        return (int)v;
    };

    SUM acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = SUM{0, 0, 0, 0};
    Piece wv[2][NB][kPieces], xv[2][kPieces];
    int wsv[2][NB], xsv[2];
    const auto fetch_w = [&](int side, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            load(w[j], b, wv[side][j], w_end);
            if constexpr (FP4) wsv[side][j] = load_scales(ws[j], b);
        }
    };
    const auto fetch_x = [&](int side, int b) __attribute__((always_inline)) {
        load(x, b, xv[side], x_end);
        if constexpr (FP4) xsv[side] = load_scales(xs, b);
    };
    const auto fetch = [&](int side, int b) __attribute__((always_inline)) {
        fetch_w(side, b);
        fetch_x(side, b);
    };
    const auto piece = [&](int side, int b, auto at) __attribute__((always_inline)) {
        constexpr int u = decltype(at)::value;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            if constexpr (FP4) {
                const i32x4 &p = wv[side][j][u], &q = xv[side][u];
                const i32x8 A = {p[0], p[1], p[2], p[3], 0, 0, 0, 0}, B = {q[0], q[1], q[2], q[3], 0, 0, 0, 0};
                acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc[j], 4, 4, u, wsv[side][j], u, xsv[side]);
            } else if constexpr (FORM == kI8) {
                acc[j] = mfma_i8(wv[side][j][u], xv[side][u], acc[j]);
            } else {
                acc[j] = mfma<T>(settled(wv[side][j][u], w[j], b, u), settled(xv[side][u], x, b, u), acc[j]);
            }
        }
    };
    const auto multiply = [&](int side, int b) __attribute__((always_inline)) {
        piece(side, b, std::integral_constant<int, 0>());
        piece(side, b, std::integral_constant<int, 1>());
        if constexpr (kPieces > 2) {
            piece(side, b, std::integral_constant<int, 2>());
            piece(side, b, std::integral_constant<int, 3>());
        }
    };
    int b = wave;
    if (b < blocks) fetch_w(0, b);
    const long long x_row = row_of_slot(a, t.begin + min(m0 + r, count - 1));
    x = a.p + a.ld_p * x_row;
    if constexpr (FP4) xs = a.p_scales + blocks32 * x_row;
    if (b < blocks) fetch_x(0, b);
    while (b < blocks) {
        if (b + kWaves < blocks) fetch(1, b + kWaves);
        multiply(0, b);
        b += kWaves;
        if (b >= blocks) break;
        if (b + kWaves < blocks) fetch(0, b + kWaves);
        multiply(1, b);
        b += kWaves;
    }

#pragma unroll
    for (int j = 0; j < NB; ++j) *(SUM *)&sums[wave][j][r * 16 + g * 4] = acc[j];
    __syncthreads();
    const int s = m0 + threadIdx.x / 16, n = t.n * 16 + threadIdx.x % 16;
    float v[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j)
        v[j] = (float)((sums[0][j][threadIdx.x] + sums[1][j][threadIdx.x]) + (sums[2][j][threadIdx.x] + sums[3][j][threadIdx.x]));
    if (s >= count || n >= a.n) return;
    if constexpr (FORM == kI8) {
        const float mine = a.p_unit[row_of_slot(a, t.begin + s)];
#pragma unroll
        for (int j = 0; j < NB; ++j) v[j] = v[j] * mine * a.q_unit[(long long)NB * a.n * t.e + (long long)j * a.n + n];
    }
    T *out = (T *)(a.out + a.ld_out * ((long long)t.begin + s)) + n;
    if constexpr (ACT) {
        *out = (T)(silu(v[0]) * v[1]);
        if (a.pre) {
            T *pre = (T *)(a.pre + a.ld_pre * ((long long)t.begin + s)) + n;
            pre[0] = (T)v[0];
            pre[a.n] = (T)v[1];
        }
    } else {
        *out = (T)v[0];
    }
}

}  // namespace

template <typename T, int FORM, int ACT, bool ALIGNED>
int launch_rows(const Args &a, hipStream_t stream)
{
    const long long tiles = ((long long)a.slots / 16 + (a.experts < a.slots ? a.experts : a.slots)) * ((a.n + 15) / 16);
    return launch_tiles(k_mm_rows<T, FORM, ACT, ALIGNED>, a, tiles, kWaves * kWave, stream, "k_mm_rows");
}

template int launch_rows<f16, kHalf, 0, true>(const Args &, hipStream_t);
template int launch_rows<f16, kHalf, 0, false>(const Args &, hipStream_t);
template int launch_rows<f16, kHalf, 1, true>(const Args &, hipStream_t);
template int launch_rows<f16, kHalf, 1, false>(const Args &, hipStream_t);
template int launch_rows<f16, kMx4, 0, true>(const Args &, hipStream_t);
template int launch_rows<f16, kI8, 0, true>(const Args &, hipStream_t);
template int launch_rows<f16, kMx4, 1, true>(const Args &, hipStream_t);
template int launch_rows<f16, kI8, 1, true>(const Args &, hipStream_t);
template int launch_rows<bf16, kHalf, 0, true>(const Args &, hipStream_t);
template int launch_rows<bf16, kHalf, 0, false>(const Args &, hipStream_t);
template int launch_rows<bf16, kHalf, 1, true>(const Args &, hipStream_t);
template int launch_rows<bf16, kHalf, 1, false>(const Args &, hipStream_t);
template int launch_rows<bf16, kMx4, 0, true>(const Args &, hipStream_t);
template int launch_rows<bf16, kI8, 0, true>(const Args &, hipStream_t);
template int launch_rows<bf16, kMx4, 1, true>(const Args &, hipStream_t);
template int launch_rows<bf16, kI8, 1, true>(const Args &, hipStream_t);

}  // namespace pfmoe
