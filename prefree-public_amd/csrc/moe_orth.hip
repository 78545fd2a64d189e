// moe_orth.hip — orthogonal updates on gfx950 (include/prefree_moe.h): X = G / |G|, then a few times
// X <- a X + (b A + c A A) X with A = X X^T, in 16-bit products on the matrix cores.
//
// X is carried in two f16 pieces, of which the products take the first.  What a rounding of X puts where G has nothing is
// multiplied by a in every step (3.4445^5 = 485), and so are G's small directions with it: in one f16 piece the result of a
// momentum of rank n / 8 came out 1.5 to 4% off (in bf16 11 to 30%), in two 0.14 to 0.17%.  With a second piece of 8 bits
// (e5m2) those were 0.15 to 0.23%, but of rank 3 0.4 to 0.5%, and of rank 1 0.7%, for 0.15 to 0.21 and 0.2 to 0.28 so.  (Emulated
// in 64 bits, 96 to 2048 rows.)  With a X formed from both pieces the roundings of the first reach X by way of A and of B X alone,
// and there they are small beside what X has in the same directions.  A and B = b A + c A A are one f16 piece: where all
// elements of a matrix are of one magnitude, their roundings are alike and add up, to 1% at the most of 1376 sizes.
#include <algorithm>
#include <utility>

#include "moe_orth.hpp"
#include "moe_tiles.hpp"

namespace {

using namespace pfmoe;

// One product of all matrices of a batch; they lie one after the other, rows and columns padded with zeros to multiples of 32.
struct Product {
    const f16 *p, *q;           // rows operand, and columns operand
    int m, n, k;                // of a matrix
    int batch, first;
    int whole, parts;           // tiles in one piece; quarters of the others
    float alpha, beta, gamma;
    const f16 *old;             // kPoly: A
    const f16 *old_rest;
    f16 *out, *rest;
    char *result;               // the last step's, instead of the pieces: [rows][columns], ld_result apart
    long long ld_result;
    int rows, columns, result_f16, wide;
};

// kSquare: A = alpha P P^T
// kPoly: B = gamma I + beta P + alpha P P, P symmetric.  Both are symmetric: the tiles on and under the diagonal, stored twice.
// kApply: X' = P X + beta rest(X): P is B with a on its diagonal, so that a X of the first piece is part of the product.
//         X is read across its rows.
enum { kSquare = 0, kPoly = 1, kApply = 2 };

// Four numbers as their first pieces, and what is left of them.
struct Pieces {
    unsigned first[2], rest[2];
    __device__ __forceinline__ explicit Pieces(const float v[4])
    {
        float left[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) left[i] = (v[i] - (float)(f16)v[i]) * kRest;
        first[0] = pair_of(v[0], v[1]);
        first[1] = pair_of(v[2], v[3]);
        rest[0] = pair_of(left[0], left[1]);
        rest[1] = pair_of(left[2], left[3]);
    }
};
__device__ __forceinline__ void rest_of(unsigned lo, unsigned hi, float v[4])
{
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 a = __builtin_bit_cast(f16x2, lo), b = __builtin_bit_cast(f16x2, hi);
    v[0] = (float)a[0] * (1.0f / kRest);
    v[1] = (float)a[1] * (1.0f / kRest);
    v[2] = (float)b[0] * (1.0f / kRest);
    v[3] = (float)b[1] * (1.0f / kRest);
}

// The tile from row m0 and column n0 of a matrix's product, by KS times WM x WN waves with STAGES times KS tiles of k in LDS.
// Each set of waves takes every KS-th tile of k; in the end they add up, and each finishes its share of the rows.
template <int KIND, int BM, int BN, int WM, int WN, int STAGES, int KS>
__device__ __forceinline__ void orth_tile(const Product &a, int matrix, int m0, int n0, char *shared)
{
    constexpr int THREADS = WM * WN * KS * 64, FM = BM / WM / 16, FN = BN / WN / 16, DONE = FM / KS;
    typedef Along<BM, THREADS, true> P;
    typedef typename std::conditional<KIND == kApply, Across<BN, THREADS, true>, Along<BN, THREADS, true>>::type Q;
    constexpr int TILE = P::kBytes + Q::kBytes, SLOT = KS * TILE, EACH = P::kLoads + Q::kLoads, LOADS = KS * EACH;
    const int id = wave_id(), set = KS > 1 ? id / (WM * WN) : 0, wave = KS > 1 ? id % (WM * WN) : id, wm = wave / WN, wn = wave % WN, k = a.k;
    const auto row_of = [&](int i) { return m0 + ((i + set * DONE) * WM + wm) * 16; };   // of the blocks that this wave finishes
    int lane = threadIdx.x & (kWave - 1);
    const long long base = (long long)matrix * a.m * a.n;

    // The second pieces of what this lane will store: half of them are long there when the products are, the others follow, each as
    // the registers of one are free.  None of the last step's: what they would add is not multiplied any more.
    typedef unsigned Rest __attribute__((ext_vector_type(2 * FN), aligned(16)));
    constexpr int HELD = KIND == kApply ? DONE / 2 : 1;
    Rest rest[HELD];
    const auto read_rest = [&](int i) {
        const int r = row_of(i) + (lane & 15), c = n0 + wn * FN * 16 + (lane >> 4) * 4 * FN;   // 4 FN columns, all there or none
        rest[i % HELD] = Rest{};
        if (a.old_rest && r < a.m && c < a.n) rest[i % HELD] = *(const Rest *)(a.old_rest + base + (long long)r * a.n + c);
    };
    if constexpr (KIND == kApply) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) read_rest(i);
    }

    P p;
    Q q;
    {
        const char *from = (const char *)(a.p + (long long)matrix * a.m * k);
        p.init(from, 2ull * a.m * k, 2LL * k, [&](int r) { return min(m0 + r, a.m - 1); }, k, 8);
    }
    if constexpr (KIND == kApply) {
        q.init((const char *)(a.q + (long long)matrix * k * a.n), 2ull * k * a.n, 2LL * a.n, n0, a.n, k);
    } else {
        const char *from = (const char *)(a.q + (long long)matrix * a.m * k);
        q.init(from, 2ull * a.m * k, 2LL * k, [&](int r) { return min(n0 + r, a.m - 1); }, k, 8);
    }
    const auto lds = [&](int place) { return shared + place * SLOT; };
    const auto issue = [&](int l, int s, char *to) {
        const int i = l % EACH, t = s * KS + l / EACH;
        to += l / EACH * TILE;
        if (i < P::kLoads) p.issue(i, t, to);
        else if constexpr (KIND == kApply) q.template issue<false>(i - P::kLoads, t, to + P::kBytes, 0);
        else q.issue(i - P::kLoads, t, to + P::kBytes);
    };
    const auto read_x = [&](const char *from, int i) { return P::fragment(from + set * TILE, (i * WM + wm) * 16); };
    const auto read_w = [&](const char *from, int j) { return Q::fragment(from + set * TILE + P::kBytes, (wn * FN + j) * 16); };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    i32x4 x[4], w[2][FN];
    // As in k_mm fragments are read ahead of the products, the columns' of the next tile beside this one's; of the STAGES - 1
    // tiles on their way all but the last STAGES - 3 have to be there when the waves meet.
    constexpr int kAhead = STAGES - 1;
    // LDS reads after the last one of this step's own tile: two fragments of rows, and those of columns behind it
    constexpr int kNextReads = 2 + (FN - (FM - 3) * FN / FM) * (KIND == kApply ? 2 : 1);
    const auto step = [&](auto side, int s, char *__restrict__ fill, const char *__restrict__ here, const char *__restrict__ next) {
        constexpr int now = decltype(side)::value;   // of w; the next tile's fragments go to the other
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const char *from = i + 2 < FM ? here : next;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                acc[i][j] = mfma<f16>(w[now][j], x[i % 4], acc[i][j]);
                if (j == 0) x[(i + 2) % 4] = read_x(from, (i + 2) % FM);
                if (j == 1) {
#pragma unroll
                    for (int c = i * FN / FM; c < (i + 1) * FN / FM; ++c) w[1 - now][c] = read_w(next, c);
                }
                if (j == FN / 2) {
#pragma unroll
                    for (int l = i * LOADS / FM; l < (i + 1) * LOADS / FM; ++l) issue(l, s + kAhead, fill);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        wait_and_meet<(STAGES - 3) * LOADS, kNextReads>();
        __builtin_amdgcn_sched_barrier(0);
    };
    const int steps = (k / 32 + KS - 1) / KS;   // by twos: behind k tiles are zeros
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) issue(i, s, lds(s));
    wait_and_meet<(STAGES - 3) * LOADS>();
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = read_x(lds(0), i);
#pragma unroll
    for (int j = 0; j < FN; ++j) w[0][j] = read_w(lds(0), j);
#pragma unroll 1
    for (int s = 0; s < steps; s += 2) {
        step(std::integral_constant<int, 0>(), s, lds((s + kAhead) % STAGES), lds(s % STAGES), lds((s + 1) % STAGES));
        step(std::integral_constant<int, 1>(), s + 1, lds((s + 1 + kAhead) % STAGES), lds((s + 1) % STAGES), lds((s + 2) % STAGES));
    }
    wait_and_meet<0>();   // nothing may still be on its way to LDS when the workgroup ends
    if constexpr (KS > 1) {
        static_assert(FM * FN * 16 * THREADS <= STAGES * SLOT, "sums of all sets");
        f32x4 *box = (f32x4 *)shared + threadIdx.x % (THREADS / KS);
        const auto at = [&](int set, int i, int j) { return ((set * FM + i) * FN + j) * (THREADS / KS); };
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) box[at(set, i, j)] = acc[i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < DONE; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                acc[i][j] = box[at(0, set * DONE + i, j)];
#pragma unroll
                for (int other = 1; other < KS; ++other) acc[i][j] += box[at(other, set * DONE + i, j)];
            }
    }

    // Rows and columns are multiples of 32: blocks of 16 x 16 are there as a whole or not at all.
    asm volatile("" : "+v"(lane));   // addresses are formed here, not kept over the loop before
    const int g = lane >> 4, c0 = n0 + wn * FN * 16;
    typedef f16 f16x4 __attribute__((ext_vector_type(4)));
    f16x4 old[2][FN];   // kPoly: P's, a block of rows ahead
    const auto read_old = [&](int i) {
        if constexpr (KIND == kPoly) {
            const int r = row_of(i) + (lane & 15);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int c = c0 + j * 16 + g * 4;
                old[i % 2][j] = f16x4{0, 0, 0, 0};
                if (r < a.m && c < a.n) old[i % 2][j] = *(const f16x4 *)(a.old + base + (long long)r * a.n + c);
            }
        }
    };
    read_old(0);
#pragma unroll
    for (int i = 0; i < DONE; ++i) {
        if (i + 1 < DONE) read_old(i + 1);
        __builtin_amdgcn_sched_barrier(0);
        const int r0 = row_of(i), r = r0 + (lane & 15);
        if (r0 >= a.m) continue;
        if constexpr (KIND == kApply) {
            unsigned v[FN][4];
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) v[j][c] = __float_as_uint(acc[i][j][c]);
            gather_columns<FN>(v);
            const int c = c0 + g * 4 * FN;
            if (c >= a.n) continue;
            float y[4 * FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                rest_of(rest[i % HELD][2 * j], rest[i % HELD][2 * j + 1], y + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[4 * j + e] = __builtin_fmaf(a.beta, y[4 * j + e], __uint_as_float(v[j][e]));
            }
            if (i + HELD < DONE) read_rest(i + HELD);
            if (a.result) {
                if (r >= a.rows) continue;
#pragma unroll
                for (int e = 0; e < 4 * FN; ++e) y[e] *= a.alpha;
                char *row = a.result + 2 * a.ld_result * ((long long)matrix * a.rows + r);
                if (a.result_f16) store_row<f16, 4 * FN>((f16 *)row, c, a.columns, a.wide, y);
                else store_row<bf16, 4 * FN>((bf16 *)row, c, a.columns, a.wide, y);
                continue;
            }
            const long long to = base + (long long)r * a.n + c;
            Rest left;
#pragma unroll
            for (int j = 0; j < FN; j += 2) {
                const Pieces one(y + 4 * j), two(y + 4 * j + 4);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    left[2 * j + e] = one.rest[e];
                    left[2 * j + 2 + e] = two.rest[e];
                }
                *(i32x4 *)(a.out + to + 4 * j) = i32x4{(int)one.first[0], (int)one.first[1], (int)two.first[0], (int)two.first[1]};
            }
            if (a.rest) *(Rest *)(a.rest + to) = left;
        } else {
            unsigned h[FN][2];
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                f32x4 y = acc[i][j];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[e] *= a.alpha;
                    if constexpr (KIND == kPoly) {
                        y[e] = __builtin_fmaf(a.beta, (float)old[i % 2][j][e], y[e]);
                        if (r == c0 + j * 16 + g * 4 + e) y[e] += a.gamma;
                    }
                }
                h[j][0] = pair_of(y[0], y[1]);
                h[j][1] = pair_of(y[2], y[3]);
            }
            if (m0 != n0) {
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    unsigned z[2] = {h[j][0], h[j][1]};
                    transpose4(z, lane);
                    const int col = c0 + j * 16 + g * 4 + (lane & 3), row = r0 + (lane & 12);
                    if (col < a.n) *(u32x2 *)(a.out + base + (long long)col * a.n + row) = u32x2{z[0], z[1]};
                }
            }
            gather_columns<FN>(h);
            const int c = c0 + g * 4 * FN;
            if (c < a.n) {
#pragma unroll
                for (int j = 0; j < FN; j += 2)
                    *(i32x4 *)(a.out + base + (long long)r * a.n + c + 4 * j) = i32x4{(int)h[j][0], (int)h[j][1], (int)h[j + 1][0], (int)h[j + 1][1]};
            }
        }
    }
}

// Tile `at` of all matrices' tiles of BM x BN.
template <int KIND, int BM, int BN>
__device__ __forceinline__ void find_orth_tile(const Product &a, int at, int &matrix, int &m0, int &n0)
{
    const int mt = (a.m + BM - 1) / BM, nt = (a.n + BN - 1) / BN, each = KIND == kApply ? mt * nt : mt * (mt + 1) / 2;
    matrix = at / each;
    const int t = at - matrix * each;
    if constexpr (KIND == kApply) {   // eight tiles of rows side by side over the columns
        const int group = t / (8 * nt), side = min(8, mt - group * 8), j = t - group * 8 * nt;
        m0 = (group * 8 + j % side) * BM;
        n0 = j / side * BN;
    } else {
        int tm = (int)((__builtin_sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
        while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
        while (tm * (tm + 1) / 2 > t) --tm;
        m0 = tm * BM;
        n0 = (t - tm * (tm + 1) / 2) * BM;
    }
}

// Tiles of 128 x 128.  Up to as many as compute units a workgroup each, with eight waves and seven tiles of k on their way;
// else three a compute unit, of four waves and two tiles on their way, which are one round where two with three would take a
// second one (12 x 717 x 1111, X': 34 us; with a second piece of X in 8 bits 31, for 33).  Even and odd tiles of k by half of the
// waves each, or two more on their way, changed nothing for the former: beside 10 us of tiles a launch of 18 us starts, and ends with
// its stores.
template <int KIND, int WN, int STAGES>
__global__ __launch_bounds__(128 * WN, WN == 2 ? 3 : 2) void k_orth_small(const Product a)
{
    __shared__ __align__(1024) char lds[STAGES * 256 * 64];
    const int id = a.first + blockIdx.x, chunk = (a.whole + kXcds - 1) / kXcds, at = id % kXcds * chunk + id / kXcds;
    if (id / kXcds >= chunk || at >= a.whole) return;
    int matrix, m0, n0;
    find_orth_tile<KIND, 128, 128>(a, at, matrix, m0, n0);
    orth_tile<KIND, 128, 128, 2, WN, STAGES, 1>(a, matrix, m0, n0, lds);
}

// Tiles of 64 rows, where there are few: a step over a tile of k takes a workgroup some 0.25 us however small it is, so that
// it is worth to have more of them, and several tiles of k in a step.
template <int KIND, int BN, int WN, int STAGES, int KS>
__global__ __launch_bounds__(256) void k_orth_tiny(const Product a)
{
    __shared__ __align__(1024) char lds[STAGES * KS * (64 + BN) * 64];
    const int id = a.first + blockIdx.x, chunk = (a.whole + kXcds - 1) / kXcds, at = id % kXcds * chunk + id / kXcds;
    if (id / kXcds >= chunk || at >= a.whole) return;
    int matrix, m0, n0;
    find_orth_tile<KIND, 64, BN>(a, at, matrix, m0, n0);
    orth_tile<KIND, 64, BN, 1, WN, STAGES, KS>(a, matrix, m0, n0, lds);
}

// Tiles of 256 x 256, a workgroup a compute unit, and in quarters those of a last round that is at most half full.  16 x 2048 x
// 2048: A, B and X' 173, 177 and 315 us, X' at 0.87 PFLOP/s.  The products alone are some 200 us of X'; the end of a tile, with nothing
// beside it, reads 134 MB and stores 268 MB in the rest (with a second piece of X in 8 bits 287 us, two thirds of the bytes).
template <int KIND>
__global__ __launch_bounds__(512) void k_orth(const Product a)
{
    __shared__ __align__(1024) char lds[4 * 512 * 64];
    const int id = a.first + blockIdx.x;
    int matrix, m0, n0;
    const int big = (a.whole + kXcds - 1) / kXcds * kXcds;
    if (id < big) {
        const int at = id % kXcds * (big / kXcds) + id / kXcds;
        if (at >= a.whole) return;
        find_orth_tile<KIND, 256, 256>(a, at, matrix, m0, n0);
        orth_tile<KIND, 256, 256, 2, 4, 4, 1>(a, matrix, m0, n0, lds);
        return;
    }
    if (id - big >= a.parts) return;
    find_orth_tile<KIND, 256, 256>(a, a.whole + (id - big) / 4, matrix, m0, n0);
    const bool diagonal = KIND != kApply && m0 == n0;
    m0 += (id - big) / 2 % 2 * 128;
    n0 += (id - big) % 2 * 128;
    if (m0 >= a.m || n0 >= a.n || (diagonal && n0 > m0)) return;
    orth_tile<KIND, 128, 128, 2, 4, 8, 1>(a, matrix, m0, n0, lds);
}

// ---- into the two pieces, and out of them --------------------------------------------------------------------------

constexpr int kCus = 256;                // compute units of the card

constexpr int kNormThreads = 256;
// Sums of squares of every gridDim.x-th row, in 64 bits: no element is too large or too small for its square.  Rows are
// read in the 16 bytes at multiples of 16 that hold any of them, `pieces` a row, and what is not of the row is left out;
// WHOLE: they hold nothing else.  16 bytes that reach over the first matrix's begin or the last one's end are not read as
// such.  (The rows' own eights, shifted out of words: 14 us for 12 x 717 x 1111 in bf16 where this takes 10.)
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kNormThreads) void k_orth_norm(const T *g, long long ld, int rows, int columns, int pieces, double *sums)
{
    constexpr int N = 16 / sizeof(T), LOADS = 8;
    typedef T Piece __attribute__((ext_vector_type(N)));
    __shared__ double part[kNormThreads / kWave];
    const int have = (rows - (int)blockIdx.x - 1) / (int)gridDim.x + 1, units = have * pieces;
    const long long last_row = (long long)gridDim.y * rows - 1;
    const auto row_at = [&](int i) { return g + ((long long)blockIdx.y * rows + blockIdx.x + (long long)gridDim.x * i) * ld; };
    const uintptr_t first = (uintptr_t)g, last = (uintptr_t)(g + last_row * ld + columns);
    const auto outside = [&](uintptr_t p) { return p < first || p + 16 > last; };
    const auto square = [](T v, double sum) { return __builtin_fma((double)(float)v, (double)(float)v, sum); };
    double sum = 0;
    for (int u0 = threadIdx.x; u0 < units; u0 += kNormThreads * LOADS) {
        Piece v[LOADS];
        int at[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {   // their loads go out together
            const int u = u0 + kNormThreads * j, r = u / pieces;
            const uintptr_t row = (uintptr_t)row_at(r), p = (row & ~(uintptr_t)15) + 16LL * (u - r * pieces);
            at[j] = (int)(long long)(p - row) / (int)sizeof(T);
            v[j] = Piece{};
            if (u < units && (WHOLE || !outside(p))) v[j] = *(const Piece *)p;
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            if (WHOLE || __all((unsigned)at[j] < (unsigned)max(columns - N + 1, 0))) {
#pragma unroll
                for (int i = 0; i < N; ++i) sum = square(v[j][i], sum);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) sum = square((unsigned)(at[j] + i) < (unsigned)columns ? v[j][i] : (T)0, sum);
            }
        }
    }
    for (int r = threadIdx.x; !WHOLE && r < have; r += kNormThreads) {   // the few elements of those
        const T *row = row_at(r);
        if ((uintptr_t)row - first >= 16 && last - (uintptr_t)(row + columns) >= 16) continue;
        const auto add = [&](int c) {
            if (outside((uintptr_t)(row + c) & ~(uintptr_t)15)) sum = square(row[c], sum);
        };
        for (int c = 0; c < min(N, columns); ++c) add(c);
        for (int c = max(columns - N, N); c < columns; ++c) add(c);
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kNormThreads / kWave; ++w) sum += part[w];
    sums[(long long)blockIdx.y * gridDim.x + blockIdx.x] = sum;
}

__device__ __forceinline__ void store_pieces(const float v[8], f16 *x, f16 *rest)
{
    const Pieces one(v), two(v + 4);
    *(i32x4 *)x = i32x4{(int)one.first[0], (int)one.first[1], (int)two.first[0], (int)two.first[1]};
    *(i32x4 *)rest = i32x4{(int)one.rest[0], (int)one.rest[1], (int)two.rest[0], (int)two.rest[1]};
}

// The pieces of scale G / |G|, in [m][n] with zeros behind the matrix.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_orth_pieces(const T *g, long long ld, int rows, int columns, const double *sums, int parts, float scale, int m,
                                                     int n, f16 *x, f16 *rest)
{
    const double by = over_norm(sums + (long long)blockIdx.y * parts, parts, scale);
    const T *from = g + (long long)blockIdx.y * rows * ld;
    const int pieces = n / 8, units = m * pieces, first = blockIdx.x * 1024 + threadIdx.x;
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int u = first + 256 * j, r = u / pieces, c = (u - r * pieces) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = 0;
        if (u < units && r < rows && c < columns) load8_any<T, VECTOR>(from + ld * r, c, columns, v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int u = first + 256 * j, r = u / pieces, c = (u - r * pieces) * 8;
        if (u >= units) break;
        // what lies behind the matrix stays zero, whatever the factor
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = r < rows && c + i < columns ? (float)((double)v[j][i] * by) : 0.0f;
        const long long to = (long long)blockIdx.y * m * n + (long long)u * 8;
        store_pieces(v[j], x + to, rest + to);
    }
}

// The same of its transpose, 64 x 64 elements a workgroup.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_orth_pieces_across(const T *g, long long ld, int rows, int columns, const double *sums, int parts, float scale,
                                                            int m, int n, f16 *x, f16 *rest)
{
    __shared__ float tile[64][65];
    const double by = over_norm(sums + (long long)blockIdx.z * parts, parts, scale);
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;   // of X: columns and rows of G
    const T *from = g + (long long)blockIdx.z * rows * ld;
    const int piece = threadIdx.x % 8 * 8, line = threadIdx.x / 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = line + 32 * h;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (c0 + i < rows && r0 + piece < columns) load8_any<T, VECTOR>(from + ld * (c0 + i), r0 + piece, columns, v);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            tile[piece + e][i] = c0 + i < rows && r0 + piece + e < columns ? (float)((double)v[e] * by) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = line + 32 * h;
        if (r0 + i >= m || c0 + piece >= n) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[i][piece + e];
        const long long to = (long long)blockIdx.z * m * n + (long long)(r0 + i) * n + c0 + piece;
        store_pieces(v, x + to, rest + to);
    }
}

// The transposed result out of the pieces.
template <typename T>
__global__ __launch_bounds__(256) void k_orth_out_across(const f16 *x, const f16 *rest, int m, int n, float scale, T *out, long long ld, int rows,
                                                         int columns, int wide)
{
    __shared__ float tile[64][65];
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;   // of X
    const int piece = threadIdx.x % 8 * 8, line = threadIdx.x / 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = line + 32 * h;
        if (r0 + i >= m || c0 + piece >= n) continue;
        const long long at = (long long)blockIdx.z * m * n + (long long)(r0 + i) * n + c0 + piece;
        const f16x8 first = *(const f16x8 *)(x + at);
        const i32x4 left = *(const i32x4 *)(rest + at);
        float v[8];
        rest_of(left[0], left[1], v);
        rest_of(left[2], left[3], v + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) tile[piece + e][i] = ((float)first[e] + v[e]) * scale;
    }
    __syncthreads();
    if (!wide) {   // a row a wave, an element a lane: unaligned rows by eight elements a lane took 26 us where this takes 14
        const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
        for (int i = wave; i < min(64, rows - c0); i += 4)
            if (r0 + lane < columns) out[ld * ((long long)blockIdx.z * rows + c0 + i) + r0 + lane] = (T)tile[i][lane];
        return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = line + 32 * h;
        if (c0 + i >= rows || r0 + piece >= columns) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[i][piece + e];
        store_row<T, 8>(out + ld * ((long long)blockIdx.z * rows + c0 + i), r0 + piece, columns, true, v);
    }
}

template <int KIND>
int product(Product a, hipStream_t s)
{
    const auto tiles = [&](long long side, long long across = 0) {
        const long long mt = (a.m + side - 1) / side, nt = (a.n + (across ? across : side) - 1) / (across ? across : side);
        return a.batch * (KIND == kApply ? mt * nt : mt * (mt + 1) / 2);
    };
    const auto run = [&](auto kernel, long long workgroups, int threads) {
        if (workgroups > 0x7fffffffLL) return pfk_internal_fail(PF_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
        in_launches(workgroups, most_workgroups(threads), [&](long long first, long long count) {
            a.first = (int)first;
            kernel<<<dim3((unsigned)count), dim3(threads), 0, s>>>(a);
        });
        return pfk_internal_launched("k_orth");
    };
    // X' of 129 to 192 rows, which larger tiles would leave empty by a quarter, in tiles of 64 x 128 / 128 x 128 / 256 x 256, whole calls
    // in us: 96 x 139 x 2765 734 / 788 / 741, 96 x 160 x 2765 762 / 815 / 773, 64 x 190 x 4000 809 / 826 / 787, 40 x 139 x 1400 179 / 198 /
    // 174, 32 x 139 x 2765 252 / 273 / 286, 128 x 150 x 1000 339 / 366 / 351, 16 x 170 x 4000 233 / 246 / 232
    if (KIND == kApply && 2 * tiles(64, 128) <= 3 * tiles(128) && tiles(64, 128) > kCus) {
        a.whole = (int)tiles(64, 128);
        if constexpr (KIND == kApply) return run(k_orth_tiny<KIND, 128, 4, 4, 1>, (a.whole + kXcds - 1LL) / kXcds * kXcds, 256);
    }
    // Tiles of 256 x 256 unless they cover over 1.4 times as much as those of 128 x 128: 128 x 289 x 1567, A and B 82, 33 / 64, 22, X'
    // 178 / 151; 96 x 101 x 3705 X' 83 / 73; 128 x 221 x 3693 X' 194 / 211.
    const long long large = tiles(256), small = tiles(128);
    if (large >= kCus && 20 * large <= 7 * small) {
        const long long over = large % kCus <= kCus / 2 ? large % kCus : 0;
        a.whole = (int)(large - over);
        a.parts = (int)(4 * over);
        return run(k_orth<KIND>, (a.whole + kXcds - 1LL) / kXcds * kXcds + a.parts, 512);
    }
    // A, B and X' (with a second piece of 8 bits; up to 0.7 more so) in us, tiles of 64 rows against 128: 1 x 500 x 1000 8.9, 7.0, 8.9
    // / 12.4, 10.5, 10.3; 1 x 512 x 4096 19.7, 7.1, 9.5 / 30.8, 10.2, 10.6 (A by twos of tiles of k 24.5); 1 x 1024 x 1024 9.9, 10.1, 12.6 / 12.9, 14.7, 13.4; 12 x 300 x 300 6.1, 7.0,
    // 7.9 / -, -, 9.1; with more of them than fit at once: 3 x 800 x 800 10.6, 11.5, 13.8 / 12.6, 13.6, 12.7; 2 x 1100 x 1100 12.4,
    // 13.4, 18.9 / 15.6, 16.7, 16.8; 16 x 500 x 500 12.5, 13.8, 14.2 / 10.7, 11.8, 13.2; 1 x 2048 x 2048 32, 33, 32 / 22, 24, 26.
    if constexpr (KIND == kApply) {
        a.whole = (int)tiles(64, 128);
        if (a.whole <= kCus) return run(k_orth_tiny<KIND, 128, 4, 6, 1>, (a.whole + kXcds - 1LL) / kXcds * kXcds, 256);
    } else {
        a.whole = (int)tiles(64);
        if (a.whole <= kCus && a.k >= 1024) return run(k_orth_tiny<KIND, 64, 1, 4, 4>, (a.whole + kXcds - 1LL) / kXcds * kXcds, 256);
        if (a.whole <= 2 * kCus) return run(k_orth_tiny<KIND, 64, 2, 4, 2>, (a.whole + kXcds - 1LL) / kXcds * kXcds, 256);
    }
    // with a long k also of more tiles one at a time: A of 96 x 139 x 2765 41 / 59, 128 x 221 x 3693 80 / 100, 128 x 1567 64 / 66
    a.whole = (int)small;
    if (a.whole <= kCus || (KIND != kApply && a.k >= 1536)) return run(k_orth_small<KIND, 4, 8>, (a.whole + kXcds - 1LL) / kXcds * kXcds, 512);
    return run(k_orth_small<KIND, 2, 3>, (a.whole + kXcds - 1LL) / kXcds * kXcds, 256);
}

// launch(grid, first matrix) with a workgroup for each 64 x 64 elements of each matrix
template <typename F>
void each_tile(int batch, int m, int n, F launch)
{
    const long long x = (n + 63) / 64, y = (m + 63) / 64;
    in_launches(batch, std::max(1LL, most_workgroups(256) / (x * y)), [&](long long first, long long count) {
        launch(dim3((unsigned)x, (unsigned)y, (unsigned)count), first);
    });
}

struct Held {
    int m, n;
    float scale;
    f16 *x, *rest;
};

// Squares' sums and, but for narrow matrices, the pieces; returns how many sums a matrix has.
template <typename T>
int into_pieces(const void *from, long long ld, int batch, int rows, int columns, double *sums, const Held &h, hipStream_t s)
{
    const T *g = (const T *)from;
    const bool vector = (uintptr_t)g % 16 == 0 && ld * sizeof(T) % 16 == 0;
    const int parts = std::min(rows, std::min(kParts, std::max(1, 2048 / batch))), m = h.m, n = h.n;   // eight workgroups a compute unit
    const bool whole = vector && columns * sizeof(T) % 16 == 0;
    const int pieces = (int)((columns * sizeof(T) + 15) / 16) + !vector;   // a row that starts inside one may reach into one more
    const auto norm = whole ? k_orth_norm<T, true> : k_orth_norm<T, false>;
    norm<<<dim3(parts, batch), dim3(kNormThreads), 0, s>>>(g, ld, rows, columns, pieces, sums);
    if (!h.x) return parts;
    if (rows > columns) {
        const auto kernel = vector ? k_orth_pieces_across<T, true> : k_orth_pieces_across<T, false>;
        each_tile(batch, m, n, [&](dim3 grid, long long at) {
            kernel<<<grid, dim3(256), 0, s>>>(g + at * rows * ld, ld, rows, columns, sums + at * parts, parts, h.scale, m, n, h.x + at * m * n,
                                              h.rest + at * m * n);
        });
        return parts;
    }
    const auto kernel = vector ? k_orth_pieces<T, true> : k_orth_pieces<T, false>;
    const long long each = ((long long)m * n / 8 + 1023) / 1024;
    in_launches(batch, std::max(1LL, most_workgroups(256) / each), [&](long long at, long long count) {
        kernel<<<dim3((unsigned)each, (unsigned)count), dim3(256), 0, s>>>(g + at * rows * ld, ld, rows, columns, sums + at * parts, parts, h.scale, m, n,
                                                                          h.x + at * m * n, h.rest + at * m * n);
    });
    return parts;
}

template <typename T>
void out_across(const Held &h, int batch, void *out, long long ld, int rows, int columns, int wide, hipStream_t s)
{
    each_tile(batch, h.m, h.n, [&](dim3 grid, long long at) {
        const long long from = at * h.m * h.n;
        k_orth_out_across<T><<<grid, dim3(256), 0, s>>>(h.x + from, h.rest + from, h.m, h.n, 1 / h.scale, (T *)out + at * rows * ld, ld, rows,
                                                        columns, wide);
    });
}

}  // namespace

extern "C" int pfk_orthogonalize(const void *g, long long ld_g, int dtype, int batch, int rows, int columns, const float *steps,
                                 int n_steps, void *out, long long ld_out, int out_dtype, void *workspace, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    const bool across = rows > columns;
    const int m = PFK_ORTH_SIDE(across ? columns : rows), n = PFK_ORTH_SIDE(across ? rows : columns);
    const long long xs = (long long)batch * m * n, as = (long long)batch * m * m;
    f16 *x = (f16 *)workspace, *rest = x + 2 * xs, *a = rest + 2 * xs, *b = a + as;
    double *sums = (double *)(b + as);
    float scale = 1;   // X is held times this: elements of about 1, and none over 2^12 where X has none over 4
    while (scale * scale * 4 <= n && scale < 1024) scale *= 2;
    const bool narrow = m <= PFK_ORTH_NARROW;
    if (narrow) sums = (double *)workspace;
    Held from = {m, n, scale, narrow ? nullptr : x, rest}, to = {m, n, scale, x + xs, rest + xs};
    const int parts = dtype == PF_F32   ? into_pieces<float>(g, ld_g, batch, rows, columns, sums, from, s)
                      : dtype == PF_F16 ? into_pieces<f16>(g, ld_g, batch, rows, columns, sums, from, s)
                                        : into_pieces<bf16>(g, ld_g, batch, rows, columns, sums, from, s);
    if (narrow)
        return launch_narrow({g, ld_g, ld_out, dtype, batch, rows, columns, n_steps, out_dtype == PF_F16, steps, scale, sums, parts, out,
                              (char *)workspace + 8LL * PFK_ORTH_PARTS * batch}, s);
    const int wide = (uintptr_t)out % 16 == 0 && ld_out % 8 == 0;
    for (int i = 0; i < n_steps; ++i) {
        const float *c = steps + 3 * i;
        Product square = {};
        square.p = square.q = from.x;
        square.m = square.n = m;
        square.k = n;
        square.batch = batch;
        square.alpha = 1 / (scale * scale);
        square.out = a;
        Product poly = square;
        poly.p = poly.q = poly.old = a;
        poly.k = m;
        poly.alpha = c[2];
        poly.beta = c[1];
        poly.gamma = c[0];
        poly.out = b;
        Product apply = {};
        apply.p = b;
        apply.q = from.x;
        apply.m = apply.k = m;
        apply.n = n;
        apply.batch = batch;
        apply.alpha = 1 / scale;
        apply.beta = c[0];
        apply.old_rest = i == 0 || i < n_steps - 1 ? from.rest : nullptr;
        apply.out = to.x;
        apply.rest = across || i < n_steps - 2 ? to.rest : nullptr;
        if (i == n_steps - 1 && !across) {
            apply.result = (char *)out;
            apply.ld_result = ld_out;
            apply.rows = rows;
            apply.columns = columns;
            apply.result_f16 = out_dtype == PF_F16;
            apply.wide = wide;
        }
        int st = product<kSquare>(square, s);
        if (st == PF_OK) st = product<kPoly>(poly, s);
        if (st == PF_OK) st = product<kApply>(apply, s);
        if (st != PF_OK) return st;
        std::swap(from, to);
    }
    if (across) {
        if (out_dtype == PF_F16) out_across<f16>(from, batch, out, ld_out, rows, columns, wide, s);
        else out_across<bf16>(from, batch, out, ld_out, rows, columns, wide, s);
    }
    return pfk_internal_launched("k_orth_out_across");
}
