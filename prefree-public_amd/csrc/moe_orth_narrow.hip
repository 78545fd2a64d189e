// moe_orth_narrow.hip — orthogonal updates of matrices with at most 64 rows (or columns) on gfx950: one launch a step.
//
// X is held by columns, of up to 64 numbers, in two f16 pieces; a workgroup takes a share of them.  In a step every workgroup
// adds the shares' parts of A = X X^T, forms B = a I + b A + c A A (64^3 products, by each of them: less than a launch),
// X' = B X of its columns and its part of the next A.  The matrix cores hand out four rows of a column a lane, and eight of
// two blocks, in whatever order, are a fragment of the product over columns: X' goes on to A as it comes.  A launch is
// loads, meetings and a few hundred products one after the other, not their number: so A and B are in two pieces as well,
// and of each product all but rest times rest is formed, for results as exact as their type.
// 64 x 2048 from fp32 in five steps: 7 launches, 64 us (60 with one piece of A, B and the products' X, then 2 10^-3 off; now
// 2 10^-4 in f16, which is its rounding); by tiles of 128 x 128, 17 launches, 152 us.  128 x 37 x 3871: 222 us, a
// share or two a matrix, columns of 40 numbers (734 with 16 shares each and columns of 64).
#include "moe_orth.hpp"

namespace {

using namespace pfmoe;

constexpr int kSide = PFK_ORTH_NARROW;
static_assert(kSide == 64, "four blocks of 16");
constexpr int kWaves = 8;   // a wave for each 32 columns of a share of 256

struct Step {
    const void *g;          // the first launch: X from the matrices
    long long ld_g;
    const double *sums;
    int parts;
    float scale;
    const float *gram;      // else: parts of A, [batch][shares][64][64]
    float over, a, b, c;    // A's factor, the step's triple
    f16 *x, *rest;          // [batch][n][side]
    int side;               // the rows of X there are, rounded up to a piece of eight
    float *next;            // parts of the next A; the last launch has none
    void *out;              // the last launch: the result
    long long ld_out;
    int out_f16;
    int rows, columns, across, m, n, shares, blocks;   // X is m x n; blocks: of 32 columns a share
};

__device__ __forceinline__ f32x4 product(const i32x4 &a, const i32x4 &b, const f32x4 &c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// four numbers in two pieces
__device__ __forceinline__ void store_two(f16 *first, f16 *rest, const f32x4 &v)
{
    float left[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) left[e] = v[e] - (float)(f16)v[e];
    *(u32x2 *)first = u32x2{pair_of(v[0], v[1]), pair_of(v[2], v[3])};
    *(u32x2 *)rest = u32x2{pair_of(left[0], left[1]), pair_of(left[2], left[3])};
}

// What is not X's is read too, from its last row or column, so that no load has to wait for a branch.
template <typename T>
__device__ __forceinline__ float element(const Step &a, int matrix, int m, int n)
{
    m = min(m, a.m - 1);
    n = min(n, a.n - 1);
    return (float)((const T *)a.g)[((long long)matrix * a.rows + (a.across ? n : m)) * a.ld_g + (a.across ? m : n)];
}

// four of a row of the matrices, that are all there, at any address
template <typename T>
__device__ __forceinline__ void four_elements(const Step &a, int matrix, int m, int n, float v[4])
{
    typedef T four __attribute__((ext_vector_type(4)));
    typedef four any_t __attribute__((aligned(sizeof(T))));
    const four h = *(const any_t *)((const T *)a.g + ((long long)matrix * a.rows + min(m, a.m - 1)) * a.ld_g + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)h[e];
}

template <typename T>
__device__ __forceinline__ void store_result(const Step &a, int matrix, int m, int n, const float v[4])
{
    if (a.across) {   // v: four rows of the result, column m
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (m < a.m && n + e < a.n) ((T *)a.out)[((long long)matrix * a.rows + n + e) * a.ld_out + m] = (T)v[e];
    } else if (m < a.m) {
        T *to = (T *)a.out + ((long long)matrix * a.rows + m) * a.ld_out + n;
        if (n + 4 <= a.n) {
            typedef T four __attribute__((ext_vector_type(4)));
            typedef four any_t __attribute__((aligned(sizeof(T))));
            *(any_t *)to = four{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < a.n) to[e] = (T)v[e];
        }
    }
}

// T: of the matrices, for the first launch.  SIDE: numbers a column, or 0 where the argument says so (of 64 by the argument, 64 x
// 2048 takes 68 us and not 64; 33 x 4000 in columns of 64 takes 70 us, of 40 61).
template <bool FIRST, bool LAST, typename T, int SIDE>
__global__ __launch_bounds__(kWaves * kWave) void k_orth_narrow(const Step a)
{
    constexpr int LD = kSide + 8;
    __shared__ __align__(16) union {
        struct {
            f16 square[2][kSide][LD], poly[2][kSide][LD];   // A and B, two pieces each
        } s;
        float parts[kWaves][kSide][kSide + 4];   // rows in other banks
    } lds;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, g = lane >> 4, i16 = lane & 15;
    const int matrix = blockIdx.y, share = blockIdx.x, side = SIDE ? SIDE : a.side;
    const long long n_held = (long long)a.shares * a.blocks * 32;   // columns of X there is room for
    f16 *x = a.x + matrix * n_held * side, *rest = a.rest + matrix * n_held * side;

    i32x4 h[2][2], l[2][2];   // 32 columns' pieces, as fragments
    const auto fetch = [&](int block) {
        const long long n0 = ((long long)share * a.blocks + block) * 32;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                // rows behind the last are not held: the first ones are loaded, and multiplied by zeros
                const long long at = (n0 + half * 16 + i16) * side + (ks * 32 + g * 8 < side ? ks * 32 + g * 8 : 0);
                h[half][ks] = *(const i32x4 *)(x + at);
                l[half][ks] = *(const i32x4 *)(rest + at);
            }
    };
    i32x4 poly[2][4][2];   // B's columns, as fragments
    double by = 0;
    if constexpr (FIRST) {
        by = over_norm(a.sums + (long long)matrix * a.parts, a.parts, a.scale);
    } else {
        // the first columns are on their way meanwhile
        if (wave < a.blocks) fetch(wave);
        const float *gram = a.gram + (long long)matrix * a.shares * kSide * kSide + threadIdx.x * 4;
        f32x4 sum[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
        for (int s0 = 0; s0 < a.shares; s0 += 8) {   // sixteen loads at a time
            f32x4 v[8][2];
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) v[s][e] = *(const f32x4 *)(gram + min(s0 + s, a.shares - 1) * kSide * kSide + 2048 * e);
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) sum[e] += s0 + s < a.shares ? v[s][e] : f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int at = threadIdx.x * 4 + 2048 * e, r = at / kSide, c = at % kSide;
            sum[e] *= a.over;
            store_two(&lds.s.square[0][r][c], &lds.s.square[1][r][c], sum[e]);
        }
        __syncthreads();
        // A is symmetric: its rows are its columns, and what a lane has of a column it stores as a piece of a row
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int rb = wave / 2, cb = wave % 2 * 2 + j;
            f32x4 d = f32x4{0, 0, 0, 0};
            const auto at = [&](int piece, int block, int ks) { return *(const i32x4 *)&lds.s.square[piece][block * 16 + i16][ks * 32 + g * 8]; };
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                d = product(at(1, rb, ks), at(0, cb, ks), d);
                d = product(at(0, rb, ks), at(1, cb, ks), d);
                d = product(at(0, rb, ks), at(0, cb, ks), d);
            }
            const int c = cb * 16 + i16, r = rb * 16 + g * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float same = (float)lds.s.square[0][c][r + e] + (float)lds.s.square[1][c][r + e];
                d[e] = __builtin_fmaf(a.b, same, a.c * d[e]) + (r + e == c ? a.a : 0.0f);
            }
            store_two(&lds.s.poly[0][c][r], &lds.s.poly[1][c][r], d);
        }
        __syncthreads();
#pragma unroll
        for (int piece = 0; piece < 2; ++piece)
#pragma unroll
            for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const i32x4 v = *(const i32x4 *)&lds.s.poly[piece][ib * 16 + i16][ks * 32 + g * 8];
                    poly[piece][ib][ks] = ks * 32 + g * 8 < side ? v : i32x4{0, 0, 0, 0};
                }
    }

    f32x4 gram[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) gram[i][j] = f32x4{0, 0, 0, 0};
    for (int block = wave; block < a.blocks; block += kWaves) {
        const int n0 = (share * a.blocks + block) * 32;
        if (n0 >= a.n) break;
        float y[4][2][4];   // row 16 ib + i16; columns n0 + 16 half + 4 g to + 3
        if constexpr (FIRST) {
            if (!a.across && n0 + 32 <= a.n) {
#pragma unroll
                for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                    for (int half = 0; half < 2; ++half) four_elements<T>(a, matrix, ib * 16 + i16, n0 + half * 16 + g * 4, y[ib][half]);
            } else {
#pragma unroll
                for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[ib][half][e] = element<T>(a, matrix, ib * 16 + i16, n0 + half * 16 + g * 4 + e);
            }
            // what lies behind the matrix stays zero, whatever the factor
#pragma unroll
            for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool is = ib * 16 + i16 < a.m && n0 + half * 16 + g * 4 + e < a.n;
                        y[ib][half][e] = is ? (float)((double)y[ib][half][e] * by) : 0.0f;
                    }
        } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f32x4 d[4];
#pragma unroll
                for (int ib = 0; ib < 4; ++ib) d[ib] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                    for (int ib = 0; ib < 4; ++ib) d[ib] = product(l[half][ks], poly[0][ib][ks], d[ib]);
#pragma unroll
                    for (int ib = 0; ib < 4; ++ib) d[ib] = product(h[half][ks], poly[1][ib][ks], d[ib]);
#pragma unroll
                    for (int ib = 0; ib < 4; ++ib) d[ib] = product(h[half][ks], poly[0][ib][ks], d[ib]);
                }
#pragma unroll
                for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[ib][half][e] = d[ib][e];
            }
            if (block + kWaves < a.blocks) fetch(block + kWaves);
        }
        if constexpr (LAST) {
#pragma unroll
            for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = y[ib][half][e] * (1 / a.scale);
                    if (a.out_f16) store_result<f16>(a, matrix, ib * 16 + i16, n0 + half * 16 + g * 4, v);
                    else store_result<bf16>(a, matrix, ib * 16 + i16, n0 + half * 16 + g * 4, v);
                }
        } else {
            i32x4 frag[2][4];
#pragma unroll
            for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    unsigned hi[2], lo[2];
                    float left[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) left[e] = y[ib][half][e] - (float)(f16)y[ib][half][e];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        hi[e] = pair_of(y[ib][half][2 * e], y[ib][half][2 * e + 1]);
                        lo[e] = pair_of(left[2 * e], left[2 * e + 1]);
                        frag[0][ib][2 * half + e] = (int)hi[e];
                        frag[1][ib][2 * half + e] = (int)lo[e];
                    }
                    transpose4(hi, lane);
                    transpose4(lo, lane);
                    const long long at = (long long)(n0 + half * 16 + g * 4 + (lane & 3)) * side + ib * 16 + (lane & 12);
                    if (ib * 16 + (lane & 12) >= side) continue;
                    *(u32x2 *)(x + at) = u32x2{hi[0], hi[1]};
                    *(u32x2 *)(rest + at) = u32x2{lo[0], lo[1]};
                }
#pragma unroll
            for (int term = 0; term < 3; ++term)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) gram[i][j] = product(frag[term == 0][i], frag[term == 1][j], gram[i][j]);
        }
    }
    if constexpr (!LAST) {
        __syncthreads();   // the parts lie where A and B did
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(f32x4 *)&lds.parts[wave][j * 16 + i16][i * 16 + g * 4] = gram[i][j];
        __syncthreads();
        float *next = a.next + ((long long)matrix * a.shares + share) * kSide * kSide;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int at = threadIdx.x * 4 + 2048 * e, r = at / kSide, c = at % kSide;
            f32x4 sum = *(const f32x4 *)&lds.parts[0][r][c];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) sum += *(const f32x4 *)&lds.parts[w][r][c];
            *(f32x4 *)(next + at) = sum;
        }
    }
}

template <bool FIRST, bool LAST, typename T>
void run(const Step &a, dim3 grid, hipStream_t s)
{
    const auto kernel = a.side == kSide ? k_orth_narrow<FIRST, LAST, T, kSide> : k_orth_narrow<FIRST, LAST, T, 0>;
    kernel<<<grid, dim3(kWaves * kWave), 0, s>>>(a);
}

}  // namespace

int pfmoe::launch_narrow(const Narrow &g, hipStream_t s)
{
    Step a = {};
    a.g = g.g;
    a.ld_g = g.ld_g;
    a.sums = g.sums;
    a.parts = g.parts;
    a.scale = g.scale;
    a.over = 1 / (g.scale * g.scale);
    a.rows = g.rows;
    a.columns = g.columns;
    a.across = g.rows > g.columns;
    a.m = a.across ? g.columns : g.rows;
    a.n = a.across ? g.rows : g.columns;
    a.shares = PFK_ORTH_SHARES(g.batch, a.n);
    a.blocks = PFK_ORTH_BLOCKS(g.batch, a.n);
    a.side = (a.m + 7) / 8 * 8;
    const long long held = (long long)g.batch * a.shares * a.blocks * 32 * a.side, gram = (long long)g.batch * a.shares * kSide * kSide;
    a.x = (f16 *)g.workspace;
    a.rest = a.x + held;
    float *parts[2] = {(float *)(a.rest + held), (float *)(a.rest + held) + gram};
    a.out_f16 = g.out_f16;
    a.ld_out = g.ld_out;
    const dim3 grid(a.shares, g.batch);
    a.next = parts[0];
    if (g.dtype == PF_F32) run<true, false, float>(a, grid, s);
    else if (g.dtype == PF_F16) run<true, false, f16>(a, grid, s);
    else run<true, false, bf16>(a, grid, s);
    for (int i = 0; i < g.n_steps; ++i) {
        a.gram = parts[i & 1];
        a.next = parts[~i & 1];
        a.a = g.steps[3 * i];
        a.b = g.steps[3 * i + 1];
        a.c = g.steps[3 * i + 2];
        a.out = g.out;
        if (i == g.n_steps - 1) run<false, true, void>(a, grid, s);
        else run<false, false, void>(a, grid, s);
    }
    return pfk_internal_launched("k_orth_narrow");
}
