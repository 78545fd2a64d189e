// moe_orth.hip — orthogonal updates on gfx950 (include/prefree_moe.h): X = G / |G|, then a few times
// X <- a X + (b A + c A A) X with A = X X^T, in 16-bit products on the matrix cores.
//
// X is carried in two f16 pieces, of which the products take the first.  What a rounding of X puts where G has nothing
// is multiplied by a in every step (3.4445^5 = 485), and so are G's small directions with it; in one piece the result of
// a momentum of rank n / 8 came out 1.5 to 4% off in f16 and 11 to 30% in bf16, in two 0.05 to 0.2% (64 to 1024 rows).
// With a X formed from both pieces the roundings of the first reach X by way of A and of B X alone, and there they are
// small beside what X has in the same directions.  A and B = b A + c A A are one f16 piece.
#include <algorithm>

#include "moe_tiles.hpp"

namespace {

using namespace pfmoe;

constexpr float kRest = 2048.0f;   // the second piece is held times this, where f16 has all its bits for it

// One product of all matrices of a batch; they lie one after the other, rows and columns padded with zeros to multiples of 32.
struct Product {
    const f16 *p, *q;       // rows operand, and columns operand
    int m, n, k;            // of a matrix
    int batch, first;
    float alpha, beta;      // results: alpha times the sums plus beta times what stands there
    const f16 *old, *old_rest;
    f16 *out, *rest;
};

// kSquare: out = alpha P P^T;  kPoly: out = alpha P P^T + beta old, P symmetric (both symmetric: the tiles on and under
// the diagonal, stored twice);  kApply: X' = beta X + P X, X and X' in two pieces, X read across its rows
enum { kSquare = 0, kPoly = 1, kApply = 2 };

// Transposes 4 x 4 values of 16 bits in each four neighbouring lanes: lane r of them has four values of row r, and gets
// value r of rows 0 to 3.
__device__ __forceinline__ void transpose4(unsigned (&h)[2], int lane)
{
    const unsigned p0 = (unsigned)pfdev::dpp<pfdev::kDppXor1>(h[0]), p1 = (unsigned)pfdev::dpp<pfdev::kDppXor1>(h[1]);
    // bytes 0 to 3 are the second argument's, 4 to 7 the first's
    const unsigned pick = lane & 1 ? 0x03020706 : 0x05040100;
    const unsigned n0 = __builtin_amdgcn_perm(p0, h[0], pick);
    const unsigned n1 = __builtin_amdgcn_perm(p1, h[1], pick);
    const unsigned q0 = (unsigned)pfdev::dpp<pfdev::kDppXor2>(n0), q1 = (unsigned)pfdev::dpp<pfdev::kDppXor2>(n1);
    h[0] = lane & 2 ? q1 : n0;
    h[1] = lane & 2 ? n1 : q0;
}

__device__ __forceinline__ unsigned pair_of(float a, float b)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef f16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2{a, b}), h2));
}

template <int KIND, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void k_orth(const Product a)
{
    constexpr int THREADS = WM * WN * 64, FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Along<BM, THREADS, true> P;
    typedef typename std::conditional<KIND == kApply, Across<BN, THREADS, true>, Along<BN, THREADS, true>>::type Q;
    constexpr int SLOT = P::kBytes + Q::kBytes, LOADS = P::kLoads + Q::kLoads;
    __shared__ __align__(1024) char lds[4][SLOT];
    static_assert(KIND == kApply || BM == BN, "tiles under the diagonal");

    const int wave = wave_id(), lane = threadIdx.x & (kWave - 1), wm = wave / WN, wn = wave % WN;
    const int mt = (a.m + BM - 1) / BM, nt = (a.n + BN - 1) / BN, each = KIND == kApply ? mt * nt : mt * (mt + 1) / 2;
    const int id = a.first + blockIdx.x, all = a.batch * each, chunk = (all + kXcds - 1) / kXcds;
    const int at = id % kXcds * chunk + id / kXcds;
    if (id / kXcds >= chunk || at >= all) return;
    const int matrix = at / each, t = at % each;
    int tm, tn;
    if constexpr (KIND == kApply) {
        const int group = t / (8 * nt), side = min(8, mt - group * 8), j = t - group * 8 * nt;
        tm = group * 8 + j % side;
        tn = j / side;
    } else {
        tm = (int)((__builtin_sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
        while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
        while (tm * (tm + 1) / 2 > t) --tm;
        tn = t - tm * (tm + 1) / 2;
    }
    const int m0 = tm * BM, n0 = tn * BN, k = a.k;
    P p;
    Q q;
    {
        const char *base = (const char *)(a.p + (long long)matrix * a.m * k);
        p.init(base, 2ull * a.m * k, 2LL * k, [&](int r) { return min(m0 + r, a.m - 1); }, k, 8);
    }
    if constexpr (KIND == kApply) {
        const char *base = (const char *)(a.q + (long long)matrix * k * a.n);
        q.init(base, 2ull * k * a.n, 2LL * a.n, n0, a.n, k);
    } else {
        const char *base = (const char *)(a.q + (long long)matrix * a.m * k);
        q.init(base, 2ull * a.m * k, 2LL * k, [&](int r) { return min(n0 + r, a.m - 1); }, k, 8);
    }
    const auto issue = [&](int i, int s, char *to) {
        if (i < P::kLoads) p.issue(i, s, to);
        else if constexpr (KIND == kApply) q.template issue<false>(i - P::kLoads, s, to + P::kBytes, 0);
        else q.issue(i - P::kLoads, s, to + P::kBytes);
    };
    const auto read_x = [&](const char *from, int i) { return P::fragment(from, (i * WM + wm) * 16); };
    const auto read_w = [&](const char *from, int j) { return Q::fragment(from + P::kBytes, (wn * FN + j) * 16); };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    i32x4 x[4], w[2][FN];
    // Four tiles of k in LDS, as k_mm has them: fragments are read ahead of the products, the columns' of the next tile
    // beside this one's, and three tiles are on their way.
    const auto step = [&](int s, char *__restrict__ fill, const char *__restrict__ here, const char *__restrict__ next) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const char *from = i + 2 < FM ? here : next;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                acc[i][j] = mfma<f16>(w[0][j], x[i % 4], acc[i][j]);
                if (j == 0) x[(i + 2) % 4] = read_x(from, (i + 2) % FM);
                if (j == 1) {
#pragma unroll
                    for (int c = i * FN / FM; c < (i + 1) * FN / FM; ++c) w[1][c] = read_w(next, c);
                }
                if (j == FN / 2) {
#pragma unroll
                    for (int l = i * LOADS / FM; l < (i + 1) * LOADS / FM; ++l) issue(l, s + 3, fill);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        wait_and_meet<LOADS>();
        __builtin_amdgcn_sched_barrier(0);
    };
    const int steps = k / 32;
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) issue(i, s, lds[s]);
    wait_and_meet<LOADS>();
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = read_x(lds[0], i);
#pragma unroll
    for (int j = 0; j < FN; ++j) w[0][j] = read_w(lds[0], j);
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        step(s, lds[(s + 3) & 3], lds[s & 3], lds[(s + 1) & 3]);
#pragma unroll
        for (int j = 0; j < FN; ++j) w[0][j] = w[1][j];
    }
    wait_and_meet<0>();   // nothing may still be on its way to LDS when the workgroup ends

    // Rows and columns are multiples of 32: blocks of 16 x 16 are there as a whole or not at all.
    const long long base = (long long)matrix * a.m * a.n;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r0 = m0 + (i * WM + wm) * 16, c0 = n0 + wn * FN * 16;
        if (r0 >= a.m) continue;
        const int r = r0 + (lane & 15), g = lane >> 4;
        if constexpr (KIND == kApply) {
            unsigned v[FN][4];
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) v[j][c] = __float_as_uint(acc[i][j][c]);
            gather_columns<FN>(v);
            const int c = c0 + g * 4 * FN;   // 4 FN columns from here, whole or not at all
            if (c >= a.n) continue;
            const long long to = base + (long long)r * a.n + c;
#pragma unroll
            for (int j = 0; j < FN; j += 2) {
                const f16x8 h = *(const f16x8 *)(a.old + to + 4 * j), l = *(const f16x8 *)(a.old_rest + to + 4 * j);
                f16x8 nh, nl;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float old = __builtin_fmaf((float)l[e], 1.0f / kRest, (float)h[e]);
                    const float y = __builtin_fmaf(a.beta, old, __uint_as_float(v[j + e / 4][e % 4]));
                    nh[e] = (f16)y;
                    nl[e] = (f16)((y - (float)nh[e]) * kRest);
                }
                *(f16x8 *)(a.out + to + 4 * j) = nh;
                *(f16x8 *)(a.rest + to + 4 * j) = nl;
            }
        } else {
            unsigned h[FN][2];
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                f32x4 y = acc[i][j];
                const int c = c0 + j * 16 + g * 4;
                if constexpr (KIND == kPoly) {
                    typedef f16 f16x4 __attribute__((ext_vector_type(4)));
                    f16x4 o = f16x4{0, 0, 0, 0};
                    if (c < a.n) o = *(const f16x4 *)(a.old + base + (long long)r * a.n + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(a.alpha, y[e], a.beta * (float)o[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] *= a.alpha;
                }
                h[j][0] = pair_of(y[0], y[1]);
                h[j][1] = pair_of(y[2], y[3]);
            }
            if (tm != tn) {
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

// ---- into the two pieces, and out of them --------------------------------------------------------------------------

constexpr int kParts = PFK_ORTH_PARTS;   // sums of squares of a matrix, at most

// Sums of squares of `per` rows each, in 64 bits: no element is too large or too small for its square.
template <typename T>
__global__ __launch_bounds__(256) void k_orth_norm(const T *g, long long ld, int rows, int columns, int per, double *sums)
{
    __shared__ double part[4];
    const int begin = blockIdx.x * per, end = min(rows, begin + per);
    const T *from = g + (long long)blockIdx.y * rows * ld;
    double sum = 0;
    for (int r = begin; r < end; ++r)
        for (int c = threadIdx.x; c < columns; c += 256) {
            const double v = (double)(float)from[ld * r + c];
            sum = __builtin_fma(v, v, sum);
        }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) sums[(long long)blockIdx.y * gridDim.x + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// The pieces of scale G / |G|, or of its transpose, in [m][n] with zeros behind the matrix; 64 x 64 elements a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void k_orth_pieces(const T *g, long long ld, int rows, int columns, int transposed, const double *sums, int parts,
                                                     float scale, int m, int n, f16 *x, f16 *rest)
{
    __shared__ float tile[64][65];
    const double *mine = sums + (long long)blockIdx.z * parts;
    double sum = 0;
    for (int i = 0; i < parts; ++i) sum += mine[i];
    // no number for a matrix that holds none; zeros stay zeros
    const double by = !(sum < INFINITY) ? (double)NAN : sum > 0 ? scale / __builtin_sqrt(sum) : 0.0;
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;   // of X
    const T *from = g + (long long)blockIdx.z * rows * ld;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = wave; i < 64; i += 4) {
        const int r = transposed ? c0 + i : r0 + i, c = transposed ? r0 + lane : c0 + lane;
        float v = 0;
        if (r < rows && c < columns) v = (float)((double)(float)from[ld * r + c] * by);
        if (transposed) tile[lane][i] = v; else tile[i][lane] = v;
    }
    __syncthreads();
    const long long base = (long long)blockIdx.z * m * n;
    for (int i = wave; i < 64; i += 4) {
        if (r0 + i >= m || c0 + lane >= n) continue;
        const float v = tile[i][lane];
        const f16 h = (f16)v;
        x[base + (long long)(r0 + i) * n + c0 + lane] = h;
        rest[base + (long long)(r0 + i) * n + c0 + lane] = (f16)((v - (float)h) * kRest);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_orth_out(const f16 *x, const f16 *rest, int m, int n, float scale, int transposed, T *out, long long ld,
                                                  int rows, int columns)
{
    __shared__ float tile[64][65];
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;   // of X
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long base = (long long)blockIdx.z * m * n;
    for (int i = wave; i < 64; i += 4) {
        float v = 0;
        if (r0 + i < m && c0 + lane < n) {
            const long long at = base + (long long)(r0 + i) * n + c0 + lane;
            v = __builtin_fmaf((float)rest[at], 1.0f / kRest, (float)x[at]) * scale;
        }
        if (transposed) tile[lane][i] = v; else tile[i][lane] = v;
    }
    __syncthreads();
    T *to = out + (long long)blockIdx.z * rows * ld;
    for (int i = wave; i < 64; i += 4) {
        const int r = (transposed ? c0 : r0) + i, c = (transposed ? r0 : c0) + lane;
        if (r < rows && c < columns) to[ld * r + c] = (T)tile[i][lane];
    }
}

template <int KIND, int B, int WM, int WN>
int launch(Product a, hipStream_t s)
{
    const long long mt = (a.m + B - 1) / B, nt = (a.n + B - 1) / B, all = a.batch * (KIND == kApply ? mt * nt : mt * (mt + 1) / 2);
    const long long grid = (all + kXcds - 1) / kXcds * kXcds;
    if (grid > 0x7fffffffLL) return pfk_internal_fail(PF_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
    in_launches(grid, most_workgroups(WM * WN * 64), [&](long long first, long long count) {
        a.first = (int)first;
        k_orth<KIND, B, B, WM, WN><<<dim3((unsigned)count), dim3(WM * WN * 64), 0, s>>>(a);
    });
    return pfk_internal_launched("k_orth");
}

template <int KIND>
int product(const Product &a, hipStream_t s)
{
    const long long mt = (a.m + 255) / 256, nt = (a.n + 255) / 256, tiles = a.batch * (KIND == kApply ? mt * nt : mt * (mt + 1) / 2);
    if (tiles >= 256) return launch<KIND, 256, 2, 4>(a, s);
    return launch<KIND, 128, 2, 2>(a, s);
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

template <typename T>
void out_of_pieces(const f16 *x, const f16 *rest, int batch, int m, int n, float scale, int transposed, void *out, long long ld, int rows, int columns,
                   hipStream_t s)
{
    each_tile(batch, m, n, [&](dim3 grid, long long at) {
        k_orth_out<T><<<grid, dim3(256), 0, s>>>(x + at * m * n, rest + at * m * n, m, n, scale, transposed, (T *)out + at * rows * ld, ld, rows, columns);
    });
}

template <typename T>
void into_pieces(const void *g, long long ld, int batch, int rows, int columns, int transposed, double *sums, float scale, int m, int n, f16 *x,
                 f16 *rest, hipStream_t s)
{
    const int per = (rows + kParts - 1) / kParts, parts = (rows + per - 1) / per;
    k_orth_norm<T><<<dim3(parts, batch), dim3(256), 0, s>>>((const T *)g, ld, rows, columns, per, sums);
    each_tile(batch, m, n, [&](dim3 grid, long long at) {
        k_orth_pieces<T><<<grid, dim3(256), 0, s>>>((const T *)g + at * rows * ld, ld, rows, columns, transposed, sums + at * parts, parts, scale, m, n,
                                                    x + at * m * n, rest + at * m * n);
    });
}

}  // namespace

extern "C" int pfk_orthogonalize(const void *g, long long ld_g, int dtype, int batch, int rows, int columns, const float *steps, int n_steps, void *out,
                                 long long ld_out, int out_dtype, void *workspace, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    const int transposed = rows > columns;
    const int m = PFK_ORTH_SIDE(transposed ? columns : rows), n = PFK_ORTH_SIDE(transposed ? rows : columns);
    const long long xs = (long long)batch * m * n, as = (long long)batch * m * m;
    f16 *x[2] = {(f16 *)workspace, (f16 *)workspace + 2 * xs}, *a = (f16 *)workspace + 4 * xs, *b = a + as;
    double *sums = (double *)(b + as);
    float scale = 1;   // X is held times this: elements of about 1, and none over 2^11 where X has none over 2
    while (scale * scale * 4 <= n && scale < 1024) scale *= 2;
    if (dtype == PF_F32) into_pieces<float>(g, ld_g, batch, rows, columns, transposed, sums, scale, m, n, x[0], x[0] + xs, s);
    else if (dtype == PF_F16) into_pieces<f16>(g, ld_g, batch, rows, columns, transposed, sums, scale, m, n, x[0], x[0] + xs, s);
    else into_pieces<bf16>(g, ld_g, batch, rows, columns, transposed, sums, scale, m, n, x[0], x[0] + xs, s);
    for (int i = 0; i < n_steps; ++i) {
        f16 *from = x[i & 1], *to = x[~i & 1];
        Product square = {from, from, m, m, n, batch, 0, 1 / (scale * scale), 0, nullptr, nullptr, a, nullptr};
        Product poly = {a, a, m, m, m, batch, 0, steps[3 * i + 2], steps[3 * i + 1], a, nullptr, b, nullptr};
        Product apply = {b, from, m, n, m, batch, 0, 1, steps[3 * i], from, from + xs, to, to + xs};
        int st = product<kSquare>(square, s);
        if (st == PF_OK) st = product<kPoly>(poly, s);
        if (st == PF_OK) st = product<kApply>(apply, s);
        if (st != PF_OK) return st;
    }
    const f16 *last = x[n_steps & 1];
    if (out_dtype == PF_F16) out_of_pieces<f16>(last, last + xs, batch, m, n, 1 / scale, transposed, out, ld_out, rows, columns, s);
    else out_of_pieces<bf16>(last, last + xs, batch, m, n, 1 / scale, transposed, out, ld_out, rows, columns, s);
    return pfk_internal_launched("k_orth_out");
}
