// moe_mm.hip — products grouped by expert on gfx950 (include/prefree_moe.h): y[s] = x[row(s)] w[e(s)]^T and its two
// gradients, for f16, bf16 and 4-bit blocks, on the matrix cores.
#include "moe_common.hpp"
#include "moe_launch.hpp"
#include "prefree_moe_kernels.h"

namespace {

using namespace pfmoe;

// What the three products have in common: C[m][n] = sum over k of P[m][k] Q[n][k], tile by tile.  Both operands
// are staged through LDS in tiles of 128 bytes of k per row (64 elements of 16 bits, 256 of 4 bits).
//   forward    m: slots of an expert (P: x, gathered)   n: rows of w                k: x's columns, both row by row
//   kDx        m: slots of an expert (P: dy)            n: columns of w             k: rows of w: Q lies across
//   kDw        m: columns of dy                         n: columns of x (gathered)  k: slots of an expert: both across
enum { kFwd = 0, kDx = 1, kDw = 2 };

struct Args {
    const char *p, *q;
    const unsigned char *p_scales, *q_scales;
    long long ld_p, ld_q, q_expert, ld_out, ld_pre;
    const int *rows, *offsets;
    int row_div, p_rows, experts, slots;
    int m, n, k;         // m only for kDw; n: results per row (the gate's half under SwiGLU)
    int out_f32, wide;   // wide: the output takes stores of four elements
    char *out, *pre;
};

// 16 zero bytes in global memory: what a lane loads whose k lies behind the operand's end.  (Loads that go straight
// to LDS cannot be masked per lane without leaving old bytes there.)
__device__ const i32x4 g_zero = {0, 0, 0, 0};

__device__ __forceinline__ void to_lds16(const char *src, char *dst)
{
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

template <typename T>
__device__ __forceinline__ f32x4 mfma(const i32x4 &a, const i32x4 &b, const f32x4 &c)
{
    if constexpr (__is_same(T, f16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The tile of workgroup `id`: expert, tile of rows, tile of columns.  The experts' tiles are counted from the offsets,
// 64 experts at a time over the lanes, in every wave by itself.  Workgroups reach the 8 XCDs in turn, so each XCD is
// given consecutive tiles (an eighth of those there are), whose operands then meet in its L2; inside an expert eight
// tiles of rows go side by side over the columns.
struct Tile {
    int e, m, n, begin, end;
};

template <int BM>
__device__ __forceinline__ bool find_tile(const Args &a, int nt, int id, Tile &t)
{
    const int lane = threadIdx.x & (kWave - 1);
    int total = 0, mine = 0, incl = 0, b = 0, e = 0;
    for (int base = 0; base < a.experts; base += kWave) {
        mine = 0;
        if (base + lane < a.experts) {
            expert_rows(a.offsets, base + lane, a.slots, b, e);
            mine = (e - b + BM - 1) / BM * nt;
        }
        incl = scan_wave(mine);
        total += __builtin_amdgcn_readlane(incl, kWave - 1);
    }
    const int chunk = (total + kXcds - 1) / kXcds;
    const int at = (id % kXcds) * chunk + id / kXcds;
    if (id / kXcds >= chunk || at >= total) return false;
    int before = 0;
    for (int base = 0; base < a.experts; base += kWave) {
        if (a.experts > kWave) {
            mine = 0;
            if (base + lane < a.experts) {
                expert_rows(a.offsets, base + lane, a.slots, b, e);
                mine = (e - b + BM - 1) / BM * nt;
            }
            incl = scan_wave(mine);
        }
        const unsigned long long past = __ballot(before + incl > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            t.e = base + l;
            t.begin = __builtin_amdgcn_readlane(b, l);
            t.end = __builtin_amdgcn_readlane(e, l);
            const int tiles = __builtin_amdgcn_readlane(mine, l);
            const int i = at - before - (__builtin_amdgcn_readlane(incl, l) - tiles);
            const int mt = tiles / nt, group = i / (8 * nt), rows = min(8, mt - group * 8), j = i - group * 8 * nt;
            t.m = group * 8 + j % rows;
            t.n = j / rows;
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, kWave - 1);
    }
    return false;
}

// Elements [at, at+8) of a row of `have` elements, zeros behind its end, from any alignment of two bytes.
__device__ __forceinline__ i32x4 load8_any(const char *row, int at, int have)
{
    i32x4 v = {0, 0, 0, 0};
    if (at + 8 <= have) {
        v = load16_any(row + 2LL * at);
    } else {
        unsigned short h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < have) h[i] = *(const unsigned short *)(row + 2LL * (at + i));
        __builtin_memcpy(&v, h, 16);
    }
    return v;
}

// An operand whose k lies along its rows: a tile is ROWS rows of 128 bytes.  The 16-byte piece c of row r lies at
// place c ^ ((r >> 1) & 7) of the row, so that the 16 lanes that read one piece of 16 rows touch each bank once.
template <int ROWS, int THREADS, bool ALIGNED>
struct Along {
    static constexpr int kBytes = ROWS * 128;
    static constexpr int kLoads = ROWS * 8 / THREADS;
    const char *row[kLoads];
    int piece;          // this thread's piece of its rows (the same for all its loads)
    int k_pieces, k;
    i32x4 held[ALIGNED ? 1 : kLoads];

    static __device__ __forceinline__ int tile_row(int i) { return i * (THREADS / 8) + (int)(threadIdx.x >> 3); }

    __device__ __forceinline__ void init(int k_, int per_piece)
    {
        piece = (threadIdx.x & 7) ^ ((threadIdx.x >> 4) & 7);
        k = k_;
        k_pieces = k_ / per_piece;
    }
    __device__ __forceinline__ void issue(int t, char *lds)
    {
        const int at = t * 8 + piece;
        if constexpr (ALIGNED) {
            const bool in = at < k_pieces;
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                to_lds16(in ? row[i] + 16LL * at : (const char *)&g_zero,
                         lds + i * THREADS * 16 + (threadIdx.x & ~(kWave - 1)) * 16);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) held[i] = load8_any(row[i], at * 8, k);
        }
    }
    __device__ __forceinline__ void commit(char *lds)
    {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) *(i32x4 *)(lds + i * THREADS * 16 + threadIdx.x * 16) = held[i];
        }
    }
    // 16 rows from r0 (a multiple of 16), step kk of 4 pieces: lane l has row l % 16, piece 4 kk + l / 16
    static __device__ __forceinline__ i32x4 fragment(const char *lds, int r0, int kk)
    {
        const int l = threadIdx.x & (kWave - 1);
        return *(const i32x4 *)(lds + r0 * 128 + (l & 15) * 128 + (((kk * 4 + (l >> 4)) ^ ((l >> 1) & 7)) * 16));
    }
};

// An operand whose k lies across its rows: a tile is 64 rows of COLS columns (16 bits), read with the transposing LDS
// read, which hands a group of 16 lanes a block of 4 rows x 16 columns by columns.  The 32-byte unit u of row r lies
// at place u ^ f(r), f of bits 0, 1 and 3 of r, so that the eight rows which half a wave reads lie in other banks.
template <int COLS, int THREADS, bool ALIGNED>
struct Across {
    static constexpr int kBytes = COLS * 128;
    static constexpr int kLoads = COLS * 8 / THREADS;
    static constexpr int kPieces = COLS / 8;             // 16-byte pieces a row
    static constexpr int kStride = THREADS / kPieces;    // rows a load of all threads covers
    static_assert(kPieces >= 16 && kStride % 16 == 0, "the swizzle repeats every 16 rows");
    const char *base;
    long long ld;
    int col, cols;       // this thread's first column, and the columns there are
    int k;
    i32x4 held[ALIGNED ? 1 : kLoads];

    static __device__ __forceinline__ int f(int r) { return (r & 3) | ((r >> 1) & 4); }
    static __device__ __forceinline__ int tile_row(int i) { return i * kStride + (int)threadIdx.x / kPieces; }

    // columns from c0 of rows of `cols_` columns
    __device__ __forceinline__ void init(const char *base_, long long ld_, int c0, int cols_, int k_)
    {
        const int place = threadIdx.x % kPieces, r = threadIdx.x / kPieces;
        col = c0 + (((place >> 1) ^ f(r)) * 2 + (place & 1)) * 8;
        cols = cols_;
        if (ALIGNED && col >= cols) col = 0;   // columns behind the end: any, their results are not stored
        base = base_;
        ld = ld_;
        k = k_;
    }
    // row_of(r): the operand's row for k = r < k
    template <typename F>
    __device__ __forceinline__ void issue(int t, char *lds, F row_of)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = t * 64 + tile_row(i);
            if constexpr (ALIGNED) {
                const char *src = (const char *)&g_zero;
                if (r < k) src = base + ld * row_of(r) + 2LL * col;
                to_lds16(src, lds + i * THREADS * 16 + (threadIdx.x & ~(kWave - 1)) * 16);
            } else {
                held[i] = i32x4{0, 0, 0, 0};
                if (r < k && col < cols) held[i] = load8_any(base + ld * row_of(r), col, cols);
            }
        }
    }
    __device__ __forceinline__ void commit(char *lds)
    {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) *(i32x4 *)(lds + i * THREADS * 16 + threadIdx.x * 16) = held[i];
        }
    }
    // 16 columns from c0 (a multiple of 16), step kk of 32 rows: lane l has column l % 16, rows 32 kk + 8 (l / 16) ..+7
    static __device__ __forceinline__ i32x4 fragment(const char *lds, int c0, int kk)
    {
        const int l = threadIdx.x & (kWave - 1), g = l >> 4, q = (l >> 2) & 3, part = l & 3;
        const int unit = (c0 / 16) ^ (q | ((g & 1) << 2));
        const char *at = lds + (kk * 32 + g * 8 + q) * (COLS * 2) + unit * 32 + part * 8;
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)at);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(at + 4 * COLS * 2));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        return i32x4{(int)a[0], (int)a[1], (int)b[0], (int)b[1]};
    }
};

template <typename T>
__device__ __forceinline__ void store4(char *row, int n, int have, bool wide, const f32x4 &v)
{
    T *out = (T *)row + n;
    if (wide && n + 4 <= have) {
        typename vec<T>::x4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = (T)v[i];
        *(typename vec<T>::x4 *)out = h;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < have) out[i] = (T)v[i];
    }
}

__device__ __forceinline__ void store4_f32(char *row, int n, int have, bool wide, const f32x4 &v)
{
    float *out = (float *)row + n;
    if (wide && n + 4 <= have) {
        *(f32x4 *)out = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < have) out[i] = v[i];
    }
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + __expf(-g)); }

__device__ __forceinline__ int row_of_slot(const Args &a, int s)
{
    if (!a.rows) return s;
    const int r = a.rows[s] / a.row_div;
    return (unsigned)r < (unsigned)a.p_rows ? r : 0;
}

// T: f16 or bf16 of the results; FP4: 4-bit operands
template <typename T, bool FP4, int MODE, int ACT, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void k_mm(const Args a)
{
    constexpr int THREADS = WM * WN * 64;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    typedef typename std::conditional<MODE == kDw, Across<BM, THREADS, ALIGNED>, Along<BM, THREADS, ALIGNED>>::type P;
    typedef typename std::conditional<MODE == kFwd, Along<BN, THREADS, ALIGNED>, Across<BN, THREADS, ALIGNED>>::type Q;
    __shared__ __align__(1024) char lds[2][P::kBytes + Q::kBytes];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    constexpr int OUT_N = ACT ? BN / 2 : BN;   // results of a tile's row
    const int nt = (a.n + OUT_N - 1) / OUT_N;
    Tile t;
    if constexpr (MODE == kDw) {
        const int mt = (a.m + BM - 1) / BM, all = a.experts * mt * nt, chunk = (all + kXcds - 1) / kXcds;
        const int at = (blockIdx.x % kXcds) * chunk + blockIdx.x / kXcds;
        if ((int)blockIdx.x / kXcds >= chunk || at >= all) return;
        t.e = at / (mt * nt);
        t.m = at % (mt * nt) % mt;
        t.n = at % (mt * nt) / mt;
        expert_rows(a.offsets, t.e, a.slots, t.begin, t.end);
    } else {
        if (!find_tile<BM>(a, nt, blockIdx.x, t)) return;
    }

    const int k = MODE == kDw ? t.end - t.begin : a.k;
    const int steps = FP4 ? (k + 255) / 256 : (k + 63) / 64;
    P p;
    Q q;
    const int m0 = t.m * BM, count = t.end - t.begin;
    if constexpr (MODE == kDw) {
        p.init(a.p + a.ld_p * t.begin, a.ld_p, m0, a.m, k);
        q.init(a.q, a.ld_q, t.n * BN, a.n, k);
    } else {
        p.init(k, FP4 ? 32 : 8);
#pragma unroll
        for (int i = 0; i < P::kLoads; ++i)
            p.row[i] = a.p + a.ld_p * row_of_slot(a, t.begin + min(m0 + P::tile_row(i), count - 1));
        if constexpr (MODE == kFwd) {
            q.init(k, FP4 ? 32 : 8);
#pragma unroll
            for (int i = 0; i < Q::kLoads; ++i) {
                const int r = Q::tile_row(i);
                int n;
                if constexpr (ACT) {  // rows of the gate and of the rest by turns of 16, so that a wave holds both
                    n = min(t.n * OUT_N + r / 32 * 16 + r % 16, a.n - 1) + (r / 16 % 2) * a.n;
                } else {
                    n = min(t.n * BN + r, a.n - 1);
                }
                q.row[i] = a.q + a.q_expert * t.e + a.ld_q * n;
            }
        } else {
            q.init(a.q + a.q_expert * t.e, a.ld_q, t.n * BN, a.n, k);
        }
    }
    const auto own_row = [&](int r) { return (long long)r; };
    const auto slot_row = [&](int r) { return (long long)row_of_slot(a, t.begin + r); };
    const auto issue = [&](int s, char *to) {
        if constexpr (MODE == kDw) p.issue(s, to, own_row); else p.issue(s, to);
        if constexpr (MODE == kFwd) q.issue(s, to + P::kBytes);
        else if constexpr (MODE == kDx) q.issue(s, to + P::kBytes, own_row);
        else q.issue(s, to + P::kBytes, slot_row);
    };

    // 4-bit operands: the scale rows of this lane's fragments' rows
    const unsigned char *ps[FP4 ? FM : 1], *qs[FP4 ? FN : 1];
    if constexpr (FP4) {
        const long long blocks = k / 32;
#pragma unroll
        for (int i = 0; i < FM; ++i)
            ps[i] = a.p_scales + blocks * row_of_slot(a, t.begin + min(m0 + (wm * FM + i) * 16 + (lane & 15), count - 1));
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int r = (wn * FN + j) * 16 + (lane & 15);
            int n;
            if constexpr (ACT) n = min(t.n * OUT_N + r / 32 * 16 + r % 16, a.n - 1) + (r / 16 % 2) * a.n;
            else n = min(t.n * BN + r, a.n - 1);
            qs[j] = a.q_scales + blocks * ((ACT ? 2LL : 1LL) * a.n * t.e + n);
        }
    }

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    if (steps > 0) {
        issue(0, lds[0]);
        p.commit(lds[0]);
        q.commit(lds[0] + P::kBytes);
    }
    for (int s = 0; s < steps; ++s) {
        __syncthreads();
        char *now = lds[s & 1], *next = lds[(s & 1) ^ 1];
        if (s + 1 < steps) issue(s + 1, next);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            i32x4 x[FM], w[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) x[i] = P::fragment(now, (wm * FM + i) * 16, kk);
#pragma unroll
            for (int j = 0; j < FN; ++j) w[j] = Q::fragment(now + P::kBytes, (wn * FN + j) * 16, kk);
            if constexpr (FP4) {
                const int block = s * 8 + kk * 4 + (lane >> 4), blocks = k / 32;
                int xs[FM], ws[FN];
#pragma unroll
                for (int i = 0; i < FM; ++i) xs[i] = block < blocks ? ps[i][block] : 127;
#pragma unroll
                for (int j = 0; j < FN; ++j) ws[j] = block < blocks ? qs[j][block] : 127;
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        const i32x8 A = {w[j][0], w[j][1], w[j][2], w[j][3], 0, 0, 0, 0};
                        const i32x8 B = {x[i][0], x[i][1], x[i][2], x[i][3], 0, 0, 0, 0};
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc[i][j], 4, 4, 0, ws[j], 0, xs[i]);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mfma<T>(w[j], x[i], acc[i][j]);
            }
        }
        if (s + 1 < steps) {
            p.commit(next);
            q.commit(next + P::kBytes);
        }
    }

    // lane l holds row l % 16 of each block and four consecutive columns
    const int have = MODE == kDw ? a.m - m0 : count - m0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r = (wm * FM + i) * 16 + (lane & 15);
        if (r >= have) continue;
        const long long at = MODE == kDw ? (long long)t.e * a.m + m0 + r : (long long)t.begin + m0 + r;
        char *out = a.out + a.ld_out * at;
        if constexpr (ACT) {
            char *pre = a.pre ? a.pre + a.ld_pre * at : nullptr;
#pragma unroll
            for (int j = 0; j < FN; j += 2) {
                const int n = t.n * OUT_N + (wn * FN + j) * 8 + (lane >> 4) * 4;
                f32x4 h;
#pragma unroll
                for (int c = 0; c < 4; ++c) h[c] = silu(acc[i][j][c]) * acc[i][j + 1][c];
                store4<T>(out, n, a.n, a.wide, h);
                if (pre) {
                    store4<T>(pre, n, a.n, a.wide, acc[i][j]);
                    store4<T>(pre + 2LL * a.n, n, a.n, a.wide, acc[i][j + 1]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int n = t.n * BN + (wn * FN + j) * 16 + (lane >> 4) * 4;
                if (MODE == kDw && a.out_f32) store4_f32(out, n, a.n, a.wide, acc[i][j]);
                else store4<T>(out, n, a.n, a.wide, acc[i][j]);
            }
        }
    }
}

template <typename T, bool FP4, int MODE, int ACT, int BM, int BN, int WM, int WN, bool ALIGNED>
int launch(const Args &a, hipStream_t stream)
{
    const long long out_n = ACT ? BN / 2 : BN, nt = (a.n + out_n - 1) / out_n;
    long long tiles;
    if (MODE == kDw) tiles = (long long)a.experts * ((a.m + BM - 1) / BM) * nt;
    else tiles = ((long long)a.slots / BM + (a.experts < a.slots ? a.experts : a.slots)) * nt;
    const long long grid = (tiles + kXcds - 1) / kXcds * kXcds;
    if (grid > 0x7fffffffLL) return pfk_internal_fail(PF_ERR_UNSUPPORTED, "grouped product: too many tiles");
    k_mm<T, FP4, MODE, ACT, BM, BN, WM, WN, ALIGNED><<<dim3((unsigned)grid), dim3(WM * WN * 64), 0, stream>>>(a);
    return pfk_internal_launched("k_mm");
}

template <typename T, bool FP4, int MODE, int ACT, bool ALIGNED>
int launch_size(const Args &a, hipStream_t stream)
{
    const long long rows = a.experts > 0 ? a.slots / a.experts : 0;  // an expert's, on average
    if (!ALIGNED || rows < 128) return launch<T, FP4, MODE, ACT, 128, 128, 2, 2, ALIGNED>(a, stream);
    return launch<T, FP4, MODE, ACT, 256, 256, 2, 4, ALIGNED>(a, stream);
}

bool lies16(const void *p, long long ld) { return ((uintptr_t)p | (unsigned long long)ld) % 16 == 0; }

template <int MODE, int ACT>
int run(const pfk_moe_mm_args *g, Args a, bool aligned, hipStream_t stream)
{
    if (g->dtype == PF_F16)
        return aligned ? launch_size<f16, false, MODE, ACT, true>(a, stream) : launch_size<f16, false, MODE, ACT, false>(a, stream);
    return aligned ? launch_size<bf16, false, MODE, ACT, true>(a, stream) : launch_size<bf16, false, MODE, ACT, false>(a, stream);
}

Args common(const pfk_moe_mm_args *g)
{
    Args a = {};
    a.p = (const char *)g->p;
    a.q = (const char *)g->q;
    a.ld_p = g->ld_p;
    a.ld_q = g->ld_q;
    a.rows = g->rows;
    a.row_div = g->row_div;
    a.p_rows = g->p_rows;
    a.offsets = g->offsets;
    a.experts = g->experts;
    a.slots = g->slots;
    a.out = (char *)g->out;
    a.ld_out = g->ld_out;
    a.pre = (char *)g->pre;
    a.ld_pre = g->ld_pre;
    return a;
}

// whether rows of `bytes` an element may be written four elements at a time
bool wide(const void *p, long long ld, long long bytes) { return ((uintptr_t)p | (unsigned long long)ld) % (4 * bytes) == 0; }

}  // namespace

extern "C" {

int pfk_moe_mm(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.n = g->n;
    a.k = g->k;
    const int each = g->act == PF_ACT_SWIGLU ? 2 : 1;
    a.q_expert = g->ld_q * g->n * each;
    a.wide = wide(g->out, g->ld_out, 2) && (!g->pre || (wide(g->pre, g->ld_pre, 2) && g->n % 4 == 0));
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->k % 8 == 0;
    hipStream_t s = (hipStream_t)stream;
    return g->act == PF_ACT_SWIGLU ? run<kFwd, 1>(g, a, aligned, s) : run<kFwd, 0>(g, a, aligned, s);
}

int pfk_moe_mm_dx(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.n = g->k;   // columns of w are the results, its rows are summed over
    a.k = g->n;
    a.q_expert = g->ld_q * g->n;
    a.wide = wide(g->out, g->ld_out, 2);
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->n % 8 == 0 && g->k % 8 == 0;
    return run<kDx, 0>(g, a, aligned, (hipStream_t)stream);
}

int pfk_moe_mm_dw(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.m = g->n;
    a.n = g->k;
    a.out_f32 = g->out_f32;
    a.wide = wide(g->out, g->ld_out, g->out_f32 ? 4 : 2);
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->n % 8 == 0 && g->k % 8 == 0;
    return run<kDw, 0>(g, a, aligned, (hipStream_t)stream);
}

int pfk_moe_mm_mx4(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.n = g->n;
    a.k = g->k;
    a.p_scales = (const unsigned char *)g->p_scales;
    a.q_scales = (const unsigned char *)g->q_scales;
    a.q_expert = g->ld_q * g->n * (g->act == PF_ACT_SWIGLU ? 2 : 1);
    a.wide = wide(g->out, g->ld_out, 2);
    hipStream_t s = (hipStream_t)stream;
    if (g->act == PF_ACT_SWIGLU)
        return g->dtype == PF_F16 ? launch_size<f16, true, kFwd, 1, true>(a, s) : launch_size<bf16, true, kFwd, 1, true>(a, s);
    return g->dtype == PF_F16 ? launch_size<f16, true, kFwd, 0, true>(a, s) : launch_size<bf16, true, kFwd, 0, true>(a, s);
}

}  // extern "C"
