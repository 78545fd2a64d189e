// moe_mm.hip — products grouped by expert on gfx950 (include/prefree_moe.h): y[s] = x[row(s)] w[e(s)]^T and its two
// gradients, for f16, bf16 and 4-bit blocks, on the matrix cores.
#include "moe_common.hpp"
#include "moe_launch.hpp"
#include "prefree_moe_kernels.h"

namespace {

using namespace pfmoe;

// What the three products have in common: C[m][n] = sum over k of P[m][k] Q[n][k], tile by tile.  Both operands
// are staged through LDS in tiles of 64 bytes of k per row (32 elements of 16 bits, 128 of 4 bits).
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

// Loads straight to LDS go through buffer descriptors: 32-bit offsets from a base in scalar registers, and a lane whose
// offset lies behind the operand writes zeros, which is how k is cut off at its end.  (The other form, global_load_lds,
// counts as a flat access: the compiler then waits for every LDS read under way wherever it waits for one.)
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr unsigned kOutside = 0xffffffffu;       // an offset behind every operand
constexpr unsigned long long kBufferMax = 0xfffff000ull;

__device__ __forceinline__ Buffer buffer_of(const char *base, unsigned long long bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)(unsigned)(bytes < kBufferMax ? bytes : kBufferMax), 0x00020000);
}

__device__ __forceinline__ void to_lds16(Buffer from, unsigned lane_offset, unsigned offset, char *dst)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)dst, 16, (int)lane_offset,
                                             (int)offset, 0, 0);
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

// An operand whose k lies along its rows: a tile is ROWS rows of 64 bytes.  The 16-byte piece c of row r lies at place
// c ^ ((r >> 1) & 3) of the row, so that eight lanes that read one piece of eight rows touch each bank of 128 bytes once.
template <int ROWS, int THREADS, bool ALIGNED>
struct Along {
    static constexpr int kBytes = ROWS * 64;
    static constexpr int kLoads = ROWS * 4 / THREADS;
    Buffer from;                          // ALIGNED: the operand, and this thread's pieces of its rows in the first tile
    unsigned at[ALIGNED ? kLoads : 1];
    const char *row[ALIGNED ? 1 : kLoads];
    int piece;          // this thread's piece of its rows (the same for all its loads)
    int k_pieces, k;
    i32x4 held[ALIGNED ? 1 : kLoads];

    static __device__ __forceinline__ int tile_row(int i) { return i * (THREADS / 4) + (int)(threadIdx.x >> 2); }

    // row_of(r): the operand's row for row r of the tile
    template <typename F>
    __device__ __forceinline__ void init(const char *base, unsigned long long bytes, long long ld, F row_of, int k_, int per_piece)
    {
        piece = (threadIdx.x & 3) ^ ((threadIdx.x >> 3) & 3);
        k = k_;
        k_pieces = k_ / per_piece;
        if constexpr (ALIGNED) from = buffer_of(base, bytes);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const long long r = ld * row_of(tile_row(i));
            if constexpr (ALIGNED) at[i] = (unsigned)r + piece * 16;
            else row[i] = base + r;
        }
    }
    __device__ __forceinline__ void issue(int i, int t, char *lds)
    {
        const int c = t * 4 + piece;
        if constexpr (ALIGNED)
            to_lds16(from, c < k_pieces ? at[i] : kOutside, t * 64, lds + i * THREADS * 16 + (threadIdx.x & ~(kWave - 1)) * 16);
        else
            held[i] = load8_any(row[i], c * 8, k);
    }
    __device__ __forceinline__ void commit(char *lds)
    {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) *(i32x4 *)(lds + i * THREADS * 16 + threadIdx.x * 16) = held[i];
        }
    }
    // 16 rows from r0 (a multiple of 16): lane l has row l % 16, piece l / 16
    static __device__ __forceinline__ i32x4 fragment(const char *lds, int r0)
    {
        const int l = threadIdx.x & (kWave - 1);
        return *(const i32x4 *)(lds + r0 * 64 + (l & 15) * 64 + (((l >> 4) ^ ((l >> 1) & 3)) * 16));
    }
};

// An operand whose k lies across its rows: a tile is 32 rows of COLS columns (16 bits), read with the transposing LDS
// read, which hands a group of 16 lanes a block of 4 rows x 16 columns by columns.  The 32-byte unit u of row r lies
// at place u ^ f(r), f of bits 0, 1 and 3 of r, so that the eight rows which half a wave reads lie in other banks.
template <int COLS, int THREADS, bool ALIGNED>
struct Across {
    static constexpr int kBytes = COLS * 64;
    static constexpr int kLoads = COLS * 4 / THREADS;
    static constexpr int kPieces = COLS / 8;             // 16-byte pieces a row
    static constexpr int kStride = THREADS / kPieces;    // rows a load of all threads covers
    static constexpr int kWaveRows = kWave / kPieces;    // and of one wave
    static_assert(kPieces >= 16 && kPieces <= 32 && kStride % 8 == 0, "see f");
    Buffer from;         // ALIGNED
    const char *base;
    long long ld;
    int col[2], cols;    // this thread's first column in loads of even and odd number, and the columns there are
    int k;
    i32x4 held[ALIGNED ? 1 : kLoads];

    static __device__ __forceinline__ int f(int r) { return (r & 3) | ((r >> 1) & 4); }
    static __device__ __forceinline__ int tile_row(int i) { return i * kStride + (int)threadIdx.x / kPieces; }

    // columns from c0 of rows of `cols_` columns
    __device__ __forceinline__ void init(const char *base_, unsigned long long bytes, long long ld_, int c0, int cols_, int k_)
    {
        if constexpr (ALIGNED) from = buffer_of(base_, bytes);
        const int place = threadIdx.x % kPieces, r = threadIdx.x / kPieces;
        cols = cols_;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            col[i] = c0 + (((place >> 1) ^ f(i * kStride + r)) * 2 + (place & 1)) * 8;
            if (ALIGNED && col[i] >= cols) col[i] = 0;   // columns behind the end: any, their results are not stored
        }
        base = base_;
        ld = ld_;
        k = k_;
    }
    // Load i of tile t; with GATHER its rows are numbered by `rows` (see lookup), else by k itself.
    template <bool GATHER>
    __device__ __forceinline__ void issue(int i, int t, char *lds, int rows)
    {
        const int r = t * 32 + tile_row(i);
        const int at = GATHER ? __shfl(rows, i * kWaveRows + (int)(threadIdx.x & (kWave - 1)) / kPieces) : r;
        if constexpr (ALIGNED) {
            const unsigned first = GATHER ? (unsigned)at * (unsigned)ld : (unsigned)tile_row(i) * (unsigned)ld;
            to_lds16(from, r < k ? first + 2 * col[i & 1] : kOutside, GATHER ? 0 : (unsigned)(t * 32) * (unsigned)ld,
                     lds + i * THREADS * 16 + (threadIdx.x & ~(kWave - 1)) * 16);
        } else {
            held[i] = i32x4{0, 0, 0, 0};
            if (r < k && col[i & 1] < cols) held[i] = load8_any(base + ld * at, col[i & 1], cols);
        }
    }
    // The k of tile t whose row lane l looks up for its wave: load l / kWaveRows, row l % kWaveRows of the wave's.
    static __device__ __forceinline__ int lookup(int t)
    {
        const int l = (threadIdx.x & (kWave - 1)) % (kLoads * kWaveRows), w = threadIdx.x / kWave;
        return t * 32 + l / kWaveRows * kStride + w * kWaveRows + l % kWaveRows;
    }
    __device__ __forceinline__ void commit(char *lds)
    {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) *(i32x4 *)(lds + i * THREADS * 16 + threadIdx.x * 16) = held[i];
        }
    }
    // 16 columns from c0 (a multiple of 16): lane l has column l % 16, rows 8 (l / 16) .. +7
    static __device__ __forceinline__ i32x4 fragment(const char *lds, int c0)
    {
        const int l = threadIdx.x & (kWave - 1), g = l >> 4, q = (l >> 2) & 3, part = l & 3;
        const int unit = (c0 / 16) ^ (q | ((g & 1) << 2));
        const char *at = lds + (g * 8 + q) * (COLS * 2) + unit * 32 + part * 8;
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

// The four scale bytes of each row of a tile of either operand, by way of registers (scale rows have any alignment):
// thread r takes row r, those of the rows operand first.
struct Scales {
    const unsigned char *row;
    unsigned held;

    // whether tile t has all its scales, and loading them is one load
    static __device__ __forceinline__ bool whole(int t, int blocks) { return t * 4 + 4 <= blocks; }
    __device__ __forceinline__ void issue(int t, int blocks)
    {
        if (whole(t, blocks)) {
            __builtin_memcpy(&held, row + t * 4, 4);
        } else {
            held = 0x7f7f7f7fu;   // 1 where the codes are zeros behind the row's end
            for (int b = 0; t * 4 + b < blocks; ++b) held = (held & ~(0xffu << 8 * b)) | (unsigned)row[t * 4 + b] << 8 * b;
        }
    }
    __device__ __forceinline__ void commit(char *lds) { *(unsigned *)(lds + threadIdx.x * 4) = held; }
    // the scale of this lane's row of 16 from r0 and piece
    static __device__ __forceinline__ int fragment(const char *lds, int r0)
    {
        const int l = threadIdx.x & (kWave - 1);
        return *(const unsigned char *)(lds + (r0 + (l & 15)) * 4 + (l >> 4));
    }
};

// Waits until at most LOADS of this wave's loads to LDS are under way and all its LDS reads are done, then for the
// other waves.  (__syncthreads() would wait for every load.)
template <int LOADS>
__device__ __forceinline__ void wait_and_meet()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
}

// T: f16 or bf16 of the results; FP4: 4-bit operands
template <typename T, bool FP4, int MODE, int ACT, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void k_mm(const Args a)
{
    constexpr int THREADS = WM * WN * 64;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    typedef typename std::conditional<MODE == kDw, Across<BM, THREADS, ALIGNED>, Along<BM, THREADS, ALIGNED>>::type P;
    typedef typename std::conditional<MODE == kFwd, Along<BN, THREADS, ALIGNED>, Across<BN, THREADS, ALIGNED>>::type Q;
    constexpr int SCALES = P::kBytes + Q::kBytes;   // where a tile's scales lie
    constexpr int SLOT = SCALES + (FP4 ? (BM + BN) * 4 : 0);
    static_assert(!FP4 || BM + BN == THREADS, "see Scales");
    __shared__ __align__(1024) char lds[4][SLOT];

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
    const int steps = FP4 ? (k + 127) / 128 : (k + 31) / 32;
    const int m0 = t.m * BM, count = t.end - t.begin;
    // Row of w that row r of the tile stands for.  Under SwiGLU rows of the gate and of the rest take turns of 16, so
    // that a wave holds both.
    const auto weight_row = [&](int r) {
        if constexpr (ACT) return min(t.n * OUT_N + r / 32 * 16 + r % 16, a.n - 1) + (r / 16 % 2) * a.n;
        else return min(t.n * BN + r, a.n - 1);
    };
    const auto slot_row = [&](int r) { return row_of_slot(a, t.begin + min(m0 + r, count - 1)); };
    P p;
    Q q;
    Scales scales;
    int rows = 0;   // kDw: x's rows of the next tile to be loaded
    if constexpr (MODE == kDw) {
        p.init(a.p + a.ld_p * t.begin, a.ld_p * k, a.ld_p, m0, a.m, k);
        q.init(a.q, a.ld_q * a.p_rows, a.ld_q, t.n * BN, a.n, k);
        if (k > 0) rows = row_of_slot(a, t.begin + min(Q::lookup(0), k - 1));
    } else {
        p.init(a.p, a.ld_p * a.p_rows, a.ld_p, slot_row, k, FP4 ? 32 : 8);
        if constexpr (MODE == kFwd) q.init(a.q + a.q_expert * t.e, a.q_expert, a.ld_q, weight_row, k, FP4 ? 32 : 8);
        else q.init(a.q + a.q_expert * t.e, a.q_expert, a.ld_q, t.n * BN, a.n, k);
    }
    if constexpr (FP4) {
        const long long blocks = k / 32;
        if (tid < BM) scales.row = a.p_scales + blocks * slot_row(tid);
        else scales.row = a.q_scales + blocks * ((ACT ? 2LL : 1LL) * a.n * t.e + weight_row(tid - BM));
    }
    constexpr int LOADS = P::kLoads + Q::kLoads;   // of a tile, by each thread
    int now = 0;
    // load i of tile s
    const auto issue = [&](int i, int s, char *to) {
        if (i == 0) {
            if constexpr (MODE == kDw) {   // looked up before the loads, so that waiting for it does not wait for them
                now = rows;
                rows = row_of_slot(a, t.begin + min(Q::lookup(s + 1), k - 1));
            }
        }
        if (i < P::kLoads) {
            if constexpr (MODE == kDw) p.template issue<false>(i, s, to, 0);
            else p.issue(i, s, to);
        } else {
            if constexpr (MODE == kFwd) q.issue(i - P::kLoads, s, to + P::kBytes);
            else q.template issue<MODE == kDw>(i - P::kLoads, s, to + P::kBytes, now);
        }
    };
    const auto commit = [&](char *to) {   // what came by way of registers
        p.commit(to);
        q.commit(to + P::kBytes);
    };

    // A wave's rows are every WM-th block of 16 of the tile, its columns FN blocks side by side.
    const auto read_x = [&](const char *from, int i) { return P::fragment(from, (i * WM + wm) * 16); };
    const auto read_w = [&](const char *from, int j) { return Q::fragment(from + P::kBytes, (wn * FN + j) * 16); };
    const auto scale_x = [&](const char *from, int i) { return FP4 ? Scales::fragment(from + SCALES, (i * WM + wm) * 16) : 0; };
    const auto scale_w = [&](const char *from, int j) { return FP4 ? Scales::fragment(from + SCALES, BM + (wn * FN + j) * 16) : 0; };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    // Four tiles of k in LDS.  While tile s is multiplied its rows' fragments are read two ahead and the columns'
    // fragments of tile s+1 beside them, so that the matrix cores find their operands in registers; tile s+3 is on its
    // way into the place of tile s-1, which every wave has left.  Two tiles of loads may be under way at the meeting
    // of the waves, which only waits for tile s+2.  (The places are told apart as restricted pointers: otherwise the
    // compiler waits for all loads to LDS before each transposing read.)
    i32x4 x[4], w[FN], w_next[FN];
    int xs[4], ws[FN], ws_next[FN];
    const auto step = [&](int s, char *__restrict__ fill, const char *__restrict__ here, const char *__restrict__ next) {
        if constexpr (FP4) {   // a tile further ahead, since their loads end in a register
            scales.commit(fill + SCALES);
            scales.issue(s + 4, k / 32);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int l = i * LOADS / FM; l < (i + 1) * LOADS / FM; ++l) issue(l, s + 3, fill);
            const char *from = i + 2 < FM ? here : next;
            x[(i + 2) % 4] = read_x(from, (i + 2) % FM);
            xs[(i + 2) % 4] = scale_x(from, (i + 2) % FM);
#pragma unroll
            for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j) {
                w_next[j] = read_w(next, j);
                ws_next[j] = scale_w(next, j);
            }
            // reads and loads stay ahead of these products (mask: only address arithmetic may pass; it
            // would let the scaled products pass too)
            __builtin_amdgcn_sched_barrier(FP4 ? 0 : 0x6);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if constexpr (FP4) {
                    const i32x8 A = {w[j][0], w[j][1], w[j][2], w[j][3], 0, 0, 0, 0};
                    const i32x8 B = {x[i % 4][0], x[i % 4][1], x[i % 4][2], x[i % 4][3], 0, 0, 0, 0};
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc[i][j], 4, 4, 0, ws[j], 0, xs[i % 4]);
                } else {
                    acc[i][j] = mfma<T>(w[j], x[i % 4], acc[i][j]);
                }
            }
            __builtin_amdgcn_sched_barrier(FP4 ? 0 : 0x6);
        }
        __builtin_amdgcn_sched_barrier(0);
        commit(fill);
        if (FP4 && Scales::whole(s + 4, k / 32)) wait_and_meet<LOADS + 1>();   // the scales' load as well
        else wait_and_meet<ALIGNED ? LOADS : 0>();
        __builtin_amdgcn_sched_barrier(0);
    };
    if (steps > 0) {
#pragma unroll
        for (int s = 0; s < 3; ++s) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) issue(i, s, lds[s]);
            commit(lds[s]);
            if constexpr (FP4) {
                scales.issue(s, k / 32);
                scales.commit(lds[s] + SCALES);
            }
        }
        if constexpr (FP4) scales.issue(3, k / 32);
        wait_and_meet<ALIGNED ? LOADS : 0>();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = read_x(lds[0], i);
            xs[i] = scale_x(lds[0], i);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            w[j] = read_w(lds[0], j);
            ws[j] = scale_w(lds[0], j);
        }
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
            step(s, lds[(s + 3) & 3], lds[s & 3], lds[(s + 1) & 3]);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                w[j] = w_next[j];
                ws[j] = ws_next[j];
            }
        }
        // nothing may still be on its way to LDS when the workgroup ends
        wait_and_meet<0>();
    }

    // lane l holds row l % 16 of each block and four consecutive columns
    const int have = MODE == kDw ? a.m - m0 : count - m0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r = (i * WM + wm) * 16 + (lane & 15);
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

// whether `bytes` lie within the 32-bit offsets of a buffer descriptor
bool fits(long long rows, long long ld) { return (unsigned long long)rows * ld < kBufferMax; }

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
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->k % 8 == 0 && fits(g->p_rows, g->ld_p) && fits(1, a.q_expert);
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
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->n % 8 == 0 && g->k % 8 == 0 &&
                         fits(g->slots, g->ld_p) && fits(1, a.q_expert);
    return run<kDx, 0>(g, a, aligned, (hipStream_t)stream);
}

int pfk_moe_mm_dw(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.m = g->n;
    a.n = g->k;
    a.out_f32 = g->out_f32;
    a.wide = wide(g->out, g->ld_out, g->out_f32 ? 4 : 2);
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->n % 8 == 0 && g->k % 8 == 0 &&
                         fits(g->slots, g->ld_p) && fits(g->p_rows, g->ld_q);
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
