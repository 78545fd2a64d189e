// moe_tiles.hpp — what the kernels of products grouped by expert share: operands' tiles in LDS, fragments for the
// matrix cores, results' stores.
#pragma once

#include <type_traits>

#include "moe_common.hpp"
#include "moe_launch.hpp"
#include "prefree_moe_kernels.h"

namespace pfmoe {

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
    int first;           // number of the launch's first workgroup (k_mm, k_mm_rows)
    unsigned div_mul;    // floor(v / row_div) = (v * div_mul >> 32) >> div_shift for 0 <= v < 2^31
    int div_shift;
    int m, n, k;         // m only for kDw; n: results per row (the gate's half under SwiGLU)
    int out_f32, wide;   // wide: the output's rows take stores of 16 bytes
    char *out, *pre;
};

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }

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

// Bytes from the first to the last of `rows` rows of `columns` 16-bit elements, ld bytes apart.
__device__ __forceinline__ unsigned long long span(long long ld, long long rows, long long columns)
{
    return rows > 0 ? (unsigned long long)(ld * (rows - 1) + 2 * columns) : 0;
}

__device__ __forceinline__ void to_lds16(Buffer from, unsigned lane_offset, unsigned offset, char *dst)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)dst, 16, (int)lane_offset,
                                             (int)offset, 0, 0);
}

__device__ __forceinline__ void to_lds4(Buffer from, unsigned lane_offset, void *dst)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)dst, 4, (int)lane_offset, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ f32x4 mfma(const i32x4 &a, const i32x4 &b, const f32x4 &c)
{
    if constexpr (__is_same(T, f16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma_fp4(const i32x4 &a, const i32x4 &b, const f32x4 &c, int a_scale, int b_scale)
{
    const i32x8 A = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, B = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, a_scale, 0, b_scale);
}

// Has the sums formed here: without it the compiler moves products of 4-bit blocks down past the meeting of the waves,
// since nothing before it uses them, where no LDS reads are left to go beside them (8192 tokens x 4 of 32 experts, 2048 ->
// 2 x 2048: 223 us, 216 so).
template <int ROWS, int FM, int FN>
__device__ __forceinline__ void formed(f32x4 (&acc)[FM][FN])
{
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[i][j]));
}

// Waits for all of this wave's loads.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// An operand whose k lies along its rows: a tile is ROWS rows of 64 bytes.  The 16-byte piece c of row r lies at place
// c ^ ((r >> 1) & 3) of the row, so that eight lanes that read one piece of eight rows touch each bank of 128 bytes once.
template <int ROWS, int THREADS, bool ALIGNED, int RING = 2>
struct Along {
    static constexpr int kBytes = ROWS * 64;
    static constexpr int kLoads = ROWS * 4 / THREADS;
    int piece;          // this thread's piece of its rows (the same for all its loads)
    int k_pieces, k;
    Buffer from;                          // ALIGNED: the operand, and this thread's pieces of its rows in the first tile
    unsigned at[ALIGNED ? kLoads : 1];
    // else words: sixteen lanes share a row of the tile, whose elements may start in the middle of one
    static constexpr int kWords = ALIGNED ? 1 : ROWS * 16 / THREADS;
    uintptr_t word[kWords], end;          // this thread's of the first tile; the operand's last
    unsigned shift[kWords];               // 2: by two bytes
    unsigned held[ALIGNED ? 1 : RING][kWords];   // of tile t at place t % RING

    static __device__ __forceinline__ int tile_row(int i) { return i * (THREADS / 4) + (int)(threadIdx.x >> 2); }

    // row_of(r): the operand's row for row r of the tile
    template <typename F>
    __device__ __forceinline__ void init(const char *base, unsigned long long bytes, long long ld, F row_of, int k_, int per_piece)
    {
        piece = (threadIdx.x & 3) ^ ((threadIdx.x >> 3) & 3);
        k = k_;
        k_pieces = k_ / per_piece;
        if constexpr (ALIGNED) from = buffer_of(base, bytes);
        else end = end_of(base, bytes);
        if constexpr (ALIGNED) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) at[i] = (unsigned)(ld * row_of(tile_row(i))) + piece * 16;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const uintptr_t p = (uintptr_t)(base + ld * row_of(word_row(i)));
                word[i] = word_of(p) + (threadIdx.x & 15) * 4;
                shift[i] = (unsigned)p & 2;
            }
        }
    }
    __device__ __forceinline__ void issue(int i, int t, char *lds)
    {
        to_lds16(from, t * 4 + piece < k_pieces ? at[i] : kOutside, t * 64, lds + i * THREADS * 16 + wave_id() * (kWave * 16));
    }
    static __device__ __forceinline__ int word_row(int i) { return i * (THREADS / 16) + (int)(threadIdx.x >> 4); }
    __device__ __forceinline__ bool whole(int t) const { return t * 32 + 32 <= k; }   // whether the rows have all of tile t
    __device__ __forceinline__ void fetch(int t, int place)
    {
        if (whole(t)) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) held[place][i] = load_word(word[i] + 64LL * t);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) held[place][i] = load_word(word[i] + 64LL * t < end ? word[i] + 64LL * t : end);
        }
    }
    // With one body of the loop all tiles move on a place, and the last one is free; else the stored tile's place is.
    __device__ __forceinline__ int freed(int bodies, int place)
    {
        if (bodies > 1) return place;
#pragma unroll
        for (int r = 0; r + 1 < RING; ++r)
#pragma unroll
            for (int i = 0; i < kWords; ++i) held[r][i] = held[r + 1][i];
        return RING - 1;
    }
    // A tile is stored when the first words of the one behind it are there.
    __device__ __forceinline__ void commit(char *lds, int t, int place)
    {
        const int j = threadIdx.x & 15, row = threadIdx.x >> 4;   // rows of the other words: multiples of 8 further
        char *to = lds + row * 64 + (((j >> 2) ^ ((row >> 1) & 3)) * 16) + (j & 3) * 4;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            // the next word: the next lane's, and of the last lane the first of the tile behind
            unsigned next = __builtin_amdgcn_update_dpp(0, held[place][i], 0x101, 0xf, 0xf, true);     // row_shl 1
            next = __builtin_amdgcn_update_dpp(next, held[(place + 1) % RING][i], 0x11f, 0xf, 0xf, false);         // row_shr 15
            unsigned v = __builtin_amdgcn_alignbyte(next, held[place][i], shift[i]);
            if (!whole(t)) v = kept_word(v, k - t * 32 - j * 2);
            *(unsigned *)(to + i * (THREADS / 16) * 64) = v;
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
    uintptr_t base, end;
    long long ld;
    bool inside;         // all of the tile's columns are there
    int col[2], cols;    // this thread's first column in loads of even and odd number, and the columns there are
    int k;
    unsigned shift[ALIGNED ? 1 : kLoads];
    Words held[ALIGNED ? 1 : kLoads];

    static __device__ __forceinline__ int f(int r) { return (r & 3) | ((r >> 1) & 4); }
    static __device__ __forceinline__ int tile_row(int i) { return i * kStride + (int)threadIdx.x / kPieces; }

    // columns from c0 of rows of `cols_` columns
    __device__ __forceinline__ void init(const char *base_, unsigned long long bytes, long long ld_, int c0, int cols_, int k_)
    {
        if constexpr (ALIGNED) from = buffer_of(base_, bytes);
        else end = end_of(base_, bytes);
        inside = c0 + COLS <= cols_;
        const int place = threadIdx.x % kPieces, r = threadIdx.x / kPieces;
        cols = cols_;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            col[i] = c0 + (((place >> 1) ^ f(i * kStride + r)) * 2 + (place & 1)) * 8;
            if (ALIGNED && col[i] >= cols) col[i] = 0;   // columns behind the end: any, their results are not stored
        }
        base = (uintptr_t)base_;
        ld = ld_;
        k = k_;
    }
    // Load i of tile t; with GATHER its rows are numbered by `rows` (see lookup), else by k itself.
    template <bool GATHER>
    __device__ __forceinline__ void issue(int i, int t, char *lds, int rows)
    {
        const int r = t * 32 + tile_row(i);
        const unsigned first = (unsigned)(GATHER ? given(rows, i) : tile_row(i)) * (unsigned)ld;
        to_lds16(from, r < k ? first + 2 * col[i & 1] : kOutside, GATHER ? 0 : (unsigned)(t * 32) * (unsigned)ld,
                 lds + i * THREADS * 16 + wave_id() * (kWave * 16));
    }
    static __device__ __forceinline__ int given(int rows, int i)
    {
        return __shfl(rows, i * kWaveRows + (int)(threadIdx.x & (kWave - 1)) / kPieces);
    }
    __device__ __forceinline__ bool whole(int t) const { return inside && t * 32 + 32 <= k; }
    template <bool GATHER>
    __device__ __forceinline__ void fetch(int t, int rows)
    {
        uintptr_t p[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            p[i] = base + ld * (GATHER ? given(rows, i) : t * 32 + tile_row(i)) + 2LL * col[i & 1];
            shift[i] = Words::shift_of(p[i]);
            p[i] = word_of(p[i]);
        }
        if (whole(t)) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) held[i].load(p[i], p[i] + 8 * shift[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) held[i].load_until(p[i], end);
        }
    }
    __device__ __forceinline__ void commit(char *lds, int t)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            i32x4 v = held[i].shifted(shift[i]);
            if (!whole(t)) v = Words::kept(v, t * 32 + tile_row(i) < k ? cols - col[i & 1] : 0);
            *(i32x4 *)(lds + i * THREADS * 16 + threadIdx.x * 16) = v;
        }
    }
    // The k of tile t whose row lane l looks up for its wave: load l / kWaveRows, row l % kWaveRows of the wave's.
    static __device__ __forceinline__ int lookup(int t)
    {
        const int l = (threadIdx.x & (kWave - 1)) % (kLoads * kWaveRows), w = threadIdx.x / kWave;
        return t * 32 + l / kWaveRows * kStride + w * kWaveRows + l % kWaveRows;
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

// Stores N results from column n of a row of `have`.  WHOLE: all there, and aligned for one store.
template <typename T, bool WHOLE, int N>
__device__ __forceinline__ void store(char *row, int n, int have, const T (&v)[N])
{
    T *out = (T *)row + n;
    if constexpr (WHOLE) {
        typedef T vec_t __attribute__((ext_vector_type(N)));
        vec_t h;
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = v[i];
        *(vec_t *)out = h;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (n + i < have) out[i] = v[i];
    }
}

// Lane l holds, of its row l % 16, four consecutive columns of each of N blocks of 16: those from 4 (l / 16).  Stores of
// these would cover 32 bytes of a row at a time.  The two lane-swapping instructions hand each group of 16 lanes 4 N
// consecutive columns instead, those from 4 N (l / 16), so that a store covers whole lines (N = 4) or halves.
// in: the blocks' four results each, as two registers of two; out: 4 N columns in order.
__device__ __forceinline__ void swap32(unsigned &a, unsigned &b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap16(unsigned &a, unsigned &b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
template <int N>
__device__ __forceinline__ void gather_columns(unsigned (&v)[N][2])
{
    static_assert(N == 1 || N == 2 || N == 4, "blocks");
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) swap32(v[i][c], v[i + N / 2][c]);
#pragma unroll
        for (int i = 0; i + 1 < N; i += 2) swap16(v[i][c], v[i + 1][c]);
    }
}

// Stores N blocks of 16 columns of a row from column n0, as T of 16 bits.  Whole waves only: lanes of rows that do not
// exist (`is` false) take part in the exchange.
template <typename T, bool WHOLE, int N>
__device__ __forceinline__ void store_columns(char *row, bool is, int n0, int have, const f32x4 (&v)[N], int lane)
{
    unsigned h[N][2];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // by pairs: one conversion instruction a pair to bf16, rather than one a value and two to join them
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int c = 0; c < 2; ++c)
            h[i][c] = __builtin_bit_cast(unsigned, __builtin_convertvector((f2{v[i][2 * c], v[i][2 * c + 1]}), t2));
    }
    gather_columns<N>(h);
    if (!is) return;
    constexpr int EACH = N == 1 ? 1 : 2;   // blocks a store
#pragma unroll
    for (int i = 0; i < N; i += EACH) {
        T x[4 * EACH];
        __builtin_memcpy(x, h[i], 8 * EACH);
        store<T, WHOLE, 4 * EACH>(row, n0 + (lane >> 4) * 4 * N + 4 * i, have, x);
    }
}

// The reciprocal instruction is within one unit in the last place, where the result is rounded to 16 bits; a division takes
// eight more instructions for each of a tile's results.
__device__ __forceinline__ float silu(float g) { return g * kUnder * __builtin_amdgcn_rcpf(inverse_sigmoid(g)); }

__device__ __forceinline__ int row_of_slot(const Args &a, int s)
{
    if (!a.rows) return s;
    const int r = a.rows[s] / a.row_div;
    return (unsigned)r < (unsigned)a.p_rows ? r : 0;
}

// The four scale bytes of each row of a tile of either operand, by way of registers (scale rows have any alignment):
// the rows operand's first, a thread takes every THREADS-th.
template <int ROWS, int THREADS>
struct Scales {
    static constexpr int kLoads = (ROWS + THREADS - 1) / THREADS;
    static constexpr int kBytes = kLoads * THREADS * 4;   // behind the rows' there may be some of no row
    const unsigned char *row[kLoads];
    unsigned held[kLoads];

    // whether tile t has all its scales, and loading them is kLoads loads
    static __device__ __forceinline__ bool whole(int t, int blocks) { return t * 4 + 4 <= blocks; }
    __device__ __forceinline__ void issue(int t, int blocks)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            if (whole(t, blocks)) {
                __builtin_memcpy(&held[i], row[i] + t * 4, 4);
            } else {
                held[i] = 0x7f7f7f7fu;   // 1 where the codes are zeros behind the row's end
                for (int b = 0; t * 4 + b < blocks; ++b)
                    held[i] = (held[i] & ~(0xffu << 8 * b)) | (unsigned)row[i][t * 4 + b] << 8 * b;
            }
        }
    }
    __device__ __forceinline__ void commit(char *lds)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) *(unsigned *)(lds + (threadIdx.x + i * THREADS) * 4) = held[i];
    }
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

// Stores a wave's results: FMV of its FM blocks of 16 rows (every WM-th of the tile's, of which `have` rows exist),
// FN blocks of 16 columns.  first: the tile's first row of the output, n0 its first column.
template <typename T, int MODE, int ACT, bool WHOLE, int FMV, int FM, int FN, int WM>
__device__ __forceinline__ void store_blocks(const Args &a, const f32x4 (&acc)[FM][FN], int wm, int wn, long long first, int have, int n0)
{
    int lane = threadIdx.x & (kWave - 1);
    asm volatile("" : "+v"(lane));   // addresses are formed here, not kept over the loop before
#pragma unroll
    for (int i = 0; i < FMV; ++i) {
        __builtin_amdgcn_sched_barrier(0);   // one block's results at a time
        if ((i * WM + wm) * 16 >= have) continue;
        const int r = (i * WM + wm) * 16 + (lane & 15);
        const bool is = r < have;
        char *out = a.out + a.ld_out * (first + r);
        if constexpr (ACT) {
            f32x4 h[FN / 2], gate[FN / 2], rest[FN / 2];
#pragma unroll
            for (int j = 0; j < FN / 2; ++j) {
                gate[j] = acc[i][2 * j];
                rest[j] = acc[i][2 * j + 1];
#pragma unroll
                for (int c = 0; c < 4; ++c) h[j][c] = silu(gate[j][c]) * rest[j][c];
            }
            const int n = n0 + wn * FN * 8;
            store_columns<T, WHOLE, FN / 2>(out, is, n, a.n, h, lane);
            if (a.pre) {
                char *pre = a.pre + a.ld_pre * (first + r);
                store_columns<T, WHOLE, FN / 2>(pre, is, n, a.n, gate, lane);
                store_columns<T, WHOLE, FN / 2>(pre + 2LL * a.n, is, n, a.n, rest, lane);
            }
        } else if (MODE == kDw && a.out_f32) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const float x[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                if (is) store<float, WHOLE, 4>(out, n0 + (wn * FN + j) * 16 + (lane >> 4) * 4, a.n, x);
            }
        } else {
            store_columns<T, WHOLE, FN>(out, is, n0 + wn * FN * 16, a.n, acc[i], lane);
        }
    }
}

template <typename T, int MODE, int ACT, int FMV, int FM, int FN, int WM, int OUT_N>
__device__ __forceinline__ void store_results(const Args &a, const f32x4 (&acc)[FM][FN], int wm, int wn, long long first, int have, int n0)
{
    if (a.wide && n0 + OUT_N <= a.n) store_blocks<T, MODE, ACT, true, FMV, FM, FN, WM>(a, acc, wm, wn, first, have, n0);
    else store_blocks<T, MODE, ACT, false, FMV, FM, FN, WM>(a, acc, wm, wn, first, have, n0);
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

// Launches kernel(args) for all `tiles`, whose workgroups number themselves from args.first on; they reach the XCDs in turn.
template <typename K>
int launch_tiles(K kernel, Args a, long long tiles, int threads, hipStream_t stream, const char *what)
{
    const long long grid = (tiles + kXcds - 1) / kXcds * kXcds;
    if (grid > 0x7fffffffLL) return pfk_internal_fail(PF_ERR_UNSUPPORTED, "grouped product: too many tiles");   // 32-bit numbers
    in_launches(grid, most_workgroups(threads), [&](long long first, long long count) {
        a.first = (int)first;
        kernel<<<dim3((unsigned)count), dim3(threads), 0, stream>>>(a);
    });
    return pfk_internal_launched(what);
}

// moe_mm_stream.hip
template <typename T, bool FP4, int MODE, int ACT>
int launch_stream(const Args &a, hipStream_t stream);

// moe_mm_rows.hip
template <typename T, bool FP4, int ACT, bool ALIGNED>
int launch_rows(const Args &a, hipStream_t stream);

}  // namespace pfmoe
