// moe_mm.hip — products grouped by expert on gfx950 (include/prefree_moe.h): y[s] = x[row(s)] w[e(s)]^T and its two
// gradients, for f16, bf16 and 4-bit blocks, on the matrix cores.
#include "moe_tiles.hpp"

namespace {

using namespace pfmoe;

// A workgroup a tile, for products too small for k_mm_stream and, by way of registers, for operands of any alignment.  8192
// rows of 16 experts, 2048 -> 2048, in 114 us against its 106; 311 tokens x 2 of 12, 1111 -> 717, in 22.6 us.  There one
// workgroup a CU waits for its loads: four tiles of k under way in registers (with two 25.7, with three 23.5); larger tiles
// have no registers for that.  An operand along k is loaded by single words, sixteen lanes a row, since the L1 takes one
// lane a cycle of wider loads that do not lie in their width (32764 slots of 32 experts, 2049 -> 1023, 128 x 128 tiles: 503
// with 16 bytes a lane, 435 so); an operand across k, with longer rows, by 16 bytes a lane (dw 540, by words 778).
// T: f16 or bf16 of the results; FORM: what the operands hold
template <typename T, int FORM, int MODE, int ACT, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void k_mm(const Args a)
{
    constexpr bool FP4 = FORM == kMx4;
    constexpr int THREADS = WM * WN * 64;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int RING = ALIGNED || MODE == kDw ? 1 : BM == 64 ? 4 : 2;   // tiles under way in registers
    constexpr int BODIES = BM == 64 ? RING : 1;   // of the loop; with one the ring's tiles move on from place to place
    typedef typename std::conditional<MODE == kDw, Across<BM, THREADS, ALIGNED>, Along<BM, THREADS, ALIGNED, RING>>::type P;
    typedef typename std::conditional<MODE == kFwd, Along<BN, THREADS, ALIGNED, RING>, Across<BN, THREADS, ALIGNED>>::type Q;
    typedef Scales<BM + BN, THREADS> S;
    constexpr int SCALES = P::kBytes + Q::kBytes;   // where a tile's scales lie
    constexpr int SLOT = SCALES + (FP4 ? S::kBytes : 0);
    __shared__ __align__(1024) char lds[4][SLOT];

    const int tid = threadIdx.x, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    constexpr int OUT_N = ACT ? BN / 2 : BN;   // results of a tile's row
    const int nt = (a.n + OUT_N - 1) / OUT_N;
    const int id = a.first + blockIdx.x;
    Tile t;
    if constexpr (MODE == kDw) {
        const int mt = (a.m + BM - 1) / BM, all = a.experts * mt * nt, chunk = (all + kXcds - 1) / kXcds;
        const int at = id % kXcds * chunk + id / kXcds;
        if (id / kXcds >= chunk || at >= all) return;
        t.e = at / (mt * nt);
        t.m = at % (mt * nt) % mt;
        t.n = at % (mt * nt) / mt;
        expert_rows(a.offsets, t.e, a.slots, t.begin, t.end);
    } else {
        if (!find_tile<BM>(a, nt, id, t)) return;
    }

    const int k = MODE == kDw ? t.end - t.begin : a.k;
    const int steps = (k + kPerTile<FORM> - 1) / kPerTile<FORM>;
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
    S scales;
    int rows = 0;   // kDw: x's rows of the next tile to be loaded
    if constexpr (MODE == kDw) {
        p.init(a.p + a.ld_p * t.begin, span(a.ld_p, k, a.m), a.ld_p, m0, a.m, k);
        q.init(a.q, span(a.ld_q, a.p_rows, a.n), a.ld_q, t.n * BN, a.n, k);
        if (k > 0) rows = row_of_slot(a, t.begin + min(Q::lookup(0), k - 1));
    } else {
        p.init(a.p, FORM != kHalf ? a.ld_p * a.p_rows : span(a.ld_p, a.p_rows, k), a.ld_p, slot_row, k, kPerPiece<FORM>);
        if constexpr (MODE == kFwd) q.init(a.q + a.q_expert * t.e, a.q_expert, a.ld_q, weight_row, k, kPerPiece<FORM>);
        else q.init(a.q + a.q_expert * t.e, a.q_expert, a.ld_q, t.n * BN, a.n, k);
    }
    if constexpr (FP4) {
        const long long blocks = k / 32;
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
            const int r = min(tid + i * THREADS, BM + BN - 1);
            scales.row[i] = r < BM ? a.p_scales + blocks * slot_row(r)
                                   : a.q_scales + blocks * ((ACT ? 2LL : 1LL) * a.n * t.e + weight_row(r - BM));
        }
    }
    constexpr int LOADS = P::kLoads + Q::kLoads;   // of a tile, by each thread
    int now = 0;
    const auto look_up = [&](int s) {   // before the loads, so that waiting for it does not wait for them
        if constexpr (MODE == kDw) {
            now = rows;
            rows = row_of_slot(a, t.begin + min(Q::lookup(s + 1), k - 1));
        }
    };
    // load i of tile s, straight to LDS
    const auto issue = [&](int i, int s, char *to) {
        if constexpr (ALIGNED) {
            if (i == 0) look_up(s);
            if (i < P::kLoads) {
                if constexpr (MODE == kDw) p.template issue<false>(i, s, to, 0);
                else p.issue(i, s, to);
            } else {
                if constexpr (MODE == kFwd) q.issue(i - P::kLoads, s, to + P::kBytes);
                else q.template issue<MODE == kDw>(i - P::kLoads, s, to + P::kBytes, now);
            }
        }
    };
    // By way of registers: tile s to LDS, and then what comes into its place, of an operand along k tile s + RING and of
    // one across it tile s + 1.
    const auto refill = [&](int s, int place) {
        if constexpr (!ALIGNED) {
            look_up(s + 1);
            if constexpr (MODE == kDw) p.template fetch<false>(s + 1, 0);
            else p.fetch(s + RING, p.freed(BODIES, place));
            if constexpr (MODE == kFwd) q.fetch(s + RING, q.freed(BODIES, place));
            else q.template fetch<MODE == kDw>(s + 1, now);
        }
    };
    const auto commit = [&](char *to, int s, int place) {
        if constexpr (!ALIGNED) {
            if constexpr (MODE == kDw) p.commit(to, s);
            else p.commit(to, s, place);
            if constexpr (MODE == kFwd) q.commit(to + P::kBytes, s, place);
            else q.commit(to + P::kBytes, s);
        }
    };

    // A wave's rows are every WM-th block of 16 of the tile, its columns FN blocks side by side.
    const auto read_x = [&](const char *from, int i) { return P::fragment(from, (i * WM + wm) * 16); };
    const auto read_w = [&](const char *from, int j) { return Q::fragment(from + P::kBytes, (wn * FN + j) * 16); };
    const auto scale_x = [&](const char *from, int i) { return FP4 ? S::fragment(from + SCALES, (i * WM + wm) * 16) : 0; };
    const auto scale_w = [&](const char *from, int j) { return FP4 ? S::fragment(from + SCALES, BM + (wn * FN + j) * 16) : 0; };

    typedef typename sums_of<FORM>::type SUM;
    SUM acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = SUM{0, 0, 0, 0};

    // Four tiles of k in LDS.  While tile s is multiplied its rows' fragments are read two ahead and the columns'
    // fragments of tile s+1 beside them, so that the matrix cores find their operands in registers; tile s+3 is on its
    // way into the place of tile s-1, which every wave has left.  Two tiles of loads may be under way at the meeting
    // of the waves, which only waits for tile s+2.  (The places are told apart as restricted pointers: otherwise the
    // compiler waits for all loads to LDS before each transposing read.)
    i32x4 x[4], w[2][FN];
    int xs[4], ws[2][FN];
    const auto step = [&](int s, int place, char *__restrict__ fill, const char *__restrict__ here, const char *__restrict__ next) {
        if constexpr (FP4) {   // a tile further ahead, since their loads end in a register
            scales.commit(fill + SCALES);
            scales.issue(s + 4, k / 32);
        }
        if constexpr (!ALIGNED) {   // the same
            commit(fill, s + 3, place);
            refill(s + 3, place);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const char *from = i + 2 < FM ? here : next;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if constexpr (FP4) {
                    acc[i][j] = mfma_fp4(w[0][j], x[i % 4], acc[i][j], ws[0][j], xs[i % 4]);
                } else if constexpr (FORM == kI8) {
                    acc[i][j] = mfma_i8(w[0][j], x[i % 4], acc[i][j]);
                } else {
                    acc[i][j] = mfma<T>(w[0][j], x[i % 4], acc[i][j]);
                }
                // a product occupies the matrix core for 16 cycles: what else there is to issue goes between them
                if (j == 0) {
                    x[(i + 2) % 4] = read_x(from, (i + 2) % FM);
                    xs[(i + 2) % 4] = scale_x(from, (i + 2) % FM);
                }
                if (j == 1) {
#pragma unroll
                    for (int c = i * FN / FM; c < (i + 1) * FN / FM; ++c) {
                        w[1][c] = read_w(next, c);
                        ws[1][c] = scale_w(next, c);
                    }
                }
                if (j == FN / 2 && ALIGNED) {
#pragma unroll
                    for (int l = i * LOADS / FM; l < (i + 1) * LOADS / FM; ++l) issue(l, s + 3, fill);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (FP4) formed<FM>(acc);
        __builtin_amdgcn_sched_barrier(0);
        if (FP4 && S::whole(s + 4, k / 32)) wait_and_meet<LOADS + S::kLoads>();   // the scales' loads as well
        else wait_and_meet<ALIGNED ? LOADS : 63>();
        __builtin_amdgcn_sched_barrier(0);
    };
    if (steps > 0) {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int r = 0; r < RING; ++r) {
                if constexpr (MODE != kDw) p.fetch(r, r);
                if constexpr (MODE == kFwd) q.fetch(r, r);
            }
            look_up(0);
            if constexpr (MODE == kDw) p.template fetch<false>(0, 0);
            if constexpr (MODE != kFwd) q.template fetch<MODE == kDw>(0, now);
        }
#pragma unroll
        for (int s = 0; s < 3; ++s) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) issue(i, s, lds[s]);
            commit(lds[s], s, s % BODIES);
            refill(s, s % BODIES);
            if constexpr (FP4) {
                scales.issue(s, k / 32);
                scales.commit(lds[s] + SCALES);
            }
        }
        if constexpr (FP4) scales.issue(3, k / 32);
        wait_and_meet<ALIGNED ? LOADS : 63>();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = read_x(lds[0], i);
            xs[i] = scale_x(lds[0], i);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            w[0][j] = read_w(lds[0], j);
            ws[0][j] = scale_w(lds[0], j);
        }
        // With loads to LDS one body a tile: the pointers of two would not be told apart.
#pragma unroll 1
        for (int s0 = 0; s0 < steps; s0 += BODIES) {
#pragma unroll
            for (int r = 0; r < BODIES; ++r) {
                const int s = s0 + r;
                if (r > 0 && s >= steps) break;
                step(s, (r + 3) % BODIES, lds[(s + 3) & 3], lds[s & 3], lds[(s + 1) & 3]);
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    w[0][j] = w[1][j];
                    ws[0][j] = ws[1][j];
                }
                if constexpr (FM == 2) {   // read two ahead is a tile ahead
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        x[i] = x[i + 2];
                        xs[i] = xs[i + 2];
                    }
                }
            }
        }
        // nothing may still be on its way to LDS when the workgroup ends
        wait_and_meet<0>();
    }

    typename std::conditional<FORM == kI8, Units<ACT, FM, FN, WM>, NoUnits>::type units;
    if constexpr (FORM == kI8) units.load(a, a.q_unit + (ACT ? 2LL : 1LL) * a.n * t.e, wm, wn, t.n * OUT_N, count - m0, slot_row);
    store_results<T, MODE, ACT, FM, FM, FN, WM, OUT_N>(a, acc, wm, wn, MODE == kDw ? (long long)t.e * a.m + m0 : (long long)t.begin + m0,
                                                MODE == kDw ? a.m - m0 : count - m0, t.n * OUT_N, units);
}

template <typename T, int FORM, int MODE, int ACT, int BM, int BN, int WM, int WN, bool ALIGNED>
int launch(const Args &a, hipStream_t stream)
{
    const long long out_n = ACT ? BN / 2 : BN, nt = (a.n + out_n - 1) / out_n;
    long long tiles;
    if (MODE == kDw) tiles = (long long)a.experts * ((a.m + BM - 1) / BM) * nt;
    else tiles = ((long long)a.slots / BM + (a.experts < a.slots ? a.experts : a.slots)) * nt;
    return launch_tiles(k_mm<T, FORM, MODE, ACT, BM, BN, WM, WN, ALIGNED>, a, tiles, WM * WN * 64, stream, "k_mm");
}

// Which kernel takes a product.  Figures in us with the weights not in cache, bf16 unless said otherwise; "rows" are an
// expert's on average, n counts both halves under SwiGLU.
//
// Few rows: k_mm_rows, the weights straight to registers, against the 128 x 128 tiles: 64 experts, 2048 -> 2 x 1024, rows
// 1: 94 against 115, 8: 104 / 128, 16: 137 / 128; 16 experts, 2048 -> 2048, rows 1: 26 / 37, 8: 32 / 38, 16: 48 / 38.  With
// many tiles (512 and more of 128 x 128, which go to k_mm_stream) it depends on the weights' rows.  128 experts, k -> 2 x 512,
// rows 1, 4, 8 against k_mm_stream: of 1 KB 42, 46, 48 / 32, 33, 33; 2 KB 57, 67, 69 / 54, 57, 57; 3 KB 78, 87, 91 / 82, 85, 86;
// 3.5 KB 84, 94, 97 / 93, 97, 96; 4 KB 93, 102, 105 / 121, 130, 131; 5 KB 113, 127, 132 / 137, 142, 142.  In 4-bit blocks, of
// 1 KB 36, 42, 44 / 37, 39, 39; 2 KB 58, 67, 72 / 67, 69, 70; 3 KB 83, 92, 102 / 103, 107, 108; 4 KB 103, 118, 131 / 138, 145, 146.
//
// Many: k_mm_stream, 256 x 256 tiles, against 128 x 128.  It wins from a tile a CU on, whatever the rows, since its loads
// run ahead of everything: dx of 64 experts, 2048 x 2048, rows 1: 91 / 94, 64: 104 / 120, 512: 334 / 409; dw of 16, rows
// 64: 44 / 50, 512: 101 / 128, of 128, 1024 x 1024, rows 64: 82 / 116, 1: 81 / 76; forward, 32 experts, 2048 -> 2 x 2048,
// rows 96: 129 / 141, 512: 343 / 412, in 4-bit blocks 51 / 65, 128 / 172.  With fewer tiles, half of them at least, it
// still wins from 96 rows on, where a tile's half is full (16 experts, 2048 -> 2048, 96: 52 / 56, 256: 66 / 75, but 192:
// 65 / 56; rows 64: 51 / 39), and loses under that (8 experts, 1024 -> 1024, 256: 26 / 19, 512: 27 / 24; dw 8 of 1024 x
// 1024, 512: 30 / 21).
//
// Operands that do not lie in 16 bytes come by way of registers, which favours many small workgroups.  Forward, the rows'
// kernel against 64 x 64 and 128 x 128 tiles: 12 experts, 1111 -> 717, rows 8: 15 / 23 / 42, 32: 25 / 24 / 43, 400: 179 /
// 55 / 61; 16 experts, 2047 -> 2047, 4: 48 / 45 / 74, 64: 189 / 78 / 81, 100: 277 / 105 / 105, 200: 518 / 151 / 113; 64
// experts, 1025 -> 513, 8: 35 / 34 / 48, 64: 129 / 55 / 59, 400: 661 / 163 / 148; 32 experts, 2047 -> 2 x 1023, 4: 82 / 89 /
// 98, 16: 120 / 93 / 96, 64: 317 / 136 / 107.  Of the 64 x 64 tiles five go to a CU at a time, 1280 to all: up to about there
// they win, with 1152 of them (64 experts, 1025 -> 513, rows 64) 55 / 59, (32, 2047 -> 2 x 1023, 8) 90 / 94, with 1280 (the same,
// 16) 91 / 94, and behind that lose, with 1312 (16, 2047 -> 2047, 100) 105 / 101, (32, 2047 -> 2 x 511, 100) 100 / 96, 1456 (16,
// 1025 -> 1023, 300) 67 / 63, 1536 (32, 2047 -> 2 x 1023, 32) 104 / 97.  It costs up to 16% where the 128 x 128 tiles, two a CU,
// just fit a round, with 1024 (32, 2047 -> 2 x 511, 64) 89 / 77, or just do not, with 2112 (16, 2047 -> 2047, 200) 156 / 173.
//
// 8-bit integers, the rows' kernel, 128 x 128 tiles and k_mm_stream: 64 experts, 2048 -> 2 x 1024, rows 2: 42 / 57 / 61, 8: 56 /
// 61 / 65, 12: 64 / 61 / 64, 25: - / 63 / 65, 64: - / 82 / 70; 128 experts, 1024 -> 2 x 512, 4: 33 / 37 / 38, 12: 44 / 39 / 39; 16
// experts, 4096 -> 2048, 8: 35 / 43 / 51, 12: 41 / 42 / 51, 20: 53 / 42 / 51; 32 experts, 2047 -> 2 x 1023, 18: 43 / 34 / 37, 37: 69 /
// 36 / 38; 2048 -> 2 x 2048, 128: - / 104 / 95.  Columns that fill less of 256 x 256 tiles by a third or more: 16 experts, 3169 ->
// 265, 2181: - / 89 / 92; 24, 4013 -> 287, 1460: - / 108 / 113; 96, 3728 -> 304, 350: - / 119 / 135; 12, 1189 -> 317, 3298: - / 46 / 49; 16,
// 2048 -> 384, 2048: - / 50 / 53; but 2048 -> 768: - / 89 / 65, 1024 -> 640: - / 47 / 42.  Where
// even the 128 x 128 tiles are few the rows' kernel fills the card longer: 12 experts, 1111 -> 717, 16: 6 / 12 / 16, 52: 9 / 15 / 21,
// 100: 13 / 17 / 25; 8 experts, 1024 -> 1024, 32: 8 / 11 / 14, 64: 12 / 12 / 15, 96: 16 / 12 / 16; 4 experts, 2048 -> 2 x 512, 50:
// 9 / 17 / 22.  So it ends somewhere between 50 and 100 rows, by the number of tiles: with 60 for all, up to 4 us are lost above.
//
// Gradients with 128 x 128 against 256 x 256: 32764 slots of 32 experts, 1023 x 2049, dx 522 / 423, dw 628 / 540; 8000 of 16,
// 2047 x 2047, dx 243 / 270, dw 377 / 287; 2000 of 16, 1023 x 1025, dx 45 / 72, dw 90 / 91.
//
// Figures of results whose rows do not lie in 16 bytes are of when they were stored one element at a time.  By 16 bytes at any
// address those kernels gain alike: 32764 of 32, 1023 x 2049 dx 325, dw 409; 8192 of 8, 1024 -> 1023 48 to 32; 8-bit integers,
// 28812 slots of 12, 673 -> 525 78 to 37, 32634 of 24, 1024 -> 549 93 to 46.
template <typename T, int FORM, int MODE, int ACT, bool ALIGNED>
int launch_size(const Args &a, hipStream_t stream)
{
    const long long rows = a.experts > 0 ? a.slots / a.experts : 0, used = a.experts < a.slots ? a.experts : a.slots;
    const auto tiles = [&](long long side) {   // at most, of side x side results
        return (MODE == kDw ? a.experts * ((a.m + side - 1) / side) : a.slots / side + used) * ((a.n * (ACT ? 2LL : 1LL) + side - 1) / side);
    };
    if constexpr (MODE == kFwd) {
        const bool few = FORM == kI8 ? rows <= (tiles(128) < 128 ? 60 : 8)
                         : ALIGNED   ? rows <= 8 && (tiles(128) < 512 || a.ld_q >= 4000)
                                     : rows <= (tiles(128) < 128 ? 24 : 4);
        if (few) return launch_rows<T, FORM, ACT, ALIGNED>(a, stream);
    }
    if constexpr (ALIGNED) {
        const long long columns = a.n * (ACT ? 2LL : 1LL);
        const bool half = FORM == kI8 && (rows < 48 || 20 * ((columns + 255) / 256) >= 13 * ((columns + 127) / 128));   // half empty tiles
        if (tiles(256) >= (MODE != kDw && rows >= 96 ? 128 : 256) && !half) return launch_stream<T, FORM, MODE, ACT>(a, stream);
    } else if constexpr (MODE == kFwd) {
        if (tiles(64) < 1300) return launch<T, FORM, MODE, ACT, 64, 64, 2, 2, ALIGNED>(a, stream);
    } else {
        if (MODE == kDw ? tiles(256) >= 256 : tiles(256) >= 512 && rows >= 256) return launch<T, FORM, MODE, ACT, 256, 256, 2, 4, ALIGNED>(a, stream);
    }
    return launch<T, FORM, MODE, ACT, 128, 128, 2, 2, ALIGNED>(a, stream);
}

// whether `bytes` lie within the 32-bit offsets of a buffer descriptor
bool fits(long long rows, long long ld) { return (unsigned long long)rows * ld < kBufferMax; }

bool lies16(const void *p, long long ld) { return ((uintptr_t)p | (unsigned long long)ld) % 16 == 0; }

template <int MODE, int ACT>
int run(const pfk_moe_mm_args *g, Args a, bool aligned, hipStream_t stream)
{
    if (g->dtype == PF_F16)
        return aligned ? launch_size<f16, kHalf, MODE, ACT, true>(a, stream) : launch_size<f16, kHalf, MODE, ACT, false>(a, stream);
    return aligned ? launch_size<bf16, kHalf, MODE, ACT, true>(a, stream) : launch_size<bf16, kHalf, MODE, ACT, false>(a, stream);
}

// Operands of 4-bit blocks and of 8-bit integers lie in 16 bytes always; beyond the descriptors' offsets k_mm_rows has
// 64-bit addresses.
template <int FORM, typename T, int ACT>
int run_type(const Args &a, bool fit, hipStream_t stream)
{
    return fit ? launch_size<T, FORM, kFwd, ACT, true>(a, stream) : launch_rows<T, FORM, ACT, true>(a, stream);
}

template <int FORM>
int run_codes(const pfk_moe_mm_args *g, Args a, hipStream_t s)
{
    a.n = g->n;
    a.q_expert = g->ld_q * g->n * (g->act == PF_ACT_SWIGLU ? 2 : 1);
    a.wide = lies16(g->out, g->ld_out);
    const bool fit = fits(g->p_rows, g->ld_p) && fits(1, a.q_expert) && fits(g->slots, 4);
    if (g->act == PF_ACT_SWIGLU) return g->dtype == PF_F16 ? run_type<FORM, f16, 1>(a, fit, s) : run_type<FORM, bf16, 1>(a, fit, s);
    return g->dtype == PF_F16 ? run_type<FORM, f16, 0>(a, fit, s) : run_type<FORM, bf16, 0>(a, fit, s);
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
    if (g->rows) {   // 2^(32+s) / d rounded up, with 2^s < d <= 2^(s+1): exact for v < 2^31, and 32 bits wide
        unsigned d = (unsigned)g->row_div;
        while (d > 1 && (1u << (a.div_shift + 1)) < d && a.div_shift < 30) ++a.div_shift;
        a.div_mul = d == 1 ? 0 : (unsigned)(((1ull << (32 + a.div_shift)) + d - 1) / d);
    }
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

}  // namespace

extern "C" {

int pfk_moe_mm(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.n = g->n;
    a.k = g->k;
    const int each = g->act == PF_ACT_SWIGLU ? 2 : 1;
    a.q_expert = g->ld_q * g->n * each;
    a.wide = lies16(g->out, g->ld_out) && (!g->pre || (lies16(g->pre, g->ld_pre) && g->n % 8 == 0));
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->k % 8 == 0 && fits(g->p_rows, g->ld_p) && fits(1, a.q_expert) &&
                         fits(g->slots, 4);
    hipStream_t s = (hipStream_t)stream;
    return g->act == PF_ACT_SWIGLU ? run<kFwd, 1>(g, a, aligned, s) : run<kFwd, 0>(g, a, aligned, s);
}

int pfk_moe_mm_dx(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.n = g->k;   // columns of w are the results, its rows are summed over
    a.k = g->n;
    a.q_expert = g->ld_q * g->n;
    a.wide = lies16(g->out, g->ld_out);
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
    a.wide = lies16(g->out, g->ld_out);
    const bool aligned = lies16(g->p, g->ld_p) && lies16(g->q, g->ld_q) && g->n % 8 == 0 && g->k % 8 == 0 &&
                         fits(g->slots, g->ld_p) && fits(g->p_rows, g->ld_q);
    return run<kDw, 0>(g, a, aligned, (hipStream_t)stream);
}

int pfk_moe_mm_mx4(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.k = g->k;
    a.p_scales = (const unsigned char *)g->p_scales;
    a.q_scales = (const unsigned char *)g->q_scales;
    return run_codes<kMx4>(g, a, (hipStream_t)stream);
}

int pfk_moe_mm_i8(const pfk_moe_mm_args *g, void *stream)
{
    Args a = common(g);
    a.k = (int)g->ld_q;   // zeros behind the elements there are
    a.p_unit = (const float *)g->p_scales;
    a.q_unit = (const float *)g->q_scales;
    return run_codes<kI8>(g, a, (hipStream_t)stream);
}

}  // extern "C"
