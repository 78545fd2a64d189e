// moe_mm_stream.hip — grouped products with many rows an expert: one workgroup a CU takes tile after tile, its loads
// running ahead of the products across the tiles' ends.
//
// 8192 tokens x 4 of 32 experts, 2048 -> 2 x 2048, SwiGLU, bf16: 524 to 563 us by the card and how long it has run, 1.0
// PFLOP/s (with the pre-activations, 268 MB more to write, 565 to 573); a library's product of the same size in one piece 366
// to 400.  In one piece this kernel takes 503.  The clock falls to 1.75 GHz with random operands, and what is left out then
// counts by its power: all-zero operands 402; without loads to LDS 440, without LDS reads 443, without either 340; without the
// meetings of the waves no less.  So what a product costs in LDS reads is the bound, and that follows from the tiling: a wave
// of 128 x 64 results reads 12 fragments for 32 products.  Ragged rows add 7% of rows that are not there and a tenth round of
// tiles where 9.2 would do.  With 4-bit operands 215 to 227 us, 2.5 PFLOP/s; gradients of 16384 slots of 16 experts, 2048 x
// 2048, 166 us (dx) and 177 to 188 us (dw, fp32).
#include "moe_tiles.hpp"

namespace pfmoe {
namespace {

constexpr int kTile = 256;      // rows and columns of a tile
constexpr int kThreads = 512;   // eight waves, two a SIMD, of 128 x 64 results each
constexpr int kCus = 256;       // workgroups, a CU each
constexpr int kMinSteps = 4;    // tiles of k an output tile takes at least: the loads run three ahead

// One output tile.
struct Work {
    int e, m0, n, begin, count;   // expert, first row, tile of columns; the expert's slots
    int rows;                     // of the tile, at most
};

// The tiles of this workgroup, by number.  Each XCD has consecutive tiles, whose operands then meet in its L2: inside an
// expert eight tiles of rows go side by side over the columns, its last one, with fewer rows, among them.  (With these
// last ones kept for the end, to even out the workgroups' shares, the weights are read once more: 8192 tokens x 4 of 32
// experts, 2048 -> 2 x 2048, in 606 us, 545 so.)  Where at most half the workgroups have a tile in the last round, two
// share each, by rows: 16 experts, 2048 -> 2048, 128 rows each in 53 us and not 63, 512 in 106 and not 120.
struct Plan {
    const int *before, *begins, *counts;   // in LDS: tiles before each expert, its first slot, its slots
    const int *ranked;                     // the weights' gradient: the experts by their slots, most first
    int experts, nt, mt;
    int tile0, tiles;                      // this XCD's
    int first, step;

    __device__ __forceinline__ int expert_of(int id) const
    {
        const int lane = threadIdx.x & (kWave - 1);
        for (int base = 0;; base += kWave) {
            const unsigned long long past = __ballot(base + lane >= experts || before[base + lane + 1] > id);
            if (past) return base + __builtin_ctzll(past);
        }
    }
    __device__ __forceinline__ bool get(int i, Work &w) const
    {
        int q = first + i * step, half = -1;
        if (i == tiles / step && 2 * (tiles % step) <= step) {
            q = i * step + first / 2;
            half = first % 2;
        }
        if (q >= tiles) return false;
        const int id = tile0 + q;
        w.e = expert_of(id);
        w.begin = __builtin_amdgcn_readfirstlane(begins[w.e]);
        w.count = __builtin_amdgcn_readfirstlane(counts[w.e]);
        const int at = id - __builtin_amdgcn_readfirstlane(before[w.e]), rows = (w.count + kTile - 1) / kTile;
        const int group = at / (8 * nt), side = min(8, rows - group * 8), j = at - group * 8 * nt;
        w.m0 = (group * 8 + j % side) * kTile;
        w.n = j / side;
        w.rows = half < 0 ? kTile : kTile / 2;
        if (half > 0) w.m0 += kTile / 2;
        return w.m0 < w.count;
    }
    // The weights' gradient: each XCD takes its share of every expert's tiles, since experts differ in their slots; those
    // with most come first, and the workgroups take them forth and back by turns, so that their sums of slots are alike.
    __device__ __forceinline__ bool get_dw(const Args &a, int i, Work &w) const
    {
        const int q = (i % 2 ? step - 1 - first : first) + i * step, each = mt * nt;
        const long long at = (long long)q * kXcds + tile0;   // tile0: the XCD
        if (at >= (long long)a.experts * each) return false;
        w.e = __builtin_amdgcn_readfirstlane(ranked[(int)(at / each)]);
        const int j = (int)(at % each);
        w.m0 = j % mt * kTile;
        w.n = j / mt;
        w.rows = kTile;
        w.begin = __builtin_amdgcn_readfirstlane(begins[w.e]);
        w.count = __builtin_amdgcn_readfirstlane(counts[w.e]);
        return true;
    }
};

// floor(v / d) of 0 <= v < 2^31 by multiplication
__device__ __forceinline__ unsigned divide(unsigned v, unsigned mul, int shift) { return (unsigned)(((unsigned long long)v * mul) >> 32) >> shift; }

template <typename T, bool FP4, int MODE, int ACT>
__global__ __launch_bounds__(kThreads) void k_mm_stream(const Args a)
{
    constexpr int WM = 2, WN = 4, FM = kTile / WM / 16, FN = kTile / WN / 16;
    typedef typename std::conditional<MODE == kDw, Across<kTile, kThreads, true>, Along<kTile, kThreads, true>>::type P;
    typedef typename std::conditional<MODE == kFwd, Along<kTile, kThreads, true>, Across<kTile, kThreads, true>>::type Q;
    typedef Scales<2 * kTile, kThreads> S;
    constexpr int SCALES = P::kBytes + Q::kBytes, SLOT = SCALES + (FP4 ? S::kBytes : 0);
    constexpr int LOADS = P::kLoads + Q::kLoads;
    // One array for all: of several the compiler would tell accesses apart, but not the loads to LDS, and wait for those
    // before every read.  Four tiles of k; the experts' tables (Plan); rows of this output tile and of the next, as `rows`
    // has them.
    constexpr int TABLE = PF_MOE_MAX_EXPERTS + 1, IDS = MODE == kDw ? 0 : 2 * kTile;
    __shared__ __align__(1024) char shared[4 * SLOT + 4 * (3 * TABLE + IDS)];
    const auto lds = [&](int place) { return shared + place * SLOT; };
    const auto table = [&](int i) { return (int *)(shared + 4 * SLOT) + i * TABLE; };
    const auto ids = [&](int side) { return (int *)(shared + 4 * SLOT) + 3 * TABLE + side * kTile; };

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), wm = wave / WN, wn = wave % WN;
    constexpr int OUT_N = ACT ? kTile / 2 : kTile;
    Plan plan;
    plan.experts = a.experts;
    plan.nt = (a.n + OUT_N - 1) / OUT_N;
    plan.mt = (a.m + kTile - 1) / kTile;
    plan.first = blockIdx.x / kXcds;
    plan.step = gridDim.x / kXcds;
    const int xcd = blockIdx.x % kXcds;
    plan.before = plan.ranked = table(0);
    plan.begins = table(1);
    plan.counts = table(2);
    if constexpr (MODE == kDw) {
        plan.tile0 = xcd;
        for (int e = tid; e < a.experts; e += kThreads) {
            int b, f;
            expert_rows(a.offsets, e, a.slots, b, f);
            table(1)[e] = b;
            table(2)[e] = f - b;
        }
        __syncthreads();
        for (int e = tid; e < a.experts; e += kThreads) {
            const int mine = table(2)[e];
            int rank = 0;
            for (int i = 0; i < a.experts; ++i) {
                const int other = table(2)[i];
                rank += other > mine || (other == mine && i < e);
            }
            table(0)[rank] = e;
        }
        __syncthreads();
    } else {
        if (wave == 0) {
            int before = 0;   // held at kMost where offsets that decrease give the experts more slots than there are
            constexpr int kMost = 1 << 30;
            for (int base = 0; base < a.experts; base += kWave) {
                int b = 0, e = 0;
                if (base + lane < a.experts) expert_rows(a.offsets, base + lane, a.slots, b, e);
                const int sum = scan_wave((e - b + kTile - 1) / kTile * plan.nt);
                if (base + lane < a.experts) {
                    table(0)[base + lane + 1] = min(before + sum, kMost);
                    table(1)[base + lane] = b;
                    table(2)[base + lane] = e - b;
                }
                before = min(before + __builtin_amdgcn_readlane(sum, kWave - 1), kMost);
            }
            if (lane == 0) table(0)[0] = 0;
        }
        __syncthreads();
        const int all = __builtin_amdgcn_readfirstlane(table(0)[a.experts]), each = (all + kXcds - 1) / kXcds;
        plan.tile0 = min(xcd * each, all);
        plan.tiles = min(plan.tile0 + each, all) - plan.tile0;
    }
    const auto get = [&](int i, Work &w) {
        if constexpr (MODE == kDw) return plan.get_dw(a, i, w);
        else return plan.get(i, w);
    };
    const auto depth = [&](const Work &w) { return MODE == kDw ? w.count : a.k; };
    const auto steps_of = [&](const Work &w) {   // tiles of k; zeros behind k
        const int steps = FP4 ? (depth(w) + 127) / 128 : (depth(w) + 31) / 32;
        return steps < kMinSteps ? kMinSteps : steps;
    };
    const auto weight_row = [&](const Work &w, int r) {
        if constexpr (ACT) return min(w.n * OUT_N + r / 32 * 16 + r % 16, a.n - 1) + (r / 16 % 2) * a.n;
        else return min(w.n * kTile + r, a.n - 1);
    };
    // the slot of row r of a tile, and the operand's row by what `rows` has for it
    const auto slot_of = [&](const Work &w, int r) { return w.begin + min(w.m0 + r, w.count - 1); };
    const auto looked_up = [&](int v) {
        if (!a.rows) return v;
        const unsigned r = v < 0 ? 0u : a.row_div == 1 ? (unsigned)v : divide((unsigned)v, a.div_mul, a.div_shift);
        return r < (unsigned)a.p_rows ? (int)r : 0;
    };

    Work now, next;
    if (!get(0, now)) return;
    bool more = get(1, next);

    // ---- loads: a cursor of their own goes over the tiles of k, three ahead of the products ----------------------
    P p;
    Q q;
    S scales;
    int load_k = 0, load_steps = 0, load_begin = 0, load_depth = 0;   // tile of k, of how many; the output tile's slots
    int rows = 0;                                                     // kDw: x's rows of the cursor's tile
    if constexpr (MODE != kDw) p.piece = (tid & 3) ^ ((tid >> 3) & 3);
    if constexpr (MODE == kFwd) q.piece = (tid & 3) ^ ((tid >> 3) & 3);
    // Straight to LDS as well: registers of a load under way would be waited for in the innermost loop.
    const auto load_ids = [&](const Work &w, int side) {
        if constexpr (MODE != kDw) {
            if (a.rows && wave < kTile / kWave)
                to_lds4(buffer_of((const char *)a.rows, 4ull * a.slots), 4u * (unsigned)slot_of(w, tid), ids(side) + wave * kWave);
        }
    };
    const auto row_of = [&](const Work &w, int side, int r) { return a.rows ? looked_up(ids(side)[r]) : slot_of(w, r); };
    const auto aim = [&](const Work &w, int side) {   // the cursor at an output tile's first tile of k
        load_k = 0;
        load_steps = steps_of(w);
        load_begin = w.begin;
        load_depth = depth(w);
        if constexpr (MODE == kDw) {
            p.init(a.p + a.ld_p * w.begin, span(a.ld_p, load_depth, a.m), a.ld_p, w.m0, a.m, load_depth);
            q.init(a.q, span(a.ld_q, a.p_rows, a.n), a.ld_q, w.n * kTile, a.n, load_depth);
        } else {
            p.from = buffer_of(a.p, FP4 ? a.ld_p * a.p_rows : span(a.ld_p, a.p_rows, a.k));
            p.k_pieces = a.k / (FP4 ? 32 : 8);
#pragma unroll
            for (int i = 0; i < P::kLoads; ++i) p.at[i] = (unsigned)row_of(w, side, P::tile_row(i)) * (unsigned)a.ld_p + p.piece * 16;
            if constexpr (MODE == kFwd) {
                q.from = buffer_of(a.q + a.q_expert * w.e, a.q_expert);
                q.k_pieces = p.k_pieces;
#pragma unroll
                for (int i = 0; i < Q::kLoads; ++i) q.at[i] = (unsigned)weight_row(w, Q::tile_row(i)) * (unsigned)a.ld_q + q.piece * 16;
            } else {
                q.init(a.q + a.q_expert * w.e, a.q_expert, a.ld_q, w.n * kTile, a.n, a.k);
            }
        }
    };
    const auto aim_at_nothing = [&]() {     // from here on the loads write zeros
        load_k = 0;
        load_steps = 1 << 24;
        load_depth = 0;
        if constexpr (MODE == kDw) p.k = 0; else p.k_pieces = 0;
        if constexpr (MODE == kFwd) q.k_pieces = 0; else q.k = 0;
    };
    const auto aim_scales = [&](const Work &w, int side) {
        if constexpr (FP4) {
            const long long blocks = a.k / 32;
#pragma unroll
            for (int i = 0; i < S::kLoads; ++i) {
                const int r = tid + i * kThreads;
                scales.row[i] = r < kTile ? a.p_scales + blocks * row_of(w, side, r)
                                          : a.q_scales + blocks * ((ACT ? 2LL : 1LL) * a.n * w.e + weight_row(w, r - kTile));
            }
        }
    };
    const auto look_rows = [&](int t, int begin, int count) {
        if constexpr (MODE == kDw) {
            if (count <= 0) return 0;
            const int slot = begin + min(Q::lookup(t), count - 1);
            return a.rows ? a.rows[slot] : slot;
        } else {
            return 0;
        }
    };
    // load i of the cursor's tile
    const auto issue = [&](int i, char *to) {
        if (i < P::kLoads) {
            if constexpr (MODE == kDw) p.template issue<false>(i, load_k, to, 0);
            else p.issue(i, load_k, to);
        } else {
            if constexpr (MODE == kFwd) q.issue(i - P::kLoads, load_k, to + P::kBytes);
            else q.template issue<MODE == kDw>(i - P::kLoads, load_k, to + P::kBytes, rows);
        }
    };

    // ---- products ---------------------------------------------------------------------------------------------------
    const auto read_x = [&](const char *from, int i) { return P::fragment(from, (i * WM + wm) * 16); };
    const auto read_w = [&](const char *from, int j) { return Q::fragment(from + P::kBytes, (wn * FN + j) * 16); };
    const auto scale_x = [&](const char *from, int i) { return FP4 ? S::fragment(from + SCALES, (i * WM + wm) * 16) : 0; };
    const auto scale_w = [&](const char *from, int j) { return FP4 ? S::fragment(from + SCALES, kTile + (wn * FN + j) * 16) : 0; };
    f32x4 acc[FM][FN];
    i32x4 x[4], w[2][FN];
    int xs[4], ws[2][FN];

    // One tile of k, in `here`: FMV of the wave's FM blocks of rows.  Its rows' fragments are read two ahead and the
    // columns' of the tile behind it (`next_at`) in its first half, so that the matrix cores find their operands in
    // registers, while the cursor's tile is loaded into `fill`, the place of the tile before it.
    int side = 1;   // of ids that the next output tile has
    const auto step = [&](auto blocks, bool fresh, char *fill, const char *here, const char *next_at) {
        constexpr int FMV = decltype(blocks)::value;
        const bool turn = load_k + 1 == load_steps;
        int rows_next = 0;
        bool scales_whole = false;
        if constexpr (FP4) {   // a tile further ahead, since their loads end in a register
            scales.commit(fill + SCALES);
            if (turn && more) aim_scales(next, side);
            const int t = turn ? 0 : load_k + 1;
            scales_whole = S::whole(t, a.k / 32);
            scales.issue(t, a.k / 32);
        }
        if constexpr (MODE == kDw)   // looked up before the loads, so that waiting for it does not wait for them
            rows_next = turn ? look_rows(0, next.begin, more ? next.count : 0) : look_rows(load_k + 1, load_begin, load_depth);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FMV; ++i) {
            const char *from = i + 2 < FMV ? here : next_at;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if constexpr (FP4) acc[i][j] = mfma_fp4(w[0][j], x[i % 4], acc[i][j], ws[0][j], xs[i % 4]);
                else acc[i][j] = mfma<T>(w[0][j], x[i % 4], acc[i][j]);
                // a product occupies the matrix core for 16 cycles: what else there is to issue goes between them
                if (j == 0) {
                    x[(i + 2) % 4] = read_x(from, (i + 2) % FMV);
                    xs[(i + 2) % 4] = scale_x(from, (i + 2) % FMV);
                } else if (j == 2) {
#pragma unroll
                    for (int l = i * LOADS / FMV; l < (i + 1) * LOADS / FMV; ++l) issue(l, fill);
                } else if (i < FMV / 2) {
                    constexpr int EACH = 2 * FN / FMV;   // a row's share
#pragma unroll
                    for (int c = i * EACH + j / 2 * EACH / 2; c < i * EACH + (j / 2 + 1) * EACH / 2; ++c) {
                        w[1][c] = read_w(next_at, c);
                        ws[1][c] = scale_w(next_at, c);
                    }
                }
                if (i == FMV - 1) {
                    w[0][j] = w[1][j];
                    ws[0][j] = ws[1][j];
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (FP4) formed<FMV>(acc);
        rows = looked_up(rows_next);
        // The tile after the next has to be there: this step's loads may still be on their way, and after an output
        // tile's end, where all before them are there, stores besides.
        if (fresh) wait_and_meet<63>();
        else if (FP4 && scales_whole) wait_and_meet<LOADS + S::kLoads>();
        else wait_and_meet<LOADS>();
        if (++load_k == load_steps) {
            if (more) aim(next, side); else aim_at_nothing();
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    // The same with its places told apart as restricted pointers: otherwise the compiler waits for all loads to LDS before
    // each transposing read (and, where it is told, before each plain one).
    const auto step_apart = [&](auto blocks, bool fresh, char *__restrict__ fill, const char *__restrict__ here,
                                const char *__restrict__ next_at) {
        step(blocks, fresh, fill, here, next_at);
    };

    load_ids(now, 0);
    if (more) load_ids(next, 1);
    wait_and_meet<0>();
    aim(now, 0);
    aim_scales(now, 0);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        if constexpr (MODE == kDw) rows = looked_up(look_rows(s, load_begin, load_depth));
        if constexpr (FP4) {
            scales.issue(s, a.k / 32);
            scales.commit(lds(s) + SCALES);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) issue(i, lds(s));
        ++load_k;
    }
    if constexpr (MODE == kDw) rows = looked_up(look_rows(3, load_begin, load_depth));
    if constexpr (FP4) scales.issue(3, a.k / 32);
    wait_and_meet<0>();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        x[i] = read_x(lds(0), i);
        xs[i] = scale_x(lds(0), i);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        w[0][j] = read_w(lds(0), j);
        ws[0][j] = scale_w(lds(0), j);
    }

    int place = 0;   // of the current tile of k
    for (int i = 0;; ++i) {
        const int steps = steps_of(now), have = min((MODE == kDw ? a.m : now.count) - now.m0, now.rows);
#pragma unroll
        for (int r = 0; r < FM; ++r)
#pragma unroll
            for (int c = 0; c < FN; ++c) acc[r][c] = f32x4{0, 0, 0, 0};
        Work after;
        bool more_after = false;
        const auto all = [&](auto blocks) {
            bool fresh = i > 0;
#pragma unroll 1
            for (int s = 0; s < steps; ++s) {
                if constexpr (MODE == kFwd) step(blocks, fresh, lds((place + 3) & 3), lds(place), lds((place + 1) & 3));
                else step_apart(blocks, fresh, lds((place + 3) & 3), lds(place), lds((place + 1) & 3));
                place = (place + 1) & 3;
                fresh = false;
            }
            more_after = more && get(i + 2, after);
            if (more_after) load_ids(after, side ^ 1);
            // Of the next output tile three tiles of k are on their way.  Stores would end behind them in no order that a
            // counted wait could use, so they have to be there first.
            wait_loads();
            store_results<T, MODE, ACT, decltype(blocks)::value, FM, FN, WM, OUT_N>(
                a, acc, wm, wn, MODE == kDw ? (long long)now.e * a.m + now.m0 : (long long)now.begin + now.m0, have, now.n * OUT_N);
        };
        if (have > kTile / 2) all(std::integral_constant<int, FM>());
        else all(std::integral_constant<int, FM / 2>());   // half the rows: half the products
        if (!more) break;
        now = next;
        next = after;
        more = more_after;
        side ^= 1;
    }
}

}  // namespace

template <typename T, bool FP4, int MODE, int ACT>
int launch_stream(const Args &a, hipStream_t stream)
{
    k_mm_stream<T, FP4, MODE, ACT><<<dim3(kCus), dim3(kThreads), 0, stream>>>(a);
    return pfk_internal_launched("k_mm_stream");
}

template int launch_stream<f16, false, kFwd, 0>(const Args &, hipStream_t);
template int launch_stream<f16, false, kFwd, 1>(const Args &, hipStream_t);
template int launch_stream<f16, false, kDx, 0>(const Args &, hipStream_t);
template int launch_stream<f16, false, kDw, 0>(const Args &, hipStream_t);
template int launch_stream<f16, true, kFwd, 0>(const Args &, hipStream_t);
template int launch_stream<f16, true, kFwd, 1>(const Args &, hipStream_t);
template int launch_stream<bf16, false, kFwd, 0>(const Args &, hipStream_t);
template int launch_stream<bf16, false, kFwd, 1>(const Args &, hipStream_t);
template int launch_stream<bf16, false, kDx, 0>(const Args &, hipStream_t);
template int launch_stream<bf16, false, kDw, 0>(const Args &, hipStream_t);
template int launch_stream<bf16, true, kFwd, 0>(const Args &, hipStream_t);
template int launch_stream<bf16, true, kFwd, 1>(const Args &, hipStream_t);

}  // namespace pfmoe
