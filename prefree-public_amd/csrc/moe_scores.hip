// moe_scores.hip — routing by scores on gfx950 (include/prefree_moe.h): sigmoid or softmax scores plus a bias, groups of
// experts, the gradient of the logits, and the bias's step.
#include "moe_route.hpp"

namespace {

using namespace pfmoe;

struct Scores : Route {
    int score, groups, group_size, kept, best;
    int group_lanes, need, vector;   // of the choice in 32 bits: lanes a group, experts a lane (0: not for these sizes), 16-byte loads
    const float *bias;
    float scale;
};

// Order-preserving key of a number, 0 for -infinity (never chosen) and the largest for NaN; -0 and 0 alike.
__device__ __forceinline__ unsigned long long key_of(double r)
{
    if (r != r) return ~0ull;
    const unsigned long long b = __double_as_longlong(r + 0.0);
    if (b == 0xfff0000000000000ull) return 0;
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value_of(unsigned long long key)   // NaN for the largest
{
    return __longlong_as_double((long long)(key >> 63 ? key & ~(1ull << 63) : ~key));
}

template <int CTRL>
__device__ __forceinline__ unsigned long long dpp64(unsigned long long v)
{
    return (unsigned long long)pfdev::dpp<CTRL>((unsigned)(v >> 32)) << 32 | pfdev::dpp<CTRL>((unsigned)v);
}
__device__ __forceinline__ unsigned long long swap16_64(unsigned long long v)
{
    return (unsigned long long)(unsigned)__builtin_amdgcn_ds_swizzle((int)(v >> 32), pfdev::swizzle_xor_pattern<16>()) << 32 |
           (unsigned)__builtin_amdgcn_ds_swizzle((int)(unsigned)v, pfdev::swizzle_xor_pattern<16>());
}
__device__ __forceinline__ unsigned long long readlane64(unsigned long long v, int l)
{
    return (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, l);
}
// v joined by op over a token's G lanes; every lane has the result
template <int G, typename F>
__device__ __forceinline__ unsigned long long joined(unsigned long long v, F op)
{
    v = op(v, dpp64<pfdev::kDppXor1>(v));
    v = op(v, dpp64<pfdev::kDppXor2>(v));
    v = op(v, dpp64<pfdev::kDppHalfMirror>(v));
    v = op(v, dpp64<pfdev::kDppMirror>(v));
    if constexpr (G == 64) {
        v = op(v, swap16_64(v));
        v = op(readlane64(v, 0), readlane64(v, 32));
    }
    return v;
}
template <int G>
__device__ __forceinline__ unsigned long long most_of64(unsigned long long v)
{
    return joined<G>(v, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
}
template <int G>
__device__ __forceinline__ double sum_of64(double v)
{
    return __longlong_as_double((long long)joined<G>(__double_as_longlong(v), [](unsigned long long a, unsigned long long b) {
        return (unsigned long long)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
    }));
}
template <int G>
__device__ __forceinline__ float most_of_floats(float v)   // not of NaN
{
    v = fmaxf(v, pfdev::dpp<pfdev::kDppXor1>(v));
    v = fmaxf(v, pfdev::dpp<pfdev::kDppXor2>(v));
    v = fmaxf(v, pfdev::dpp<pfdev::kDppHalfMirror>(v));
    v = fmaxf(v, pfdev::dpp<pfdev::kDppMirror>(v));
    if constexpr (G == 64) {
        v = fmaxf(v, pfdev::swizzle<pfdev::swizzle_xor_pattern<16>()>(v));
        v = fmaxf(pfdev::readlane(v, 0), pfdev::readlane(v, 32));
    }
    return v;
}

// The choice of a token in 64 bits: G lanes, of which lane l has logits l*PER .. l*PER + PER-1.  Lane j gets choice j.
template <int G, int PER>
__device__ __forceinline__ int choose_exactly(const Scores &a, const float (&z)[PER])
{
    const int lane = threadIdx.x % G;
    unsigned long long key[PER];
    // Without a bias, and where a group counts by one score, scores are in the order of their logits.
    if (!a.bias && (a.groups == 1 || a.best == 1)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = key_of((double)z[i]);
    } else {
        double most = 0, total = 1;
        if (a.score == PF_SCORE_SOFTMAX) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < PER; ++i) m = fmaxf(m, z[i]);
            m = most_of_floats<G>(m);
            most = m > -INFINITY ? (double)m : 0.0;
            total = 0;
#pragma unroll 1
            for (int i = 0; i < PER; ++i) total += exp((double)z[i] - most);
            total = sum_of64<G>(total);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            double s;
            if (a.score == PF_SCORE_SOFTMAX) s = exp((double)z[i] - most) / total;
            else s = 1.0 / (1.0 + exp(-(double)z[i]));
            if (a.bias && e < a.experts) s += (double)a.bias[e];
            key[i] = z[i] == -INFINITY ? 0 : key_of(s);
        }
    }
    if (a.groups > 1) {
        int group[PER], in = lane * PER % a.group_size, mine = lane * PER / a.group_size;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            group[i] = mine;
            if (++in == a.group_size) { in = 0; ++mine; }
        }
        unsigned long long value = 0;   // of group `lane`
        for (int g = 0; g < a.groups; ++g) {
            unsigned long long one = 0, two = 0;   // the two largest
            int at = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const unsigned long long k = group[i] == g ? key[i] : 0;
                if (k > one) { two = one; one = k; at = i; }
                else if (k > two) two = k;
            }
            const unsigned long long best = most_of64<G>(one);
            unsigned long long v = best;
            if (a.best == 2 && best != 0 && best != ~0ull) {
                const int owner = least_of<G>(one == best ? lane * PER + at : 0x7fffffff);
                const unsigned long long next = most_of64<G>(owner == lane * PER + at ? two : one);
                if (next != 0) v = key_of(value_of(best) + value_of(next));
            }
            if (lane == g) value = v;
        }
        int rank = 0;
        for (int g = 0; g < a.groups; ++g) {
            const unsigned long long high = (unsigned)__shfl((int)(value >> 32), g, G), low = (unsigned)__shfl((int)(unsigned)value, g, G);
            const unsigned long long other = high << 32 | low;
            rank += other > value || (other == value && g < lane);
        }
        const unsigned long long in_all = __ballot(lane < a.groups && rank < a.kept);
        const unsigned keep = (unsigned)(in_all >> (G == 64 ? 0 : (threadIdx.x & (kWave - 1)) / G * G));
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (!(keep >> (group[i] & 31) & 1)) key[i] = 0;
    }
    int expert = -1;
    for (int j = 0; j < a.top_k; ++j) {
        unsigned long long best = 0;
        int at = 0;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i)
            if (key[i] >= best) { best = key[i]; at = i; }
        const unsigned long long most = most_of64<G>(best);
        const int e = least_of<G>(best == most ? lane * PER + at : 0x7fffffff);
        if (most != 0 && lane == j) expert = e;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (e == lane * PER + i) key[i] = 0;
    }
    return expert;
}

// ---- the same choice, nearly always in 32 bits ----------------------------------------------------------------------
//
// A score in fixed point, of 24 bits (22 for more than 256 experts), and the expert's number below it are one word: words
// are sorted in each lane by maxima and minima, the top_k and three more are taken from the lanes' lists by one reduction each,
// and of equal scores the lowest expert comes first.  A score may be off by `margin` / 2 units, so the order of two is known
// where they are further apart, or where they have the same logit and bias.  Where neither holds (about one token in 600),
// the ones taken are put in order by 64 bits; and where that is not enough, all is done by choose_exactly.  16384 tokens, 8 of
// 256 experts in 8 groups, fp32: 20 us, 53 all by choose_exactly; half of it is the time of 1255 vector instructions a wave, the
// rest chains of reductions that wait for each other.  16 of 256 have to go the exact way (61 us; 15 take 37; in one group 40 and
// 32).  8 of 64, 128, 256, 384, 512 and 1024 in one group: 8, 12, 18, 54, 46 and 113, a wave a token from 257 on.
//
// The units cover the whole range of the logits, or of the biases: where a finite one lies far from the others (a mask of -1e9 or of
// the type's lowest; not -infinity), those are all within a few units, and every token goes the exact way.  8 of 128, softmax, one
// logit in eight of -infinity 8 us, of -1e9 17; 8 of 256 in 8 groups, a bias of -1e9 67.
//
// Lanes: a group of experts has lanes of its own, G / groups (rounded down to a power of two) of them, with `need` experts each.

constexpr int kTaken = 16;   // at most; lane j of a token holds the one taken as number j

// Batcher's sorting by odd-even merges, largest first.
template <int N>
__device__ __forceinline__ void sort(unsigned (&v)[N])
{
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const unsigned a = v[i + j], b = v[i + j + k];
                        v[i + j] = a > b ? a : b;
                        v[i + j + k] = a > b ? b : a;
                    }
}

__device__ __forceinline__ double shuffled(double v, int lane, int width)
{
    return __hiloint2double(__shfl(__double2hiint(v), lane, width), __shfl(__double2loint(v), lane, width));
}

template <typename T, int G, int PER>
struct Fast {
    static constexpr int kNumber = G == 64 ? 10 : 8;    // bits of an expert's number
    static constexpr unsigned kNumbers = (1u << kNumber) - 1;
    const Scores &a;
    const T *row;
    int lane;            // of the token's
    bool by_logit;
    float margin, most, total;   // softmax: the largest logit, and the sum of exponentials less it
    double total64;

    static __device__ __forceinline__ unsigned units_of(unsigned key) { return key >> kNumber; }
    static __device__ __forceinline__ int expert_of(unsigned key) { return (int)(kNumbers - (key & kNumbers)); }
    __device__ __forceinline__ float bias_of(int e) const { return a.bias ? a.bias[e] : 0.0f; }

    // what the choice goes by, in 64 bits
    __device__ __forceinline__ double exact(unsigned key) const
    {
        if (key == 0) return -INFINITY;
        const int e = expert_of(key);
        const double z = (double)(float)row[e];
        if (by_logit) return z;
        const double s = a.score == PF_SCORE_SOFTMAX ? exp(z - (double)most) / total64 : 1.0 / (1.0 + exp(-z));
        return s + (double)bias_of(e);
    }
    __device__ __forceinline__ void sum_exactly(bool is)
    {
        if (a.score != PF_SCORE_SOFTMAX || by_logit) return;
        double t = 0;
#pragma unroll 1
        for (int e = lane; e < a.experts; e += G) t += is ? exp((double)(float)row[e] - (double)most) : 0.0;
        total64 = sum_of64<G>(t);
    }

    // Lane j gets the expert taken as number j, or -1; false in `sure` for a token that this cannot decide.
    __device__ __forceinline__ int choose(bool is, bool &sure)
    {
        const int lanes = a.group_lanes, mine = lane / lanes, from = lane % lanes * a.need;
        const int first = mine * a.group_size + from, have = mine < a.groups ? min(a.need, a.group_size - from) : 0;
        float z[PER], b[PER];
        if (a.vector) {
            constexpr int EACH = 16 / sizeof(T);
            typedef T piece __attribute__((ext_vector_type(EACH)));
#pragma unroll
            for (int i = 0; i < PER; i += EACH) {
                const piece v = *(const piece *)(row + min(first + i, a.experts - EACH));   // what is not the lane's is loaded too
#pragma unroll
                for (int c = 0; c < EACH && i + c < PER; ++c) z[i + c] = is && i + c < have ? (float)v[c] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float v = (float)row[min(first + i, a.experts - 1)];
                z[i] = is && i < have ? v : -INFINITY;
            }
        }
        // the largest and the smallest that can be chosen, of the logits and of the biases
        bool odd = false;
        float low = INFINITY, high = -INFINITY;
        most = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            odd |= !(z[i] < INFINITY);
            most = fmaxf(most, z[i]);
        }
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float v = a.bias[min(first + i, a.experts - 1)];
                b[i] = i < have ? v : -INFINITY;
                odd |= !(b[i] < INFINITY);
                low = fminf(low, b[i] > -INFINITY ? b[i] : INFINITY);
                high = fmaxf(high, b[i]);
            }
        } else if (by_logit) {
#pragma unroll
            for (int i = 0; i < PER; ++i) low = fminf(low, z[i] > -INFINITY ? z[i] : INFINITY);
            high = most;
        }
        most = most_of_floats<G>(most);
        if (!(most > -INFINITY)) most = 0;
        float scale, shift = 0;
        constexpr float kUnits = (float)((1 << (32 - kNumber)) - 3);
        if (a.bias || by_logit) {
            low = -most_of_floats<G>(-low);
            high = most_of_floats<G>(high);
            const float range = high > low ? high - low : 0.0f;
            odd |= !(range < INFINITY);
            shift = low;
            scale = by_logit ? (range > 0 ? kUnits / range : 0.0f) : kUnits / (1.0f + range);
            odd |= !(scale < INFINITY);
            // around a far level sums of 64 bits may be equal where scores are not: two groups' sums are off by up to 4 levels 2^-52,
            // which stays under the 2 margins of 24 units that tell them apart
            if (!by_logit) odd |= fmaxf(fabsf(low), fabsf(high)) > 0x1p30f * (1.0f + range);
        } else {
            scale = kUnits;
        }
        constexpr float kLog2e = 0x1.715476p+0f;
        total = 1;
        if (a.score == PF_SCORE_SOFTMAX && (!by_logit || !a.normalise)) {
            float t = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) t += __builtin_amdgcn_exp2f((z[i] - most) * kLog2e);
            total = sum_of<G>(t);
        }
        const float over = total > 0 ? 1.0f / total : 0.0f;
        unsigned key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            float v;
            if (by_logit) {
                v = z[i] - shift;
            } else {
                v = a.score == PF_SCORE_SOFTMAX ? __builtin_amdgcn_exp2f((z[i] - most) * kLog2e) * over
                                                : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z[i] * -kLog2e));
                if (a.bias) v += b[i] - shift;
            }
            const bool can = z[i] > -INFINITY && (!a.bias || b[i] > -INFINITY);
            key[i] = can ? ((unsigned)(v * scale) + 1) << kNumber | (kNumbers - (unsigned)(first + i)) : 0;
        }
        sort(key);
        sure = true;
        if (a.groups > 1) {
            unsigned one = key[0], two = key[1], three = key[2];
            const auto merge = [&](unsigned x, unsigned y, unsigned w) {
                const unsigned t = min(one, x), u = max(two, y);
                one = max(one, x);
                two = max(t, u);
                three = max(min(t, u), max(three, w));
            };
#define PF_MERGE(CTRL) merge(pfdev::dpp<CTRL>(one), pfdev::dpp<CTRL>(two), pfdev::dpp<CTRL>(three))
            if (lanes > 1) PF_MERGE(pfdev::kDppXor1);
            if (lanes > 2) PF_MERGE(pfdev::kDppXor2);
            if (lanes > 4) PF_MERGE(pfdev::kDppHalfMirror);
            if (lanes > 8) PF_MERGE(pfdev::kDppMirror);
#undef PF_MERGE
            if constexpr (G == 64) {
                if (lanes > 16) {
                    constexpr int kFar = pfdev::swizzle_xor_pattern<16>();
                    merge((unsigned)__builtin_amdgcn_ds_swizzle((int)one, kFar), (unsigned)__builtin_amdgcn_ds_swizzle((int)two, kFar),
                          (unsigned)__builtin_amdgcn_ds_swizzle((int)three, kFar));
                }
            }
            // 0 for a group of which nothing can be chosen; where a second score is missing, what a score of 0 has for units
            unsigned value = one ? (1u << 30) + units_of(one) : 0;
            if (a.best == 2 && one)
                value += two ? units_of(two) : (unsigned)((int)fminf(fmaxf(-shift * scale, -0x1p29f), 0x1p29f) + 1);
            int rank = 0;
            for (int g = 0; g < a.groups; ++g) {
                const unsigned other = (unsigned)__shfl((int)value, g * lanes, G);
                rank += other > value || (other == value && g < mine);
            }
            const bool in = mine < a.groups;
            const unsigned out = most_of<G>(in && rank >= a.kept ? value : 0), least = ~most_of<G>(in && rank < a.kept ? ~value : 0);
            const bool near = out != 0 && least - out <= 2 * margin;
            if (__any(near)) {
                sum_exactly(is);
                double x = exact(one), y = exact(two), w = exact(three);
                if (y > x) { const double t = x; x = y; y = t; }
                if (w > x) { const double t = x; x = w; w = t; }
                if (w > y) y = w;
                if (a.best == 2 && y > -INFINITY) x += y;
                // a fourth may be as near as the third
                if (near && three != 0 && units_of(a.best == 2 ? two : one) - units_of(three) <= margin) sure = false;
                int again = 0;
                for (int g = 0; g < a.groups; ++g) {
                    const double other = shuffled(x, g * lanes, G);
                    again += other > x || (other == x && g < mine);
                }
                if (near) rank = again;
            }
            if (!(in && rank < a.kept)) {
#pragma unroll
                for (int i = 0; i < PER; ++i) key[i] = 0;
            }
        }
        unsigned taken = 0;
        const int count = min(a.top_k + 3, kTaken);
        for (int j = 0; j < count; ++j) {
            const unsigned best = most_of<G>(key[0]);
            if (lane == j) taken = best;
            // by masks: of a choice between two elements the compiler makes one between all
            const unsigned pop = key[0] == best ? ~0u : 0u;
#pragma unroll
            for (int i = 0; i + 1 < PER; ++i) key[i] = (key[i + 1] & pop) | (key[i] & ~pop);
            key[PER - 1] &= ~pop;
        }
        // the one behind each, in the next lane
        const unsigned next = (unsigned)__builtin_amdgcn_update_dpp(0, (int)taken, 0x101, 0xf, 0xf, true);   // row_shl 1
        const bool close = taken != 0 && next != 0 && lane + 1 < count && units_of(taken) - units_of(next) <= margin;
        const unsigned long long all = G == 64 ? ~0ull : ((1ull << G) - 1) << ((threadIdx.x & (kWave - 1)) / G * G);
        unsigned long long off = __ballot(odd) & all;
        if (__any(close)) {
            bool alike = true;
            if (close) {
                const int e = expert_of(taken), f = expert_of(next);
                alike = (float)row[e] == (float)row[f] && bias_of(e) == bias_of(f);
            }
            // up to the first gap behind the top_k: what lies behind that gap lies behind all before it
            const unsigned long long apart = __ballot(lane >= a.top_k - 1 && lane + 1 < count && !close) & all;
            const unsigned long long unlike = __ballot(!alike) & all & ((apart & (0 - apart)) - 1);
            if (!apart) off |= all;
            if (__any(unlike != 0)) {
                sum_exactly(is);
                const int e = expert_of(taken);
                const double x = lane < count ? exact(taken) : -INFINITY;
                int rank = 0;
                for (int j = 0; j < count; ++j) {
                    const double other = shuffled(x, j, G);
                    const int f = __shfl(e, j, G);
                    const bool there = __shfl((int)taken, j, G) != 0;
                    rank += there && (taken == 0 || other > x || (other == x && f < e));
                }
                if (taken == 0 || lane >= count) rank = lane;
                const int base = (threadIdx.x & (kWave - 1)) / G * G;
                const unsigned moved = (unsigned)__builtin_amdgcn_ds_permute(4 * (base + rank), (int)taken);
                if (unlike) taken = moved;
            }
        }
        sure = (__ballot(!sure) & all) == 0 && off == 0;
        return taken != 0 ? expert_of(taken) : -1;
    }
};

template <typename T, int G, int PER>
__device__ __forceinline__ void choose(const Scores &a, int t, bool is, unsigned long long *mask)
{
    const int lane = threadIdx.x % G, local = t & (kBlock - 1);
    const T *row = (const T *)a.logits + a.ld * (is ? t : 0);
    const bool by_logit = !a.bias && (a.groups == 1 || a.best == 1);
    Fast<T, G, PER> fast = {a, row, lane, by_logit, by_logit ? 8.0f : a.score == PF_SCORE_SOFTMAX ? 96.0f : 24.0f};
    bool sure = false;
    int expert = -1;
    if (a.need > 0) expert = fast.choose(is, sure);
    if (__any(is && !sure)) {
        float z[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            z[i] = is && e < a.experts ? (float)row[e] : -INFINITY;
        }
        const int exactly = choose_exactly<G, PER>(a, z);
        if (!sure) expert = exactly;
    }
    const bool has = is && expert >= 0 && lane < a.top_k;
    const float mine = has ? (float)row[expert] : -INFINITY;
    float part, total;
    if (a.score == PF_SCORE_SIGMOID) {
        // with the largest chosen logit m < 0 all are formed times exp(-m): their ratio, also where they are no normal numbers
        const float m = a.normalise ? fminf(most_of_floats<G>(mine), 0.0f) : 0.0f;
        part = !has ? 0.0f : mine > 0 ? 1.0f / (1.0f + expf(-mine)) : expf(mine - m) / (1.0f + expf(mine));
        total = a.normalise ? sum_of<G>(part) : 1.0f;
    } else if (a.normalise) {
        const float m = most_of_floats<G>(mine);   // of all lanes, before any parts
        part = has ? expf(mine - m) : 0.0f;
        total = sum_of<G>(part);
    } else {
        float m = -INFINITY;
        total = 0;
        if (__any(is && !sure)) {
#pragma unroll 1
            for (int e = lane; e < a.experts; e += G) m = is ? fmaxf(m, (float)row[e]) : m;
            m = most_of_floats<G>(m);
#pragma unroll 1
            for (int e = lane; e < a.experts; e += G) {
                const float z = is ? (float)row[e] : -INFINITY;
                total += z == -INFINITY ? 0.0f : expf(z - m);
            }
            total = sum_of<G>(total);
        }
        if (sure) {
            m = fast.most;
            total = fast.total;
        }
        part = has ? expf(mine - m) : 0.0f;
    }
    if (is && lane < a.top_k) {
        const long long at = (long long)t * a.top_k + lane;
        a.choice[at] = has ? expert : -1;
        a.weight[at] = has ? a.scale * (part / total) : 0.0f;
        if (has) atomicOr(mask + expert, 1ull << local);
    }
}

template <typename T, int G, int PER>
__global__ __launch_bounds__(1024) void k_route_scores(const Scores a)
{
    route_block<G, PER * G>(a, [&](int t, bool is, unsigned long long *mask) { choose<T, G, PER>(a, t, is, mask); });
}

// ---- the gradient -------------------------------------------------------------------------------------------------

constexpr int kTokens = 16;   // a workgroup's, 16 lanes each

struct Backward {
    const void *logits;
    long long ld, ld_d;
    int tokens, experts, top_k, score, normalise;
    float scale;
    const int *choice;
    const float *weight, *dweight;
    void *dlogits;
};

// Few of a row's elements are not zero (but for softmax over all): rows are put together in LDS and stored as they lie (16384 x 256
// fp32: 6.5 us, 2.6 TB/s of writes).
template <typename T>
__global__ __launch_bounds__(256) void k_scores_backward(const Backward a)
{
    extern __shared__ __align__(16) char image[];
    const int per = (a.experts * (int)sizeof(T) + 15) / 16 * 16 / (int)sizeof(T);   // elements between rows
    T *rows = (T *)image;
    const long long t0 = (long long)blockIdx.x * kTokens;
    const int have = (int)(a.tokens - t0 < kTokens ? a.tokens - t0 : kTokens);
    const int lane = threadIdx.x % 16, local = threadIdx.x / 16;
    const long long t = t0 + local;
    const bool is = local < have;
    const T *z = (const T *)a.logits + a.ld * t;
    int e = -1;
    float w = 0, g = 0;
    if (is && lane < a.top_k) {
        const long long at = t * a.top_k + lane;
        e = a.choice[at];
        if ((unsigned)e >= (unsigned)a.experts) e = -1;
        if (e >= 0) { w = a.weight[at]; g = a.dweight[at]; }
    }
    // the mean of what the weights get, by shares of 1: where one expert has all of it, it gets exactly 0
    const float inner = sum_of<16>((a.normalise ? w / a.scale : w) * g);
    float grad = w * (a.normalise ? g - inner : g);
    if (a.score == PF_SCORE_SIGMOID && e >= 0) {
        const float mine = (float)z[e];   // 1 - s
        grad *= mine > 0 ? expf(-mine) / (1.0f + expf(-mine)) : 1.0f / (1.0f + expf(mine));
    }
    if (a.score == PF_SCORE_SOFTMAX && !a.normalise) {
        float most = -INFINITY, total = 0;
        if (is)
            for (int c = lane; c < a.experts; c += 16) most = fmaxf(most, (float)z[c]);
        most = most_of_floats<16>(most);
        const float base = most > -INFINITY ? most : 0.0f;
        if (is)
            for (int c = lane; c < a.experts; c += 16) total += expf((float)z[c] - base);
        total = sum_of<16>(total);
        const auto all = [&](int c) {
            const float p = expf((float)z[c] - base);
            return p == 0.0f ? 0.0f : -p / total * inner;
        };
        if (is)
            for (int c = lane; c < a.experts; c += 16) rows[local * per + c] = (T)all(c);
        if (e >= 0) grad += all(e);
    } else {
        for (int i = threadIdx.x; i < kTokens * per * (int)sizeof(T) / 16; i += 256) ((i32x4 *)image)[i] = i32x4{0, 0, 0, 0};
    }
    __syncthreads();
    if (e >= 0) rows[local * per + e] = (T)grad;
    __syncthreads();
    T *out = (T *)a.dlogits + a.ld_d * t0;
    constexpr int EACH = 16 / sizeof(T);
    if (((uintptr_t)out | (unsigned long long)(a.ld_d * sizeof(T))) % 16 == 0 && a.experts % EACH == 0) {
        const int pieces = a.experts / EACH;
        for (int i = threadIdx.x; i < have * pieces; i += 256) {
            const int r = i / pieces, c = i % pieces * EACH;
            *(i32x4 *)(out + a.ld_d * r + c) = *(const i32x4 *)(rows + r * per + c);
        }
    } else {
        for (int i = threadIdx.x; i < have * a.experts; i += 256) {
            const int r = i / a.experts, c = i % a.experts;
            out[a.ld_d * r + c] = rows[r * per + c];
        }
    }
}

// The bias of experts with fewer slots than the mean rises by `rate`, that of those with more falls.
__global__ __launch_bounds__(256) void k_balance(const int *offsets, int experts, float rate, const float *bias, float *next)
{
    for (int e = threadIdx.x; e < experts; e += 256) {
        const long long off = (long long)(offsets[experts] - offsets[0]) - (long long)(offsets[e + 1] - offsets[e]) * experts;
        next[e] = bias[e] + (off > 0 ? rate : off < 0 ? -rate : 0.0f);
    }
}

template <typename T>
int route(Scores a, hipStream_t s)
{
    constexpr int kThreads = 1024;
    // lanes a token and experts a lane: as few as hold all groups in lanes of their own
    int g = 0, per = 0, wide = 1;
    while (wide < a.groups) wide *= 2;
    const auto holds = [&](int lanes, int each) {
        const int need = (a.group_size + lanes / wide - 1) / (lanes / wide);
        if (g || need > each) return;
        g = lanes;
        per = each;
        a.group_lanes = lanes / wide;
        a.need = need;
    };
    holds(16, 4);
    holds(16, 8);
    holds(16, 16);
    holds(64, 8);
    holds(64, 16);
    if (!g) {
        g = 64;
        per = 16;
        a.group_lanes = 1;
    }
    const int each = 16 / (int)sizeof(T);
    if (a.top_k >= kTaken) a.need = 0;   // there would be none behind the last
    a.vector = a.need % each == 0 && a.group_size % each == 0 && (uintptr_t)a.logits % 16 == 0 && a.ld % each == 0;
    in_launches(a.blocks, most_workgroups(kThreads), [&](long long first, long long count) {
        const dim3 grid((unsigned)count), block(kThreads);
        a.first = (int)first;
        if (per == 4 && g == 16) k_route_scores<T, 16, 4><<<grid, block, 0, s>>>(a);
        else if (per == 8 && g == 16) k_route_scores<T, 16, 8><<<grid, block, 0, s>>>(a);
        else if (g == 16) k_route_scores<T, 16, 16><<<grid, block, 0, s>>>(a);
        else if (per == 8) k_route_scores<T, 64, 8><<<grid, block, 0, s>>>(a);
        else k_route_scores<T, 64, 16><<<grid, block, 0, s>>>(a);
    });
    return a.blocks > 1 ? launch_places(a, s) : pfk_internal_launched("k_route_scores");
}

template <typename T>
int backward(Backward a, hipStream_t s)
{
    const size_t lds = (size_t)kTokens * ((a.experts * sizeof(T) + 15) / 16 * 16);
    const Backward all = a;
    in_launches(a.tokens, most_workgroups(256) * kTokens, [&](long long first, long long count) {
        a.logits = (const T *)all.logits + a.ld * first;
        a.dlogits = (T *)all.dlogits + a.ld_d * first;
        a.choice = all.choice + first * a.top_k;
        a.weight = all.weight + first * a.top_k;
        a.dweight = all.dweight + first * a.top_k;
        a.tokens = (int)count;
        k_scores_backward<T><<<dim3((unsigned)((count + kTokens - 1) / kTokens)), dim3(256), lds, s>>>(a);
    });
    return pfk_internal_launched("k_scores_backward");
}

}  // namespace

extern "C" {

int pfk_moe_route_scores(const void *logits, long long ld, int dtype, int tokens, int experts, int top_k, int score, const float *bias,
                         int groups, int groups_kept, int group_best, int normalise, float scale, int *choice, float *weight,
                         int *offsets, int *order, int *slot, int *counts, void *stream)
{
    Scores a = {};
    a.logits = logits;
    a.ld = ld;
    a.tokens = tokens;
    a.experts = experts;
    a.top_k = top_k;
    a.normalise = normalise;
    a.blocks = (int)PFK_MOE_ROUTE_BLOCKS(tokens);
    a.choice = choice;
    a.weight = weight;
    a.offsets = offsets;
    a.order = order;
    a.slot = slot;
    if (a.blocks < 1) a.blocks = 1;
    if (a.blocks > 1) a.counts = (unsigned char *)counts;
    if (PFK_MOE_ROUTE_SUPER_WORDS(a.blocks, experts) > 0) a.super = counts + PFK_MOE_ROUTE_COUNT_WORDS(a.blocks, experts);
    a.score = score;
    a.groups = groups;
    a.group_size = experts / groups;
    a.kept = groups_kept;
    a.best = group_best;
    a.bias = bias;
    a.scale = scale;
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F32 ? route<float>(a, s) : dtype == PF_F16 ? route<f16>(a, s) : route<bf16>(a, s);
}

int pfk_moe_route_scores_backward(const void *logits, long long ld, int dtype, int tokens, int experts, int top_k, int score,
                                  int normalise, float scale, const int *choice, const float *weight, const float *dweight,
                                  void *dlogits, long long ld_d, void *stream)
{
    const Backward a = {logits, ld, ld_d, tokens, experts, top_k, score, normalise, scale, choice, weight, dweight, dlogits};
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F32 ? backward<float>(a, s) : dtype == PF_F16 ? backward<f16>(a, s) : backward<bf16>(a, s);
}

int pfk_moe_balance(const int *offsets, int experts, float rate, const float *bias, float *next, void *stream)
{
    k_balance<<<dim3(1), dim3(256), 0, (hipStream_t)stream>>>(offsets, experts, rate, bias, next);
    return pfk_internal_launched("k_balance");
}

}  // extern "C"
