// moe_scores.hip — routing by scores on gfx950 (include/prefree_moe.h): sigmoid or softmax scores plus a bias, groups of
// experts, the gradient of the logits, and the bias's step.
#include "moe_route.hpp"

namespace {

using namespace pfmoe;

struct Scores : Route {
    int score, groups, group_size, kept, best;
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
            const unsigned long long other = (unsigned long long)(unsigned)__shfl((int)(value >> 32), g, G) << 32 | (unsigned)__shfl((int)(unsigned)value, g, G);
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

template <typename T, int G, int PER>
__device__ __forceinline__ void choose(const Scores &a, int t, bool is, unsigned long long *mask)
{
    const int lane = threadIdx.x % G, local = t & (kBlock - 1);
    const T *row = (const T *)a.logits + a.ld * t;
    float z[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        z[i] = is && e < a.experts ? (float)row[e] : -INFINITY;
    }
    const int expert = choose_exactly<G, PER>(a, z);
    const bool has = is && expert >= 0;
    const float mine = has ? (float)row[expert] : -INFINITY;
    float part, total;
    if (a.score == PF_SCORE_SIGMOID) {
        // with the largest chosen logit m < 0 all are formed times exp(-m): their ratio, also where they are no normal numbers
        const float m = a.normalise ? fminf(most_of_floats<G>(mine), 0.0f) : 0.0f;
        part = !has ? 0.0f : mine > 0 ? 1.0f / (1.0f + expf(-mine)) : expf(mine - m) / (1.0f + expf(mine));
        total = a.normalise ? sum_of<G>(part) : 1.0f;
    } else {
        float m = mine;
        if (!a.normalise) {
#pragma unroll
            for (int i = 0; i < PER; ++i) m = fmaxf(m, z[i]);
        }
        m = most_of_floats<G>(m);
        part = has ? expf(mine - m) : 0.0f;
        total = part;
        if (!a.normalise) {
            total = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) total += z[i] > -INFINITY || z[i] != z[i] ? expf(z[i] - m) : 0.0f;
        }
        total = sum_of<G>(total);
    }
    if (is && lane < a.top_k) {
        const long long at = (long long)t * a.top_k + lane;
        a.choice[at] = expert;
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

// Few of a row's elements are not zero (but for softmax over all): rows are put together in LDS and stored as they lie.
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
    const float inner = sum_of<16>(w * g);
    float grad = a.normalise ? w * (g - inner / a.scale) : w * g;
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
    in_launches(a.blocks, most_workgroups(kThreads), [&](long long first, long long count) {
        const dim3 grid((unsigned)count), block(kThreads);
        a.first = (int)first;
        if (a.experts <= 64) k_route_scores<T, 16, 4><<<grid, block, 0, s>>>(a);
        else if (a.experts <= 128) k_route_scores<T, 16, 8><<<grid, block, 0, s>>>(a);
        else if (a.experts <= 256) k_route_scores<T, 16, 16><<<grid, block, 0, s>>>(a);
        else if (a.experts <= 512) k_route_scores<T, 64, 8><<<grid, block, 0, s>>>(a);
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
