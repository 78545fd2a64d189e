// moe_route.hip — routing of an expert layer on gfx950 (include/prefree_moe.h): the choice of experts and their order,
// the weighted sum of the experts' rows, and the gradients of both.
#include "moe_route.hpp"

namespace {

using namespace pfmoe;

template <typename T>
__device__ __forceinline__ float as_float(T v) { return (float)v; }

// Order-preserving key of a logit: 0 for -infinity (never chosen), the largest for NaN, -0 and 0 alike.
__device__ __forceinline__ unsigned key_of(float z)
{
    if (z != z) return 0xffffffffu;
    if (z == 0.0f) z = 0.0f;
    const unsigned b = __float_as_uint(z);
    if (b == 0xff800000u) return 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// and back: NaN for the largest key, -infinity for 0
__device__ __forceinline__ float logit_of(unsigned key)
{
    if (key == 0) return -INFINITY;
    return __uint_as_float(key & 0x80000000u && key != 0xffffffffu ? key & 0x7fffffffu : key == 0xffffffffu ? 0x7fc00000u : ~key);
}

// G lanes take a token: lane l of them has logits l*PER .. l*PER + PER-1 in registers, and each choice is the largest
// key among them, at its lowest index.  With 16 lanes a token that takes shifts inside a row of lanes only, a block of 64
// tokens at once (16384 tokens, 8 of 128, fp32: 9.5 us, 21 with a wave a token; bound by the chain of top_k searches).
template <typename T, int G, int PER>
__device__ __forceinline__ void choose(const Route &a, int t, bool is, unsigned long long *mask)
{
    const int lane = threadIdx.x % G, local = t & (kBlock - 1);
    const T *row = (const T *)a.logits + a.ld * t;
    float z[PER];
    unsigned key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        z[i] = is && e < a.experts ? as_float(row[e]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = key_of(z[i]);
    unsigned mine = 0, top = 0;   // lane j: the key of choice j; the row's largest
    int expert = -1;
    for (int j = 0; j < a.top_k; ++j) {
        unsigned best = 0;
        int at = 0;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i)
            if (key[i] >= best) { best = key[i]; at = i; }
        const unsigned most = most_of<G>(best);
        const int e = least_of<G>(best == most ? lane * PER + at : 0x7fffffff);
        if (j == 0) top = most;
        if (most != 0 && lane == j) { mine = most; expert = e; }
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (e == lane * PER + i) key[i] = 0;
    }
    const float best = logit_of(top);
    const float part = expert >= 0 ? expf(logit_of(mine) - best) : 0.0f;
    float total = part;
    if (!a.normalise) {
        total = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) total += expf(z[i] - best);
    }
    total = sum_of<G>(total);
    if (is && lane < a.top_k) {
        const long long at = (long long)t * a.top_k + lane;
        a.choice[at] = expert;
        a.weight[at] = expert >= 0 ? part / total : 0.0f;
        if (expert >= 0) atomicOr(mask + expert, 1ull << local);
    }
}

// Choice and weights; with one block also offsets and order, else the block's counts.
template <typename T, int G, int PER>
__global__ __launch_bounds__(1024) void k_route(const Route a)
{
    route_block<G, PER * G>(a, [&](int t, bool is, unsigned long long *mask) { choose<T, G, PER>(a, t, is, mask); });
}

// Sums of kSuper blocks' counts each, for many blocks.
__global__ __launch_bounds__(256) void k_route_super(const Route a)
{
    const int begin = blockIdx.x * kSuper, end = min(a.blocks, begin + kSuper), ld = counts_ld(a.experts);
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        int n = 0;
        for (int b = begin; b < end; ++b) n += a.counts[(long long)b * ld + e];
        a.super[(long long)blockIdx.x * a.experts + e] = n;
    }
}

// Offsets and order from the counts: each workgroup sums all blocks' counts, and those before its own.  A thread sums
// words of four experts' counts, as two pairs of 16 bits: of at most 1024 blocks with 64 tokens each, shared out over
// the groups of threads (at least four), that is less than 2^16.  256 blocks, 128 experts: 5.4 us, 20 with a byte a load;
// every workgroup reads all counts out of the L2, which saves a launch and a wait for one workgroup's sums.  No more than 64
// groups: each adds to its experts' sums in LDS, one after the other (466 blocks, 4 experts: 18 us with 1024 of them).
__global__ __launch_bounds__(1024) void k_route_place(const Route a)
{
    extern __shared__ unsigned long long lds[];
    unsigned long long *mask = lds;
    int *total = (int *)(lds + a.experts), *before = total + a.experts, *first = before + a.experts, *used = first + a.experts;
    const int block = a.first + blockIdx.x;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        mask[e] = 0;
        total[e] = before[e] = 0;
    }
    __syncthreads();
    const int begin = block * kBlock, entries = min(kBlock, a.tokens - begin) * a.top_k;
    for (int i = threadIdx.x; i < entries; i += blockDim.x) {
        const int e = a.choice[(long long)begin * a.top_k + i];
        if (e >= 0) atomicOr(mask + e, 1ull << (i / a.top_k));
    }
    // integer sums, so the order in which they are added does not matter
    const int words = counts_ld(a.experts) / 4, groups = min((int)blockDim.x / words, 64), group = threadIdx.x / words, word = threadIdx.x % words;
    const int supers = a.super ? a.blocks / kSuper : 0, own = block / kSuper;
    if (group < groups) {
        unsigned all[2] = {0, 0}, prior[2] = {0, 0};
        const unsigned *counts = (const unsigned *)a.counts + word;
        const auto add = [](unsigned (&to)[2], unsigned v) {
            to[0] += v & 0x00ff00ffu;
            to[1] += v >> 8 & 0x00ff00ffu;
        };
#pragma unroll 8
        for (int b = supers * kSuper + group; b < a.blocks; b += groups) {
            const unsigned v = counts[(long long)b * words];
            add(all, v);
            add(prior, b < block ? v : 0);
        }
        if (own < supers) {
#pragma unroll 8
            for (int b = own * kSuper + group; b < block; b += groups) add(prior, counts[(long long)b * words]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = word * 4 + i;
            if (e >= a.experts) break;
            atomicAdd(total + e, (int)(all[i & 1] >> (i & 2) * 8 & 0xffff));
            atomicAdd(before + e, (int)(prior[i & 1] >> (i & 2) * 8 & 0xffff));
        }
    }
    const int shares = blockDim.x / a.experts, share = threadIdx.x / a.experts, e = threadIdx.x % a.experts;
    if (supers > 0 && share < shares) {
        int all = 0, prior = 0;
        for (int i = share; i < supers; i += shares) {
            const int v = a.super[(long long)i * a.experts + e];
            all += v;
            if (i < own) prior += v;
        }
        atomicAdd(total + e, all);
        atomicAdd(before + e, prior);
    }
    __syncthreads();
    if (threadIdx.x < kWave) {
        const int n = scan_experts(total, first, a.experts);
        if (threadIdx.x == 0) *used = n;
    }
    __syncthreads();
    if (block == 0) {
        for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.offsets[e] = first[e];
        if (threadIdx.x == 0) a.offsets[a.experts] = *used;
        __syncthreads();
    }
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) first[e] += before[e];
    __syncthreads();
    place(a, block, mask, first, *used);
}

// dz = w (g - sum w g) at the chosen under `normalise`, else [chosen] w g - p sum w g.  One wave a token: 16384 tokens of
// 128 experts, fp32, in 7.3 us, 8.4 MB of it written.
template <typename T, int PER>
__global__ __launch_bounds__(256) void k_route_backward(const T *logits, long long ld, int tokens, int experts, int top_k,
                                                        int normalise, const int *choice, const float *weight,
                                                        const float *dweight, T *dlogits, long long ld_d)
{
    const int lane = threadIdx.x & (kWave - 1), t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= tokens) return;
    int e = -1;
    float w = 0, g = 0;
    if (lane < top_k) {
        const long long at = (long long)t * top_k + lane;
        e = choice[at];
        if (e >= 0) { w = weight[at]; g = dweight[at]; }
    }
    const float inner = pfdev::wave_sum(w * g);
    const float grad = normalise ? w * (g - inner) : w * g;
    float p[PER], d[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) p[i] = d[i] = 0;
    if (!normalise) {
        float most = -INFINITY, sum = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = lane * PER + i;
            p[i] = c < experts ? as_float(logits[ld * t + c]) : -INFINITY;
            most = fmaxf(most, p[i]);
        }
        for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
        const float base = most > -INFINITY ? most : 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += p[i] = expf(p[i] - base);
        sum = pfdev::wave_sum(sum);
#pragma unroll
        for (int i = 0; i < PER; ++i) d[i] = p[i] == 0.0f ? 0.0f : -p[i] / sum * inner;
    }
    for (int j = 0; j < top_k; ++j) {
        const int ej = __builtin_amdgcn_readlane(e, j);
        const float gj = pfdev::readlane(grad, j);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (ej == lane * PER + i) d[i] += gj;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = lane * PER + i;
        if (c < experts) dlogits[ld_d * t + c] = (T)d[i];
    }
}

// Eight elements of a row from `at`, those behind its end as zeros; VECTOR: rows of whole 16-byte pieces.
template <typename T, bool VECTOR>
__device__ __forceinline__ void load8(const T *row, int at, int have, float v[8])
{
    if (VECTOR || at + 8 <= have) {
        typedef typename vec<T>::x8 x8;
        const x8 h = VECTOR ? *(const x8 *)(row + at) : __builtin_bit_cast(x8, load16_any(row + at));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = at + i < have ? (float)row[at + i] : 0.0f;
    }
}

template <typename T, bool VECTOR>
__device__ __forceinline__ void store8(T *row, int at, int have, const float v[8])
{
    if (VECTOR || at + 8 <= have) {
        typename vec<T>::x8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (T)v[i];
        if (VECTOR) *(typename vec<T>::x8 *)(row + at) = h;
        else __builtin_memcpy(row + at, &h, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < have) row[at + i] = (T)v[i];
    }
}

// out[t] = sum of w y[slot]: a wave takes 512 columns of a token, so that a few tokens already fill many waves.  Bound by
// reading y: 8191 tokens x 4, 2048 columns, 168 MB in 26.5 us with part of it in cache, 35.5 without.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_combine(const T *y, long long ld_y, int slots, const int *slot, const float *weight,
                                                 int tokens, int top_k, int width, T *out, long long ld_out, int parts)
{
    const int lane = threadIdx.x & (kWave - 1);
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (long long)tokens * parts) return;
    const int t = (int)(unit / parts), at = (int)(unit % parts) * 512 + lane * 8;
    int s = -1;
    float w = 0;
    if (lane < top_k) {
        s = slot[(long long)t * top_k + lane];
        if ((unsigned)s >= (unsigned)slots) s = -1;
        w = s < 0 ? 0.0f : weight ? weight[(long long)t * top_k + lane] : 1.0f;
    }
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j = 0; j < top_k; ++j) {
        const int sj = __builtin_amdgcn_readlane(s, j);
        const float wj = pfdev::readlane(w, j);
        if (sj < 0 || at >= width) continue;
        float v[8];
        load8<T, VECTOR>(y + ld_y * sj, at, width, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = __builtin_fmaf(wj, v[i], sum[i]);
    }
    if (at < width) store8<T, VECTOR>(out + ld_out * t, at, width, sum);
}

// dy[slot] = w dout[t], dweight = <dout[t], y[slot]>: a workgroup a token, which reads dout[t] once for all its slots.
// Bound by y and dy: 8191 tokens x 4, 2048 columns, 302 MB in 49 us with part of it in cache, 60 without.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_combine_backward(const T *dout, long long ld_dout, const T *y, long long ld_y,
                                                          int slots, const int *slot, const float *weight, int top_k,
                                                          int width, T *dy, long long ld_dy, float *dweight)
{
    __shared__ float part[4][PF_MOE_MAX_TOP_K];
    const int t = blockIdx.x, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    int s = -1;
    float w = 0;
    if (lane < top_k) {
        s = slot[(long long)t * top_k + lane];
        if ((unsigned)s >= (unsigned)slots) s = -1;
        w = s < 0 ? 0.0f : weight ? weight[(long long)t * top_k + lane] : 1.0f;
    }
    float dot[PF_MOE_MAX_TOP_K];
#pragma unroll
    for (int j = 0; j < PF_MOE_MAX_TOP_K; ++j) dot[j] = 0;
    for (int begin = 0; begin < width; begin += 2048) {
        const int at = begin + threadIdx.x * 8;
        const bool in = at < width;
        float g[8];
        if (in) load8<T, VECTOR>(dout + ld_dout * t, at, width, g);
#pragma unroll
        for (int j = 0; j < PF_MOE_MAX_TOP_K; ++j) {
            const int sj = __builtin_amdgcn_readlane(s, j);
            const float wj = pfdev::readlane(w, j);
            if (sj >= 0 && in) {
                float v[8], d[8];
                load8<T, VECTOR>(y + ld_y * sj, at, width, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    dot[j] = __builtin_fmaf(g[i], v[i], dot[j]);
                    d[i] = wj * g[i];
                }
                store8<T, VECTOR>(dy + ld_dy * sj, at, width, d);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < PF_MOE_MAX_TOP_K; ++j) {
        const float sum = pfdev::wave_sum(dot[j]);
        if (lane == 0) part[wave][j] = sum;
    }
    __syncthreads();
    if ((int)threadIdx.x < top_k)
        dweight[(long long)t * top_k + threadIdx.x] =
            (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
}

// h = silu(g) u: dg = dh u s (1 + g (1 - s)), du = dh g s, with s = sigmoid(g).  32768 x 2048, 403
// MB read and 268 written, in 116 us, 5.8 TB/s; rows that do not lie in 16 bytes (32764 x 1023) at 3.6 TB/s.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_swiglu_backward(const T *dh, long long ld_dh, const T *pre, long long ld_pre, int rows,
                                                         int n, T *dpre, long long ld_dpre, int parts)
{
    const long long unit = (long long)blockIdx.x * 256 + threadIdx.x;
    if (unit >= (long long)rows * parts) return;
    const long long r = unit / parts;
    const int at = (int)(unit % parts) * 8;
    float d[8], g[8], u[8], dg[8], du[8];
    load8<T, VECTOR>(dh + ld_dh * r, at, n, d);
    load8<T, VECTOR>(pre + ld_pre * r, at, n, g);
    load8<T, VECTOR>(pre + ld_pre * r + n, at, n, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = 1.0f / inverse_sigmoid(g[i]);   // over kUnder
        dg[i] = d[i] * u[i] * kUnder * s * (1.0f + g[i] * (1.0f - kUnder * s));
        du[i] = d[i] * (g[i] * kUnder) * s;
    }
    store8<T, VECTOR>(dpre + ld_dpre * r, at, n, dg);
    store8<T, VECTOR>(dpre + ld_dpre * r + n, at, n, du);
}

template <typename T>
int route(Route a, hipStream_t s)
{
    constexpr int kThreads = 1024;
    in_launches(a.blocks, most_workgroups(kThreads), [&](long long first, long long count) {
        const dim3 grid((unsigned)count), block(kThreads);
        a.first = (int)first;
        if (a.experts <= 64) k_route<T, 16, 4><<<grid, block, 0, s>>>(a);
        else if (a.experts <= 128) k_route<T, 16, 8><<<grid, block, 0, s>>>(a);
        else if (a.experts <= 256) k_route<T, 16, 16><<<grid, block, 0, s>>>(a);
        else if (a.experts <= 512) k_route<T, 64, 8><<<grid, block, 0, s>>>(a);
        else k_route<T, 64, 16><<<grid, block, 0, s>>>(a);
    });
    return a.blocks > 1 ? launch_places(a, s) : pfk_internal_launched("k_route");
}

template <typename T>
int route_backward(const void *logits, long long ld, int tokens, int experts, int top_k, int normalise, const int *choice,
                   const float *weight, const float *dweight, void *dlogits, long long ld_d, hipStream_t s)
{
    in_launches(tokens, most_workgroups(256) * 4, [&](long long first, long long count) {
        const dim3 grid((unsigned)((count + 3) / 4)), block(256);
        const T *z = (const T *)logits + ld * first;
        T *dz = (T *)dlogits + ld_d * first;
        const long long at = first * top_k;
#define PFK_BACKWARD(PER)                                                                                                  \
    k_route_backward<T, PER><<<grid, block, 0, s>>>(z, ld, (int)count, experts, top_k, normalise, choice + at, weight + at, \
                                                    dweight + at, dz, ld_d)
        if (experts <= 64) PFK_BACKWARD(1);
        else if (experts <= 128) PFK_BACKWARD(2);
        else if (experts <= 256) PFK_BACKWARD(4);
        else if (experts <= 512) PFK_BACKWARD(8);
        else PFK_BACKWARD(16);
#undef PFK_BACKWARD
    });
    return pfk_internal_launched("k_route_backward");
}

// whether rows of 16-bit elements start at, and hold, whole 16-byte pieces
bool whole(const void *p, long long ld, int width) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && width % 8 == 0; }

template <typename T>
int combine(const void *y, long long ld_y, int slots, const int *slot, const float *weight, int tokens, int top_k, int width,
            void *out, long long ld_out, hipStream_t s)
{
    const int parts = (width + 511) / 512;
    const auto kernel = whole(y, ld_y, width) && whole(out, ld_out, width) ? k_combine<T, true> : k_combine<T, false>;
    in_launches(tokens, most_workgroups(256) * 4 / parts, [&](long long first, long long count) {
        kernel<<<dim3((unsigned)((count * parts + 3) / 4)), dim3(256), 0, s>>>(
            (const T *)y, ld_y, slots, slot + first * top_k, weight ? weight + first * top_k : nullptr, (int)count, top_k, width,
            (T *)out + ld_out * first, ld_out, parts);
    });
    return pfk_internal_launched("k_combine");
}

template <typename T>
int combine_backward(const void *dout, long long ld_dout, const void *y, long long ld_y, int slots, const int *slot,
                     const float *weight, int tokens, int top_k, int width, void *dy, long long ld_dy, float *dweight,
                     hipStream_t s)
{
    const bool vector = whole(dout, ld_dout, width) && whole(y, ld_y, width) && whole(dy, ld_dy, width);
    const auto kernel = vector ? k_combine_backward<T, true> : k_combine_backward<T, false>;
    in_launches(tokens, most_workgroups(256), [&](long long first, long long count) {
        kernel<<<dim3((unsigned)count), dim3(256), 0, s>>>(
            (const T *)dout + ld_dout * first, ld_dout, (const T *)y, ld_y, slots, slot + first * top_k,
            weight ? weight + first * top_k : nullptr, top_k, width, (T *)dy, ld_dy, dweight + first * top_k);
    });
    return pfk_internal_launched("k_combine_backward");
}

template <typename T>
int swiglu_backward(const void *dh, long long ld_dh, const void *pre, long long ld_pre, int rows, int n, void *dpre,
                    long long ld_dpre, hipStream_t s)
{
    const int parts = (n + 7) / 8;
    const bool vector = whole(dh, ld_dh, n) && whole(pre, ld_pre, n) && whole(dpre, ld_dpre, n);
    const auto kernel = vector ? k_swiglu_backward<T, true> : k_swiglu_backward<T, false>;
    in_launches(rows, most_workgroups(256) * 256 / parts, [&](long long first, long long count) {
        kernel<<<dim3((unsigned)((count * parts + 255) / 256)), dim3(256), 0, s>>>(
            (const T *)dh + ld_dh * first, ld_dh, (const T *)pre + ld_pre * first, ld_pre, (int)count, n,
            (T *)dpre + ld_dpre * first, ld_dpre, parts);
    });
    return pfk_internal_launched("k_swiglu_backward");
}

}  // namespace

int pfmoe::launch_places(Route a, hipStream_t s)
{
    constexpr int kThreads = 1024;
    const size_t lds = (size_t)a.experts * 20 + 8;
    if (a.super) k_route_super<<<dim3(a.blocks / kSuper), dim3(256), 0, s>>>(a);
    in_launches(a.blocks, most_workgroups(kThreads), [&](long long first, long long count) {
        a.first = (int)first;
        k_route_place<<<dim3((unsigned)count), dim3(kThreads), lds, s>>>(a);
    });
    return pfk_internal_launched("k_route");
}

extern "C" {

int pfk_moe_route(const void *logits, long long ld, int dtype, int tokens, int experts, int top_k, int normalise,
                  int *choice, float *weight, int *offsets, int *order, int *slot, int *counts, void *stream)
{
    Route a = {logits, ld, tokens, experts, top_k, normalise, (int)PFK_MOE_ROUTE_BLOCKS(tokens), choice, weight, offsets, order, slot, nullptr, nullptr, 0};
    if (a.blocks < 1) a.blocks = 1;
    if (a.blocks > 1) a.counts = (unsigned char *)counts;
    if (PFK_MOE_ROUTE_SUPER_WORDS(a.blocks, experts) > 0) a.super = counts + PFK_MOE_ROUTE_COUNT_WORDS(a.blocks, experts);
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F32 ? route<float>(a, s) : dtype == PF_F16 ? route<f16>(a, s) : route<bf16>(a, s);
}

int pfk_moe_route_backward(const void *logits, long long ld, int dtype, int tokens, int experts, int top_k, int normalise,
                           const int *choice, const float *weight, const float *dweight, void *dlogits, long long ld_d,
                           void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    if (dtype == PF_F32) return route_backward<float>(logits, ld, tokens, experts, top_k, normalise, choice, weight, dweight, dlogits, ld_d, s);
    if (dtype == PF_F16) return route_backward<f16>(logits, ld, tokens, experts, top_k, normalise, choice, weight, dweight, dlogits, ld_d, s);
    return route_backward<bf16>(logits, ld, tokens, experts, top_k, normalise, choice, weight, dweight, dlogits, ld_d, s);
}

int pfk_moe_combine(const void *y, long long ld_y, int dtype, int slots, const int *slot, const float *weight, int tokens,
                    int top_k, int width, void *out, long long ld_out, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F16 ? combine<f16>(y, ld_y, slots, slot, weight, tokens, top_k, width, out, ld_out, s)
                           : combine<bf16>(y, ld_y, slots, slot, weight, tokens, top_k, width, out, ld_out, s);
}

int pfk_moe_combine_backward(const void *dout, long long ld_dout, const void *y, long long ld_y, int dtype, int slots,
                             const int *slot, const float *weight, int tokens, int top_k, int width, void *dy,
                             long long ld_dy, float *dweight, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F16
               ? combine_backward<f16>(dout, ld_dout, y, ld_y, slots, slot, weight, tokens, top_k, width, dy, ld_dy, dweight, s)
               : combine_backward<bf16>(dout, ld_dout, y, ld_y, slots, slot, weight, tokens, top_k, width, dy, ld_dy, dweight, s);
}

int pfk_swiglu_backward(const void *dh, long long ld_dh, const void *pre, long long ld_pre, int dtype, int rows, int n,
                        void *dpre, long long ld_dpre, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F16 ? swiglu_backward<f16>(dh, ld_dh, pre, ld_pre, rows, n, dpre, ld_dpre, s)
                           : swiglu_backward<bf16>(dh, ld_dh, pre, ld_pre, rows, n, dpre, ld_dpre, s);
}

}  // extern "C"
