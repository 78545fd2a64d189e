// moe_route.hpp — what the routing kernels share: a token's lanes, the counts of a block of tokens, places by expert.
#pragma once

#include "moe_common.hpp"
#include "moe_launch.hpp"
#include "prefree_moe_kernels.h"

namespace pfmoe {

constexpr int kBlock = PFK_MOE_ROUTE_BLOCK;  // tokens a workgroup: one bit each in a 64-bit mask of an expert
static_assert(kBlock == 64, "masks of 64 tokens");
constexpr int kSuper = PFK_MOE_ROUTE_SUPER;  // blocks whose counts are summed beforehand, where each workgroup does not sum all

struct Route {
    const void *logits;
    long long ld;
    int tokens, experts, top_k, normalise, blocks;
    int *choice;
    float *weight;
    int *offsets, *order, *slot;
    unsigned char *counts;  // [blocks][counts_ld(experts)]
    int *super;             // [blocks / kSuper][experts], behind the counts
    int first;              // block of the launch's first workgroup
};

// Counts are read four experts a word: their rows are whole words, zeros behind the last expert.
__device__ constexpr int counts_ld(int experts) { return 4 * PFK_MOE_ROUTE_ROW_WORDS(experts); }

// The largest of v, and the smallest of i, over the G = 16 or 64 lanes of a token; every lane has it.
template <int G>
__device__ __forceinline__ unsigned most_of(unsigned v)
{
    const auto op = [](unsigned a, unsigned b) { return a > b ? a : b; };
    v = op(v, pfdev::dpp<pfdev::kDppXor1>(v));
    v = op(v, pfdev::dpp<pfdev::kDppXor2>(v));
    v = op(v, pfdev::dpp<pfdev::kDppHalfMirror>(v));
    v = op(v, pfdev::dpp<pfdev::kDppMirror>(v));
    if constexpr (G == 64) {
        v = op(v, (unsigned)__builtin_amdgcn_ds_swizzle((int)v, pfdev::swizzle_xor_pattern<16>()));
        v = op((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 32));
    }
    return v;
}
template <int G>
__device__ __forceinline__ int least_of(int i) { return (int)~most_of<G>(~(unsigned)i); }
template <int G>
__device__ __forceinline__ float sum_of(float v)
{
    if constexpr (G == 64) return pfdev::wave_sum(v);
    else return pfdev::group_sum<16>(v);
}

// Places the entries of block `block`: mask[e] has a bit for each of its tokens that chose expert e (a token chooses an
// expert once, so the bits below its own count the entries before it), first[e] is the slot of the first of them.
__device__ __forceinline__ void place(const Route &a, int block, const unsigned long long *mask, const int *first,
                                      int used)
{
    const int begin = block * kBlock, entries = min(kBlock, a.tokens - begin) * a.top_k;
    for (int i = threadIdx.x; i < entries; i += blockDim.x) {
        const int f = begin * a.top_k + i, e = a.choice[f], local = i / a.top_k;
        int s = -1;
        if (e >= 0) {
            s = first[e] + __popcll(mask[e] & ((1ull << local) - 1));
            a.order[s] = f;
        }
        a.slot[f] = s;
    }
    // slots that no entry takes
    for (long long s = used + (long long)block * blockDim.x + threadIdx.x; s < (long long)a.tokens * a.top_k;
         s += (long long)a.blocks * blockDim.x)
        a.order[s] = -1;
}

// Exclusive sums over the experts of total[e] into first[e] (in LDS); returns the sum.  One wave.
__device__ __forceinline__ int scan_experts(const int *total, int *first, int experts)
{
    const int lane = threadIdx.x & (kWave - 1);
    int before = 0;
    for (int base = 0; base < experts; base += kWave) {
        const int v = base + lane < experts ? total[base + lane] : 0;
        const int incl = scan_wave(v);
        if (base + lane < experts) first[base + lane] = before + incl - v;
        before += __builtin_amdgcn_readlane(incl, kWave - 1);
    }
    return before;
}

// A block of tokens: choose(t, is, mask) takes a token for each G lanes, and sets the block's bit of each expert chosen.
// With one block also offsets and order, else the block's counts.
template <int G, int EXPERTS, typename F>
__device__ __forceinline__ void route_block(const Route &a, F choose)
{
    __shared__ unsigned long long mask[EXPERTS];
    __shared__ int total[EXPERTS], first[EXPERTS], used;
    const int block = a.first + blockIdx.x;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) mask[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x / G; i < kBlock; i += 1024 / G) {   // whole waves: each lane's group has a token or none
        const int t = block * kBlock + i;
        if (block * kBlock + (i & ~(kWave / G - 1)) < a.tokens) choose(t, t < a.tokens, mask);
    }
    __syncthreads();
    if (a.blocks > 1) {
        const int ld = counts_ld(a.experts);
        for (int e = threadIdx.x; e < ld; e += blockDim.x)
            a.counts[(long long)block * ld + e] = e < a.experts ? (unsigned char)__popcll(mask[e]) : 0;
        return;
    }
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) total[e] = __popcll(mask[e]);
    __syncthreads();
    if (threadIdx.x < kWave) {
        const int n = scan_experts(total, first, a.experts);
        if (threadIdx.x == 0) used = n;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.offsets[e] = first[e];
    if (threadIdx.x == 0) a.offsets[a.experts] = used;
    place(a, block, mask, first, used);
}

// The launches behind the choice where there is more than one block: offsets and order from the counts.
__attribute__((visibility("hidden"))) int launch_places(Route a, hipStream_t s);

}  // namespace pfmoe
