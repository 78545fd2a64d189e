// moe_orth.hpp — what the kernels of orthogonal updates share.
#pragma once

#include "moe_common.hpp"
#include "moe_launch.hpp"
#include "prefree_moe_kernels.h"

namespace pfmoe {

constexpr int kParts = PFK_ORTH_PARTS;   // sums of squares of a matrix, at most
constexpr float kRest = 2048.0f;   // the second piece is held times this: about as large as the first, whose exponents it has

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

// N results from column c of a row of the result
template <typename T, int N>
__device__ __forceinline__ void store_row(T *row, int c, int columns, bool wide, const float v[N])
{
    T h[N];
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = (T)v[i];
    typedef T vec_t __attribute__((ext_vector_type(8)));
    typedef vec_t any_t __attribute__((aligned(sizeof(T))));   // one store too, of any address
    if (c + N <= columns) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            vec_t b;
            __builtin_memcpy(&b, h + i, 16);
            if (wide) *(vec_t *)(row + c + i) = b;
            else *(any_t *)(row + c + i) = b;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < columns) row[c + i] = h[i];
    }
}

// scale / |G|; no number for a matrix that holds none, and 0 for one of zeros
__device__ __forceinline__ double over_norm(const double *sums, int parts, float scale)
{
    const int lane = threadIdx.x & (kWave - 1);
    double sum = lane < parts ? sums[lane] : 0;
    static_assert(kParts <= kWave, "a lane each");
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    return !(sum < INFINITY) ? (double)NAN : sum > 0 ? scale / __builtin_sqrt(sum) : 0.0;
}

// An update of matrices whose shorter side is at most PFK_ORTH_NARROW (moe_orth_narrow.hip); X is held times `scale`.
struct Narrow {
    const void *g;
    long long ld_g, ld_out;
    int dtype, batch, rows, columns, n_steps, out_f16;
    const float *steps;
    float scale;
    const double *sums;    // of squares, `parts` a matrix
    int parts;
    void *out, *workspace;
};
__attribute__((visibility("hidden"))) int launch_narrow(const Narrow &a, hipStream_t s);

}  // namespace pfmoe
