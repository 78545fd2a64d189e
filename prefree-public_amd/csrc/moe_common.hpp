// moe_common.hpp — types and building blocks of the expert-layer kernels (routing, grouped products, 4-bit blocks).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.hpp"

namespace pfmoe {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct fp4 {};  // tag: e2m1 codes, two a byte, one e8m0 scale byte per 32

constexpr int kWave = 64;
constexpr int kXcds = 8;

template <typename T> struct vec { };
template <> struct vec<f16> { typedef f16x4 x4; typedef f16x8 x8; };
template <> struct vec<bf16> { typedef bf16x4 x4; typedef bf16x8 x8; };

// 16 bytes from an address that is only as aligned as its elements (the hardware takes any; what matters is that
// the compiler is not told otherwise).
__device__ __forceinline__ i32x4 load16_any(const void *p)
{
    i32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// sum over aligned groups of 16 lanes; every lane has it
__device__ __forceinline__ float sum16(float v) { return pfdev::group_sum<16>(v); }

// inclusive sum over the lanes of a wave
__device__ __forceinline__ int scan_wave(int v)
{
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// Rows [begin, end) of expert e, whatever the offsets hold: inside [0, slots], never negative in number.
__device__ __forceinline__ void expert_rows(const int *__restrict__ offsets, int e, int slots, int &begin, int &end)
{
    begin = offsets ? offsets[e] : 0;
    end = offsets ? offsets[e + 1] : slots;
    begin = begin < 0 ? 0 : begin > slots ? slots : begin;
    end = end < begin ? begin : end > slots ? slots : end;
}

}  // namespace pfmoe
