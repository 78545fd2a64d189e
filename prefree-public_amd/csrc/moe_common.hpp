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

// Eight 16-bit elements on their way from rows of any alignment: as the whole words that hold them, which take half the
// time of the hardware's own unaligned loads (rows of 2222 bytes out of the L2: 7.4 against 3.7 TB/s).  A word may hold
// an element that lies outside of what is asked for, but never only such.  settle() shifts them into place and clears
// what lies behind the row's end; it alone waits, and loading has no branch in which anything but loads happens, so that
// several of them can be under way.
struct Words {
    i32x4 v;
    int last, valid;
    bool odd;

    // elements [at, at + 8) of a row of `have`; `whole`, the same for all lanes: the row has them; end: the operand's last word
    __device__ __forceinline__ void load(const char *row, int at, int have, bool whole, const char *end)
    {
        typedef int words __attribute__((ext_vector_type(4), aligned(4)));
        const char *p = row + 2LL * at;
        odd = (uintptr_t)p & 2;
        valid = have - at;
        p = (const char *)((uintptr_t)p & ~(uintptr_t)3);
        if (whole) {
            v = *(const words *)p;
            last = *(const int *)(odd ? p + 16 : p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *(const int *)(p + 4 * i < end ? p + 4 * i : end);
            last = *(const int *)(p + 16 < end ? p + 16 : end);
        }
    }
    __device__ __forceinline__ i32x4 settle() const
    {
        i32x4 r = v;
        if (odd) {
            r[0] = __builtin_amdgcn_alignbyte(v[1], v[0], 2);
            r[1] = __builtin_amdgcn_alignbyte(v[2], v[1], 2);
            r[2] = __builtin_amdgcn_alignbyte(v[3], v[2], 2);
            r[3] = __builtin_amdgcn_alignbyte(last, v[3], 2);
        }
        if (valid < 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = 2 * i + 1 < valid ? r[i] : 2 * i < valid ? r[i] & 0xffff : 0;
        }
        return r;
    }
    // the last word of an operand of `bytes` > 0
    static __device__ __forceinline__ const char *end_of(const char *base, unsigned long long bytes)
    {
        return (const char *)(((uintptr_t)base + bytes - 2) & ~(uintptr_t)3);
    }
};

// 16 bytes that are all there, from an address that is a multiple of two.
__device__ __forceinline__ i32x4 load16_any(const void *p)
{
    Words w;
    w.load((const char *)p, 0, 8, true, nullptr);
    return w.settle();
}

// Inclusive sum over the lanes of a wave: inside the rows of 16 lanes by shifts, then the rows' last lanes are handed on
// (row_bcast 15 to the odd rows, row_bcast 31 to the upper half).  Whole wave active.
__device__ __forceinline__ int scan_wave(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
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
