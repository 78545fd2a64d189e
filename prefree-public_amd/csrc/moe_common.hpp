// moe_common.hpp — types and building blocks of the expert-layer kernels (routing, grouped products, 4-bit blocks).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.hpp"

namespace pfmoe {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr int kXcds = 8;

template <typename T> struct vec { };
template <> struct vec<f16> { typedef f16x8 x8; };
template <> struct vec<bf16> { typedef bf16x8 x8; };

// Rows of any alignment are loaded by the whole words that hold them, the elements then shifted into place (rows of 2222
// bytes out of the L2: 7.4 TB/s, 3.7 with the hardware's unaligned loads).  A word may hold an element that lies outside
// of what is asked for, but never only such, so it lies in the operand's memory.
//
// The words are said to be global memory: of pointers made of numbers the compiler does not know it, and its flat loads
// have to be waited for wherever an LDS read is (gradient of 32764 slots x 2049 from 1023, 32 experts: 681 us, 535 so).
__device__ __forceinline__ uintptr_t word_of(uintptr_t p) { return p & ~(uintptr_t)3; }
__device__ __forceinline__ unsigned load_word(uintptr_t p) { return *(const __attribute__((address_space(1))) unsigned *)p; }
// the last word of an operand of `bytes` > 0
__device__ __forceinline__ uintptr_t end_of(const char *base, unsigned long long bytes) { return word_of((uintptr_t)base + bytes - 2); }
// the first `valid` of a word's two elements, zeros behind them
__device__ __forceinline__ unsigned kept_word(unsigned v, int valid) { return valid >= 2 ? v : valid == 1 ? v & 0xffff : 0; }

// Eight elements of a row.  shifted() puts them into place and kept() clears what lies behind the row's end; only these
// wait, and loading has no branch in which anything but loads happens, so that several of them can be under way.
struct Words {
    i32x4 v;
    int last;

    static __device__ __forceinline__ unsigned shift_of(uintptr_t p) { return (unsigned)p & 2; }

    // the words from p, and the one at `more`: p + 16, or anything where the shift is 0
    __device__ __forceinline__ void load(uintptr_t p, uintptr_t more)
    {
        typedef int words __attribute__((ext_vector_type(4), aligned(4)));
        v = *(const __attribute__((address_space(1))) words *)p;
        last = (int)load_word(more);
    }
    // those of them before `end`, the operand's last word
    __device__ __forceinline__ void load_until(uintptr_t p, uintptr_t end)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (int)load_word(p + 4 * i < end ? p + 4 * i : end);
        last = (int)load_word(p + 16 < end ? p + 16 : end);
    }
    __device__ __forceinline__ i32x4 shifted(unsigned shift) const
    {
        return i32x4{(int)__builtin_amdgcn_alignbyte(v[1], v[0], shift), (int)__builtin_amdgcn_alignbyte(v[2], v[1], shift),
                     (int)__builtin_amdgcn_alignbyte(v[3], v[2], shift), (int)__builtin_amdgcn_alignbyte(last, v[3], shift)};
    }
    // the first `valid` of eight elements, zeros behind them
    static __device__ __forceinline__ i32x4 kept(i32x4 r, int valid)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (int)kept_word((unsigned)r[i], valid - 2 * i);
        return r;
    }
};

// 16 bytes that are all there, from an address that is a multiple of two.
__device__ __forceinline__ i32x4 load16_any(const void *p)
{
    const uintptr_t at = word_of((uintptr_t)p);
    const unsigned shift = Words::shift_of((uintptr_t)p);
    Words w;
    w.load(at, shift ? at + 16 : at);
    return w.shifted(shift);
}

// 1 / sigmoid(g), times kUnder.  As 1 + exp(-g) it would be infinite for gates under -88.7, and its reciprocal no normal number
// under -87.3, where silu(g) of bf16 still is one; scaled, both have room down to -98, where silu(g) is under 2^-134, half of
// the smallest bf16.  The scale is in the exponent (g / ln 2 rounded at up to 32: the exponential is off by 2^-20 of itself
// at the most, near g = 0) and of 16-bit gates times kUnder nothing is lost.
constexpr float kUnder = 0x1p-16f;
__device__ __forceinline__ float inverse_sigmoid(float g) { return kUnder + __builtin_amdgcn_exp2f(__builtin_fmaf(g, -0x1.715476p+0f, -16.0f)); }

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
