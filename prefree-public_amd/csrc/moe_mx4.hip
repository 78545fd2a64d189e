// moe_mx4.hip — 4-bit blocks on gfx950 (include/prefree_moe.h): blocks of 32 elements e2m1 with one scale byte e8m0.
#include <type_traits>

#include "moe_common.hpp"
#include "moe_launch.hpp"
#include "prefree_moe_kernels.h"

namespace {

using namespace pfmoe;

// Eight elements as fp32 from `at` of a row.
template <typename T, bool VECTOR>
__device__ __forceinline__ void load8(const T *p, float v[8])
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const i32x4 b = VECTOR ? *(const i32x4 *)(p + 4 * h) : load16_any(p + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * h + i] = __int_as_float(b[i]);
        }
    } else {
        typedef typename vec<T>::x8 x8;
        const x8 b = __builtin_bit_cast(x8, VECTOR ? *(const i32x4 *)p : load16_any(p));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)b[i];
    }
}

constexpr int kUnits = 4;   // pieces a thread takes, a workgroup's width apart: their loads go out together

// A lane takes eight elements at a time, four lanes a block of 32.  The block's scale exponent is its largest magnitude's
// exponent less 2, so that magnitude / scale lies in [4, 8); dividing by a power of two is exact, and the conversion
// instruction rounds to nearest even and saturates at 6, with scale 1.  65536 x 2048 of bf16, 268 MB read and 71 written, in
// 61 us, 5.6 TB/s (75 to 93 behind a fp32 result of 537 MB that is still being written back).  (Scales gathered in LDS and written as words: no difference; eight
// pieces a thread: 15% slower.)
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_quantize(const T *x, long long ld, long long units, int per_row, unsigned *codes,
                                                  unsigned char *scales)
{
    const long long first = (long long)blockIdx.x * 256 * kUnits + threadIdx.x;
    float v[kUnits][8];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const long long unit = first + j * 256;
        if (unit >= units) break;   // units come in fours
        const long long r = unit / per_row;
        load8<T, VECTOR>(x + ld * r + (unit - r * per_row) * 8, v[j]);
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const long long unit = first + j * 256;
        if (unit >= units) break;
        unsigned most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned b = __float_as_uint(v[j][i]) & 0x7fffffffu;
            most = b > most ? b : most;
        }
        unsigned o = pfdev::dpp<pfdev::kDppXor1>(most);
        most = o > most ? o : most;
        o = pfdev::dpp<pfdev::kDppXor2>(most);
        most = o > most ? o : most;
        const int e = (int)(most >> 23);                      // 255: an infinity or a NaN
        const int scale = e == 255 ? 255 : e < 2 ? 0 : e - 2;  // exponent + 127; 2^-127 at the least
        unsigned code = 0;
        if (e != 255) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = ldexpf(v[j][i], 127 - scale);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[j][0], v[j][1], 1.0f, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[j][2], v[j][3], 1.0f, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[j][4], v[j][5], 1.0f, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[j][6], v[j][7], 1.0f, 3);
        }
        codes[unit] = code;
        if ((threadIdx.x & 3) == 0) scales[unit >> 2] = (unsigned char)scale;
    }
}

// A lane writes 16 bytes at a time, next to its neighbours': four elements in fp32, eight in 16 bits.  65536 x 2048 to
// fp32, 608 MB, in 97 us with the codes in cache, 108 without, 5.6 TB/s; a large fill writes 6.9.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_dequantize(const unsigned char *codes, const unsigned char *scales, long long units,
                                                    int per_row, T *y, long long ld)
{
    constexpr int EACH = 16 / sizeof(T);
    typedef typename std::conditional<EACH == 8, unsigned, unsigned short>::type Codes;
    const long long first = (long long)blockIdx.x * 256 * kUnits + threadIdx.x;
    unsigned code[kUnits];
    int scale[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const long long unit = first + j * 256;
        if (unit >= units) break;
        code[j] = ((const Codes *)codes)[unit];
        scale[j] = scales[unit / (32 / EACH)];
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const long long unit = first + j * 256;
        if (unit >= units) break;
        T v[EACH];
        const auto put = [&](auto at) {
            constexpr int i = decltype(at)::value;
            const auto two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[j], 1.0f, i);
#pragma unroll
            for (int c = 0; c < 2; ++c)
                v[2 * i + c] = (T)(scale[j] == 255 ? __builtin_nanf("") : ldexpf(two[c], scale[j] - 127));
        };
        put(std::integral_constant<int, 0>());
        put(std::integral_constant<int, 1>());
        if constexpr (EACH == 8) {
            put(std::integral_constant<int, 2>());
            put(std::integral_constant<int, 3>());
        }
        const long long r = unit / per_row;
        T *out = y + ld * r + (unit - r * per_row) * EACH;
        if constexpr (VECTOR) {
            i32x4 b;
            __builtin_memcpy(&b, v, 16);
            *(i32x4 *)out = b;
        } else {
            __builtin_memcpy(out, v, 16);
        }
    }
}

// rows that one launch takes
long long most_rows(int per_row) { return most_workgroups(256) * 256 * kUnits / per_row; }
unsigned workgroups(long long units) { return (unsigned)((units + 256 * kUnits - 1) / (256 * kUnits)); }

template <typename T>
int quantize(const void *x, long long ld, int rows, int k, void *codes, void *scales, hipStream_t s)
{
    const bool vector = (uintptr_t)x % 16 == 0 && ld * sizeof(T) % 16 == 0;
    const auto kernel = vector ? k_quantize<T, true> : k_quantize<T, false>;
    in_launches(rows, most_rows(k / 8), [&](long long first, long long count) {
        const long long units = count * (k / 8);
        kernel<<<dim3(workgroups(units)), dim3(256), 0, s>>>((const T *)x + ld * first, ld, units, k / 8,
                                                             (unsigned *)codes + first * (k / 8), (unsigned char *)scales + first * (k / 32));
    });
    return pfk_internal_launched("k_quantize");
}

template <typename T>
int dequantize(const void *codes, const void *scales, int rows, int k, void *y, long long ld, hipStream_t s)
{
    const int per_row = k / (16 / (int)sizeof(T));
    const bool vector = (uintptr_t)y % 16 == 0 && ld * sizeof(T) % 16 == 0;
    const auto kernel = vector ? k_dequantize<T, true> : k_dequantize<T, false>;
    in_launches(rows, most_rows(per_row), [&](long long first, long long count) {
        const long long units = count * per_row;
        kernel<<<dim3(workgroups(units)), dim3(256), 0, s>>>((const unsigned char *)codes + first * (k / 2),
                                                             (const unsigned char *)scales + first * (k / 32), units, per_row,
                                                             (T *)y + ld * first, ld);
    });
    return pfk_internal_launched("k_dequantize");
}

}  // namespace

extern "C" {

int pfk_mx4_quantize(const void *x, long long ld_x, int dtype, int rows, int k, void *codes, void *scales, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F32 ? quantize<float>(x, ld_x, rows, k, codes, scales, s)
         : dtype == PF_F16 ? quantize<f16>(x, ld_x, rows, k, codes, scales, s) : quantize<bf16>(x, ld_x, rows, k, codes, scales, s);
}

int pfk_mx4_dequantize(const void *codes, const void *scales, int rows, int k, int dtype, void *y, long long ld_y, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F32 ? dequantize<float>(codes, scales, rows, k, y, ld_y, s)
         : dtype == PF_F16 ? dequantize<f16>(codes, scales, rows, k, y, ld_y, s) : dequantize<bf16>(codes, scales, rows, k, y, ld_y, s);
}

}  // extern "C"
