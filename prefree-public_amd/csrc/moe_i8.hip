// moe_i8.hip — 8-bit integers with a scale a row on gfx950 (include/prefree_moe.h).
#include <type_traits>

#include "moe_common.hpp"
#include "moe_launch.hpp"
#include "prefree_moe_kernels.h"

namespace {

using namespace pfmoe;

// The nearest integer to 127 x / most, ties to even.  per = 127 / most to 53 bits and the sum that moves the point give
// the quotient as a multiple of 2^-33, off by less than 2^-44 before.  A quotient q of numbers of 24 bits that is no half
// itself lies at least q / (127 2^25) from one, more than 2^-33 from 1/2 on: so halves come out as halves, nothing else
// does, and the second sum rounds to even, into the low bits.  (Quotients in 32 bits, for values of 16 bits, changed
// nothing in the time: the kernel waits for memory.)
__device__ __forceinline__ unsigned integer_of(float x, double per)
{
    constexpr double kPoint = 0x1.8p+19, kWhole = 0x1.8p+52;
    const double v = __builtin_fma((double)x, per, kPoint) - kPoint;
    return (unsigned)__double_as_longlong(v + kWhole);
}

__device__ __forceinline__ u32x2 eight_of(const float v[8], double per)
{
    u32x2 r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned a = integer_of(v[4 * h], per), b = integer_of(v[4 * h + 1], per), c = integer_of(v[4 * h + 2], per),
                       d = integer_of(v[4 * h + 3], per);
        const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400), hi = __builtin_amdgcn_perm(d, c, 0x04000c0c);
        r[h] = lo | hi;
    }
    return r;
}

constexpr float kLeast = 0x1p-100f;   // of a row's largest magnitude: a scale of its own for smaller ones is not worth a normal number

// G lanes take a row, whole workgroups or waves; each holds PIECES pieces of eight elements, G apart, over both passes: the
// largest magnitude, then the integers.  Rows that are longer are read again for what does not fit.  32768 x 2048 bf16: 52 to
// 56 us, as is the way back to fp32: 3.6 and 5.9 TB/s, the copy's bytes between them at 4.8.
template <typename T, int G, int PIECES, bool VECTOR>
__global__ __launch_bounds__(256) void k_i8_quantize(const T *x, long long ld, int rows, int k, unsigned char *codes, long long ld_codes,
                                                     float *scales)
{
    __shared__ unsigned most_of[4];
    const int lane = threadIdx.x % G, r = blockIdx.x * (256 / G) + threadIdx.x / G;
    if (r >= rows) return;
    const T *row = x + ld * r;
    const int units = (int)(ld_codes / 8);   // pieces of the codes, behind k zeros
    float v[PIECES][8];
    unsigned most = 0;
    const auto take = [&](const float w[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned b = __float_as_uint(w[i]) & 0x7fffffffu;
            most = b > most ? b : most;
        }
    };
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const int at = (lane + j * G) * 8;
        if (lane + j * G < units) load8_any<T, VECTOR>(row, at, k, v[j]);
        else
            for (int i = 0; i < 8; ++i) v[j][i] = 0;
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) take(v[j]);
    for (int u = lane + PIECES * G; u < units; u += G) {
        float w[8];
        load8_any<T, VECTOR>(row, u * 8, k, w);
        take(w);
    }
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned other = (unsigned)__shfl_xor((int)most, o);
        most = other > most ? other : most;
    }
    if constexpr (G == 256) {
        if (threadIdx.x % kWave == 0) most_of[threadIdx.x / kWave] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) most = most_of[w] > most ? most_of[w] : most;
    }
    const bool finite = most < 0x7f800000u;
    const float largest = fmaxf(__uint_as_float(most), kLeast);
    const double per = finite ? 127.0 / (double)largest : 0.0;
    if (lane == 0) scales[r] = finite ? largest / 127.0f : __builtin_nanf("");
    u32x2 *out = (u32x2 *)(codes + ld_codes * r);
    const auto put = [&](int u, const float w[8]) { out[u] = finite ? eight_of(w, per) : u32x2{0, 0}; };
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
        if (lane + j * G < units) put(lane + j * G, v[j]);
    for (int u = lane + PIECES * G; u < units; u += G) {
        float w[8];
        load8_any<T, VECTOR>(row, u * 8, k, w);
        put(u, w);
    }
}

// A lane writes 16 bytes at a time: four elements in fp32, eight in 16 bits.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_i8_dequantize(const unsigned char *codes, long long ld_codes, const float *scales, long long units,
                                                       int per_row, int k, T *y, long long ld)
{
    constexpr int EACH = 16 / sizeof(T), kUnits = 4;
    typedef typename std::conditional<EACH == 8, unsigned long long, unsigned>::type Codes;
    const long long first = (long long)blockIdx.x * 256 * kUnits + threadIdx.x;
    Codes code[kUnits];
    float scale[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const long long unit = first + j * 256;
        if (unit >= units) break;
        const long long r = unit / per_row;
        code[j] = *(const Codes *)(codes + ld_codes * r + (unit - r * per_row) * EACH);
        scale[j] = scales[r];
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const long long unit = first + j * 256;
        if (unit >= units) break;
        const long long r = unit / per_row;
        const int at = (int)(unit - r * per_row) * EACH;
        T v[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) v[i] = (T)((float)(signed char)(code[j] >> 8 * i) * scale[j]);
        T *out = y + ld * r + at;
        typedef T vec_t __attribute__((ext_vector_type(EACH)));
        typedef vec_t any_t __attribute__((aligned(sizeof(T))));   // one store too, of any address
        if (at + EACH <= k) {
            vec_t b;
            __builtin_memcpy(&b, v, 16);
            if (VECTOR) *(vec_t *)out = b;
            else *(any_t *)out = b;
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                if (at + i < k) out[i] = v[i];
        }
    }
}

template <typename T, int G, int PIECES>
int quantize(const void *x, long long ld, int rows, int k, void *codes, float *scales, hipStream_t s)
{
    const bool vector = (uintptr_t)x % 16 == 0 && ld * sizeof(T) % 16 == 0;
    const auto kernel = vector ? k_i8_quantize<T, G, PIECES, true> : k_i8_quantize<T, G, PIECES, false>;
    const long long ld_codes = PF_I8_ROW(k);
    in_launches(rows, most_workgroups(256) * (256 / G), [&](long long first, long long count) {
        kernel<<<dim3((unsigned)((count + 256 / G - 1) / (256 / G))), dim3(256), 0, s>>>(
            (const T *)x + ld * first, ld, (int)count, k, (unsigned char *)codes + ld_codes * first, ld_codes, scales + first);
    });
    return pfk_internal_launched("k_i8_quantize");
}

template <typename T>
int quantize(const void *x, long long ld, int rows, int k, void *codes, float *scales, hipStream_t s)
{
    if (k > 4096 || rows < 2048) return quantize<T, 256, 2>(x, ld, rows, k, codes, scales, s);
    if (k > 2048) return quantize<T, 64, 8>(x, ld, rows, k, codes, scales, s);
    return quantize<T, 64, 4>(x, ld, rows, k, codes, scales, s);
}

template <typename T>
int dequantize(const void *codes, const float *scales, int rows, int k, void *y, long long ld, hipStream_t s)
{
    constexpr int EACH = 16 / sizeof(T);
    const int per_row = (k + EACH - 1) / EACH;
    const bool vector = (uintptr_t)y % 16 == 0 && ld * sizeof(T) % 16 == 0;
    const auto kernel = vector ? k_i8_dequantize<T, true> : k_i8_dequantize<T, false>;
    const long long ld_codes = PF_I8_ROW(k);
    in_launches(rows, most_workgroups(256) * 1024 / per_row, [&](long long first, long long count) {
        const long long units = count * per_row;
        const dim3 grid((unsigned)((units + 1023) / 1024));
        kernel<<<grid, dim3(256), 0, s>>>((const unsigned char *)codes + ld_codes * first, ld_codes, scales + first, units, per_row, k,
                                          (T *)y + ld * first, ld);
    });
    return pfk_internal_launched("k_i8_dequantize");
}

}  // namespace

extern "C" {

int pfk_i8_quantize(const void *x, long long ld_x, int dtype, int rows, int k, void *codes, float *scales, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F32 ? quantize<float>(x, ld_x, rows, k, codes, scales, s)
         : dtype == PF_F16 ? quantize<f16>(x, ld_x, rows, k, codes, scales, s) : quantize<bf16>(x, ld_x, rows, k, codes, scales, s);
}

int pfk_i8_dequantize(const void *codes, const float *scales, int rows, int k, int dtype, void *y, long long ld_y, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    return dtype == PF_F32 ? dequantize<float>(codes, scales, rows, k, y, ld_y, s)
         : dtype == PF_F16 ? dequantize<f16>(codes, scales, rows, k, y, ld_y, s) : dequantize<bf16>(codes, scales, rows, k, y, ld_y, s);
}

}  // extern "C"
