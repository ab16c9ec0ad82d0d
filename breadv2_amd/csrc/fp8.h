// fp8.h — what the 8-bit floating point operators share: e4m3 codes with an
// fp32 scale for each block of 128 columns (activations) or 128 x 128
// (weights).
//
// e4m3 is the OCP type: sign, 4 bits of exponent with bias 7, 3 of mantissa,
// no infinities, largest value 448, NaN 0x7F and 0xFF.
#pragma once

#include "bread_device.h"
#include "bread_internal.h"

constexpr int F8_BLOCK = 128;
constexpr float F8_MAX = 448.f;
constexpr float F8_MIN_SCALE = 0x1p-126f;  // the smallest scale: its reciprocal is finite

typedef float f8_f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f8_half8 __attribute__((ext_vector_type(8)));

__host__ __device__ inline int f8_blocks(int n)
{
    return (n + F8_BLOCK - 1) / F8_BLOCK;
}

// The types of results and of the residual stream
__host__ __device__ inline bool f8_wide_type(int t)
{
    return t == BREAD_QTYPE_F32 || t == BREAD_QTYPE_F16 || t == BREAD_QTYPE_BF16;
}

__host__ __device__ inline int f8_type_bytes(int t)
{
    return t == BREAD_QTYPE_F32 ? 4 : t == BREAD_QTYPE_E4M3 ? 1 : 2;
}

__device__ __forceinline__ float bf2f(uint32_t b)
{
    return __builtin_bit_cast(float, b << 16);
}

__device__ __forceinline__ uint16_t f2bf(float f)
{
    return __builtin_bit_cast(uint16_t, (__bf16)f);
}

// Magnitudes as integers: in their order, NaN above infinity above every
// number, so that a maximum of them does not lose a NaN (as fmaxf does).
__device__ __forceinline__ uint32_t f8_mag(float v)
{
    return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
}

// The scale of a block with the largest magnitude m; NaN if the block holds
// an infinity or a NaN.
__device__ __forceinline__ float f8_scale(uint32_t m)
{
    if (m >= 0x7F800000u) return __builtin_nanf("");
    return fmaxf(__builtin_bit_cast(float, m) / F8_MAX, F8_MIN_SCALE);
}

// Codes of v[i] / s, r = 1 / s: to nearest, ties to even.  |v| r is at most
// 448 (1 + 2^-22), which rounds to 448; a NaN scale makes every code NaN.
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, float r)
{
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a * r, b * r, 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(c * r, d * r, p, true);
    return (uint32_t)p;
}

// Arguments of a product, as checked by the entry points
struct F8Args {
    const uint8_t *w, *up, *x;
    const float *ws, *us, *xs;
    void *y;
    float *ys;
    const float *bias;
    const void *res;
    int64_t x_stride, xs_stride, y_stride, ys_stride;
    int rows, cols, T, act, y_type;
    // groups: rows [offsets[g], offsets[g + 1]) meet weights g; G = 0: one matrix for all T rows
    int G;
    const int32_t *offsets, *x_rows, *y_rows;
    int n_x, n_y;
};

// Launches without checks (fp8_matmul.hip, fp8_grouped.hip)
int bread_launch_fp8_matmul(const F8Args &a, hipStream_t st);
int bread_launch_fp8_grouped(const F8Args &a, hipStream_t st);
