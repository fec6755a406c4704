// 8-bit floating point (e4m3: four bits of exponent, three of mantissa, no infinities) with a scale for every block of 128:
//
//   activations: x[t, k] = sx[t, k / 128] * qx[t, k]        weights: w[r, k] = sw[r / 128, k / 128] * qw[r, k]
//
// and their product is y[t, r] = sum over blocks b of sx[t, b] * sw[r / 128, b] * (sum of qx[t, k] * qw[r, k] for k in b): the inner
// sum is the matrix cores', and meets its scales in FP32.
// A row's block of values v has m = max(max |v|, 2^-100), the scale m / 448 and the codes e4m3(v * (448 / m)), to nearest even; quotients
// and product are FP32.  |v| * (448 / m) <= 448 * (1 + 2^-22): nothing passes 464, from where on a value would no longer round
// to 448, the largest code.  A NaN has the code NaN; an infinity makes the scale infinite and its own code NaN (inf * 0).
#pragma once

#include "dev_common.h"

namespace bf16n {
namespace dev {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int FP8_BLOCK = 128;
constexpr float FP8_LARGEST = 448.f, FP8_SMALLEST = 0x1p-100f;

struct fp8_scales { float scale, inverse; };
__device__ __forceinline__ fp8_scales fp8_scales_of(float most) {
    const float m = fmaxf(most, FP8_SMALLEST);
    return {m / FP8_LARGEST, FP8_LARGEST / m};
}

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
// the codes of eight values
__device__ __forceinline__ u32x2_t fp8_pack8(const float (&v)[8], float r) {
    return u32x2_t{fp8_pack4(v[0] * r, v[1] * r, v[2] * r, v[3] * r), fp8_pack4(v[4] * r, v[5] * r, v[6] * r, v[7] * r)};
}

// the largest of the 16 lanes of a row, in all of them (fmaxf passes NaN over)
__device__ __forceinline__ float row_max_dpp(float v) {
    v = fmaxf(v, __uint_as_float(dpp_take<0xB1, 0xf>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dpp_take<0x4E, 0xf>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dpp_take<0x141, 0xf>(__float_as_uint(v))));
    return fmaxf(v, __uint_as_float(dpp_take<0x140, 0xf>(__float_as_uint(v))));
}

// the same of eight lanes
__device__ __forceinline__ float eight_max_dpp(float v) {
    v = fmaxf(v, __uint_as_float(dpp_take<0xB1, 0xf>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dpp_take<0x4E, 0xf>(__float_as_uint(v))));
    return fmaxf(v, __uint_as_float(dpp_take<0x141, 0xf>(__float_as_uint(v))));
}

__device__ __forceinline__ float most_of8(const float (&v)[8]) {
    return fmaxf(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))), fmaxf(fmaxf(fabsf(v[4]), fabsf(v[5])), fmaxf(fabsf(v[6]), fabsf(v[7]))));
}

// two BF16 numbers, to nearest even, by the instruction (the tests and masks of f32_to_bf16_rne were a third of the vector instructions of
// 8192 x 2048 by 8192 tokens)
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const bf16x2_t v = {(__bf16) a, (__bf16) b};
    return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ void bf16x8_to_f32(u32x4_t u, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}

// A sum over 128 columns: lane l has 32 columns of row l % 16 of either operand (the same ones of both); result: lane = row of b,
// register = rows 4 (l / 16) .. of a.  Two ways:
//
// fp8_sum8, one instruction on the codes.  It lines up the products of eight columns at the largest of them and drops what
// falls below 2^-13 of that (seen by adding 2^16 and smaller numbers; towards zero), before it adds them in FP32: normal operands come out
// 1.5e-5 of the result's norm off, a hundredth of what the result loses when it becomes BF16 (1.7e-3), less against codes.  For results that
// are rounded so.
//
// fp8_sum16, on the codes as BF16 numbers, which are exact, as their products are in FP32: 9e-9 off.  Half the rate of the matrix cores and a
// conversion (v_cvt_scalef32_pk_bf16_fp8) for two codes.  For FP32 results, and where memory or latency bounds a product anyway.
__device__ __forceinline__ f32x4_t fp8_sum8(u32x4_t a0, u32x4_t a1, u32x4_t b0, u32x4_t b1) {
    const i32x8_t a = {(int) a0[0], (int) a0[1], (int) a0[2], (int) a0[3], (int) a1[0], (int) a1[1], (int) a1[2], (int) a1[3]};
    const i32x8_t b = {(int) b0[0], (int) b0[1], (int) b0[2], (int) b0[3], (int) b1[0], (int) b1[1], (int) b1[2], (int) b1[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4_t{}, 0, 0, 0, 0, 0, 0);
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
struct fp8_wide { bf16x8_t k[4]; };
__device__ __forceinline__ bf16x8_t fp8_to_bf16(uint32_t lo, uint32_t hi) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ fp8_wide fp8_widen(u32x4_t a0, u32x4_t a1) {
    return {{fp8_to_bf16(a0[0], a0[1]), fp8_to_bf16(a0[2], a0[3]), fp8_to_bf16(a1[0], a1[1]), fp8_to_bf16(a1[2], a1[3])}};
}
__device__ __forceinline__ f32x4_t fp8_sum16(const fp8_wide & a, const fp8_wide & b) {
    f32x4_t v = {};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.k[i], b.k[i], v, 0, 0, 0);
    }
    return v;
}

} // namespace dev
} // namespace bf16n
