// 4-bit weights with group scales: the matrix as the kernels see it and a lane's codes as operands of the matrix cores.
//
//   w[r, k] = s[r, k / group] * (u[r, k] - z[r, k / group]),   u a code 0..15, two to a byte, the even column in the low half
//
// A product is taken on the codes themselves, which BF16 holds exactly, and scaled per group in FP32:
//   y[r] = sum_g s[r, g] * (sum_{k in g} x[k] u[r, k] - z[r, g] * sum_{k in g} x[k])
// so that no weight is rounded.  A byte 0..15 is, read as e4m3, 2^-9 times its value (0..7 are denormals, 8..15 the first
// binade), so one instruction, v_cvt_scalef32_pk_bf16_fp8 with the scale 2^9, turns two codes into two BF16 values; eight codes
// take seven instructions at full rate.  They come out as columns 0, 2, 4, 6, 1, 3, 5, 7, and the activations are laid out
// in that order.
#pragma once

#include "dev_common.h"

namespace bf16n {
namespace dev {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// loads of two or four scales and of two, four or eight zero points, wherever a row begins
typedef uint64_t __attribute__((aligned(2), may_alias)) u64_at_2;
typedef uint32_t __attribute__((aligned(2), may_alias)) u32_at_2;
typedef uint64_t __attribute__((aligned(1), may_alias)) u64_at_1;
typedef uint32_t __attribute__((aligned(1), may_alias)) u32_at_1;
typedef uint16_t __attribute__((aligned(1), may_alias)) u16_at_1;

struct i4_matrix {
    const uint8_t * codes;   // [rows, K / 2], 16-byte aligned
    const uint16_t * scales; // [rows, n_groups] BF16 or FP16
    const uint8_t * zeros;   // [rows, n_groups], or null: 8
    bool f16;
};

// eight codes of a lane as one operand (columns 0, 2, 4, 6, 1, 3, 5, 7)
__device__ __forceinline__ bf16x8_t i4_operand(uint32_t w) {
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// the same in the columns' own order, two instructions more
__device__ __forceinline__ bf16x8_t i4_operand_in_order(uint32_t w) {
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
    const uint32_t l = __builtin_amdgcn_perm(hi, lo, 0x05010400u), h = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(l, 512.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(l, 512.f, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(h, 512.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(h, 512.f, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// eight BF16 activations in the operands' column order
__device__ __forceinline__ u32x4_t i4_order(u32x4_t v) {
    return u32x4_t{__builtin_amdgcn_perm(v[1], v[0], 0x05040100u), __builtin_amdgcn_perm(v[3], v[2], 0x05040100u),
                   __builtin_amdgcn_perm(v[1], v[0], 0x07060302u), __builtin_amdgcn_perm(v[3], v[2], 0x07060302u)};
}

// A lane of quarter q holds the four words of 32 columns q * 32 + 8 j; afterwards word j is that of the columns 32 j + 8 q:
// a 4 x 4 transpose of words and quarters, for groups smaller than the 128 columns of one step.
__device__ __forceinline__ u32x4_t i4_transpose(u32x4_t d) {
    const auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false), b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
    const auto e = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), f = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4_t{e[0], e[1], f[0], f[1]};
}

// an FP32 value as three BF16 parts that add up to it exactly (each takes the leading eight bits of what is left; a value
// that is not finite stays whole in the first, with zeros behind it)
__device__ __forceinline__ void f32_parts(float v, uint32_t & a, uint32_t & b, uint32_t & c) {
    const uint32_t u = __float_as_uint(v), h = u & 0xFFFF0000u;
    const bool finite = (u & 0x7F800000u) != 0x7F800000u;
    const float r = finite ? v - __uint_as_float(h) : 0.f;
    const uint32_t m = __float_as_uint(r) & 0xFFFF0000u;
    const float l = r - __uint_as_float(m);
    a = finite || (u & 0xFFFFu) == 0 ? h >> 16 : (h >> 16) | 0x40u; // a NaN whose payload is in the lower half stays one
    b = m >> 16;
    c = __float_as_uint(l) >> 16;
}

// f16: all ones or zero (a choice between two registers, not a branch)
__device__ __forceinline__ float i4_scale(uint32_t bits, uint32_t f16) {
    const float h = (float) __builtin_bit_cast(_Float16, (uint16_t) bits);
    return __uint_as_float((__float_as_uint(h) & f16) | ((bits << 16) & ~f16));
}

} // namespace dev
} // namespace bf16n
