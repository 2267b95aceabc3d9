// The 8-bit KV cache's number format (the MX format of the OCP specification with e4m3 elements) on gfx950.
//
// A head row of D elements is D / 32 blocks of 32. A block holds 32 e4m3 codes (a byte each: 4 exponent, 3 mantissa bits,
// no infinity) and one scale byte e + 127 that stands for 2^e; an element's value is code * 2^e. Quantising x:
//   a = max |x| over the block's finite elements
//   e = the least integer >= -117 with a 2^-e <= 448 (the largest code)
//   code = x 2^-e rounded to the nearest code, ties to even; an infinity or a NaN gives the NaN code.
// The specification's floor(log2 a) - 8 would clip elements above 448 (the largest ones of a block whose a has a mantissa
// over 1.75) by up to an eighth; this rule clips none, so |x - value| <= max(2^-4 |x|, 2^-10 2^e).
// A value has 4 significant bits and, by the bound on e, is no smaller than 2^-126 unless it is 0: exact in bf16 and fp32.
//
// Caches are [num_blocks, Hkv, block_size, D] codes and [num_blocks, Hkv, block_size, D / 32] scales: the rows of one head
// in one page are contiguous, so an attention block streams runs of block_size * D bytes (in the bf16 caches' order,
// [num_blocks, block_size, Hkv, D], a head's 128-byte rows would lie Hkv rows apart).
#pragma once

#include "common.h"

namespace nvhip {

constexpr int kMxBlock = 32;  // elements that share a scale

typedef __bf16 bf16x8_mx __attribute__((ext_vector_type(8)));

// e + 127 of a block whose largest finite magnitude is a >= 0: the exponent of a, less 8, one more where the mantissa of a
// is over 1.75 (448 = 1.75 2^8). Below 2^-109 the exponent stays at that of 2^-109.
__device__ __forceinline__ uint32_t mx_scale_byte(float a) {
  const uint32_t bits = __float_as_uint(fmaxf(a, 0x1p-109f));
  return (bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
}
// The byte as the float 2^(byte - 127), of which 0 (no store writes it; the caches are zeros at first) reads as 0.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// |x| if x is finite, else 0.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = __builtin_fabsf(x);
  return a < INFINITY ? a : 0.0f;  // false for NaN too
}

// The maximum over the aligned group of 4 lanes, in all of them.
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));
}

// 8 fp32 values to 8 codes (two words). The conversion divides by the power of two `scale` and rounds once (to nearest
// even); infinities become NaN first, which it keeps.
__device__ __forceinline__ u32x2 mx_encode8(const float* x, float scale) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __builtin_fabsf(x[i]) < INFINITY ? x[i] : NAN;
  s16x2 lo = {}, hi = {};
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, y[0], y[1], scale, false);
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, y[2], y[3], scale, true);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, y[4], y[5], scale, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, y[6], y[7], scale, true);
  return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

// 8 codes (two words) to the 8 bf16 values they stand for (exact).
__device__ __forceinline__ u32x4 mx_decode8(uint32_t lo, uint32_t hi, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
}

}  // namespace nvhip
