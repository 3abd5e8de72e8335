// The rows of the 8-bit key/value cache: e4m3 values with one power-of-two
// scale (an e8m0 byte s: 2^(s - 127), 255: NaN) per row of head_dim values.
//
// A power of two loses no precision against a scale of 32 bits (e4m3 keeps
// three bits behind the leading one at any magnitude above 2^-6 of the scale),
// costs one byte per row instead of four, makes the stored value the same
// whatever divides or multiplies, and is what v_cvt_scalef32_pk_bf16_fp8
// applies as it converts: two values of a cached row are two bf16 ones, scaled
// and exact, in one instruction at the rate of an FMA (measured 4.5 cycles per
// wave and SIMD; v_cvt_pk_f32_fp8, which would leave the scale and the packing
// to be done, 8.7).
#pragma once

#include "vx_gfx950.hpp"

namespace vx {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// A scale byte as the fp32 power of two it stands for (255: NaN).
__device__ __forceinline__ float e8m0_scale(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7fc00000u : s << 23);
}

// Four bytes of a cached row as bf16 values times a scale from e8m0_scale.
__device__ __forceinline__ bf16x4 e4m3x4_bf16(uint32_t x, float scale) {
  const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false);
  const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3);
}

// Eight of them.
__device__ __forceinline__ bf16x8 e4m3x8_bf16(u32x2 x, float scale) {
  return concat(e4m3x4_bf16(x[0], scale), e4m3x4_bf16(x[1], scale));
}

}  // namespace vx
