// Rows of the cache in 4 bits: where their parts lie, and what a code and a scale stand for.
#pragma once

#include "tpa_common.h"

namespace tpa {

typedef __attribute__((ext_vector_type(2))) float f32x2;

__host__ __device__ __forceinline__ constexpr int fp4_blocks(int n) { return (n + 31) / 32; }
struct Fp4Row {  // bytes from the start of a row
  int a_codes, b_scales, a_scales;  // (the codes of b come first)
  __host__ __device__ __forceinline__ constexpr Fp4Row(int H, int D)
      : a_codes((D + 1) / 2), b_scales(a_codes + (H + 1) / 2), a_scales(b_scales + fp4_blocks(D)) {}
};
inline int64_t fp4_row_bytes(int64_t H, int64_t D) { return ((D + 1) / 2 + (H + 1) / 2 + (D + 31) / 32 + (H + 31) / 32 + 3) / 4 * 4; }

// 2^(scale - 127) as the conversions take it: 255 makes infinity of it, for which they give NaN
__device__ __forceinline__ float fp4_scale(uint32_t scale) { return __uint_as_float(scale << 23); }

// the eight numbers of a word of codes, exact in bf16
__device__ __forceinline__ bf16x8 fp4_bf16x8(uint32_t codes, float scale) {
  const bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return __builtin_bit_cast(bf16x8, u32x4{__builtin_bit_cast(uint32_t, p0), __builtin_bit_cast(uint32_t, p1), __builtin_bit_cast(uint32_t, p2),
                                          __builtin_bit_cast(uint32_t, p3)});
}
__device__ __forceinline__ void fp4_f32x8(uint32_t codes, float scale, float (&x)[8]) {
  const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  x[0] = p0[0]; x[1] = p0[1]; x[2] = p1[0]; x[3] = p1[1];
  x[4] = p2[0]; x[5] = p2[1]; x[6] = p3[0]; x[7] = p3[1];
}
// number i of a part whose codes and scales start at `codes` and `scales`
__device__ __forceinline__ float fp4_number(const uint8_t* codes, const uint8_t* scales, int i) {
  const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)codes[i >> 1], fp4_scale(scales[i >> 5]), 0);
  return i & 1 ? p[1] : p[0];
}

}  // namespace tpa
