// e4m3 values (OCP FP8: 4 exponent bits, 3 mantissa bits, largest 448, one NaN, no
// infinities) in registers: four to a word, as gfx950's conversions take them.
#pragma once

#include "mfma_ops.h"

namespace vfl {

constexpr int E4M3_MIN_EXPONENT = -100;  // of a block's scale

// The smallest power of two that brings `amax` to 448 = 1.75 * 2^8 or less (2^-100 at
// least, which keeps scale * value clear of fp32's subnormals).
__device__ __forceinline__ float e4m3_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return __uint_as_float((uint32_t)(max(e, E4M3_MIN_EXPONENT) + 127) << 23);
}

// Four values of magnitude up to 448 (or NaN), rounded to nearest even.
__device__ __forceinline__ uint32_t e4m3_pack(const float *f) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
}

__device__ __forceinline__ void e4m3_unpack(uint32_t w, float *f) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1];
}

// The four values of a word times `ratio`, rounded again.
__device__ __forceinline__ uint32_t e4m3_rescale(uint32_t w, float ratio) {
  float f[4];
  e4m3_unpack(w, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] *= ratio;
  return e4m3_pack(f);
}

// Four values times `scale`, a power of two whose exponent the conversion adds, as bf16
// (exact: bf16 holds every e4m3 value and fp32's exponents).
__device__ __forceinline__ uint2 e4m3_widen(uint32_t w, float scale) {
  return make_uint2(
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)));
}

// Shared argument checks of the 8-bit cache's entry points (kv_cache_8bit.hip).
int check_8bit_cache(const char *who, int dtype, int num_heads, int head_dim, int block_size,
                     int64_t num_blocks);

}  // namespace vfl
