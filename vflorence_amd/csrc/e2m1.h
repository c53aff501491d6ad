// A paged cache held in 4 bits: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6, the fourth bit the sign)
// and, per token, head and group of 32 dims, for K and for V, the byte e of a scale 2^(e - 127)
// (255: every value of the group is NaN).
//
// A block of the pool ([num_blocks][num_heads][block_size][34 * groups] bytes, groups =
// ceil(head_dim / 32); dims past the head are 0) holds, with tokens in parts of 16:
//   keys    [head][part][group][token][16]  byte j: dims 2j (low half) and 2j + 1 of the group
//   values  [head][part][group][16][token]  byte j: dims j (low half) and j + 16 of the group
//   scales  [head][part][token / 4][K, V][group][token % 4]
// A wave of the attention takes 64 tokens, a part to each row of 16 lanes: a lane reads its token's
// dims of K and 16 tokens of two dims of V in 16-byte pieces, 256 bytes a row side by side, and
// no byte is shared by two tokens, so a token is appended without reading what lies beside it.
#pragma once

#include "mfma_ops.h"

namespace vfl {

constexpr int E2M1_GROUP = 32;
constexpr int E2M1_NAN = 255;
// Scales: 2^-100 at least, which keeps scale * value clear of fp32's subnormals, and 2^125 at
// most, which times 6 is finite (magnitudes beyond, from 1.75 * 2^127 on, are held as that).
constexpr int E2M1_MIN_EXPONENT = -100, E2M1_MAX_EXPONENT = 125;

__host__ __device__ __forceinline__ constexpr int e2m1_groups(int D) {
  return (D + E2M1_GROUP - 1) / E2M1_GROUP;
}

// Byte offsets in a block of a head's part.
struct E2m1Layout {
  int G, parts;
  int64_t half;         // bytes of the block's keys
  int64_t block_bytes;

  __host__ __device__ __forceinline__ E2m1Layout(int H, int G, int parts)
      : G(G), parts(parts), half((int64_t)H * parts * G * 256),
        block_bytes((int64_t)H * parts * G * 544) {}
  __host__ __device__ __forceinline__ int64_t keys(int h, int part) const {
    return ((int64_t)h * parts + part) * G * 256;
  }
  __host__ __device__ __forceinline__ int64_t values(int h, int part) const {
    return half + keys(h, part);
  }
  __host__ __device__ __forceinline__ int64_t scales(int h, int part) const {
    return 2 * half + ((int64_t)h * parts + part) * G * 32;
  }
};

// The exponent byte of the smallest power of two that brings `amax` to 6 = 1.5 * 2^2 or less.
__device__ __forceinline__ uint32_t e2m1_scale_byte(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 2 + ((bits & 0x7fffffu) > 0x400000u);
  return (uint32_t)(min(max(e, E2M1_MIN_EXPONENT), E2M1_MAX_EXPONENT) + 127);
}

__device__ __forceinline__ float e2m1_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight elements (as words of memory) over `scale`, whose exponent the conversion takes off,
// rounded to nearest even, past 6 to 6: nibble i is element i.
template <int DT> __device__ __forceinline__ uint32_t e2m1_pack8(const uint32_t *w, float scale) {
  uint32_t r = 0;
  if constexpr (DT == VFL_FLOAT32) {
#define VFL_PACK(i) \
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[2 * i]), \
                                               __uint_as_float(w[2 * i + 1]), scale, i)
    VFL_PACK(0); VFL_PACK(1); VFL_PACK(2); VFL_PACK(3);
#undef VFL_PACK
  } else if constexpr (DT == VFL_BFLOAT16) {
#define VFL_PACK(i) \
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, w[i]), scale, i)
    VFL_PACK(0); VFL_PACK(1); VFL_PACK(2); VFL_PACK(3);
#undef VFL_PACK
  } else {
#define VFL_PACK(i) \
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, w[i]), scale, i)
    VFL_PACK(0); VFL_PACK(1); VFL_PACK(2); VFL_PACK(3);
#undef VFL_PACK
  }
  return r;
}

// The two codes of byte BYTE times `scale`, the low one first.
template <int BYTE> __device__ __forceinline__ uint32_t e2m1_bf16x2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, BYTE));
}
template <int BYTE> __device__ __forceinline__ float2_t e2m1_f32x2(uint32_t w, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, BYTE);
}

// The eight codes of a word times `scale` as elements, rounded to nearest even where fp16 does
// not hold them.
template <int DT>
__device__ __forceinline__ void e2m1_unpack8(uint32_t w, float scale, uint32_t *out) {
  if constexpr (DT == VFL_BFLOAT16) {
    out[0] = e2m1_bf16x2<0>(w, scale), out[1] = e2m1_bf16x2<1>(w, scale);
    out[2] = e2m1_bf16x2<2>(w, scale), out[3] = e2m1_bf16x2<3>(w, scale);
  } else {
    const float2_t f[4] = {e2m1_f32x2<0>(w, scale), e2m1_f32x2<1>(w, scale),
                           e2m1_f32x2<2>(w, scale), e2m1_f32x2<3>(w, scale)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == VFL_FLOAT32) {
        out[2 * i] = __float_as_uint(f[i][0]), out[2 * i + 1] = __float_as_uint(f[i][1]);
      } else {
        out[i] = Mfma<VFL_FLOAT16>::narrow2(f[i][0], f[i][1]);
      }
    }
  }
}

// Shared argument checks of the 4-bit cache's entry points (kv_cache_4bit.hip).
int check_4bit_cache(const char *who, int dtype, int num_heads, int head_dim, int block_size,
                     int64_t num_blocks);

}  // namespace vfl
