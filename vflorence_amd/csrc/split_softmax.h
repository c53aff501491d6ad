// What the decode attention kernels over quantised caches share: the rows of a group, softmax
// weights and queries as bf16 terms, and the join of a context that several workgroups split.
#pragma once

#include <float.h>
#include <math.h>

#include "mfma_ops.h"

namespace vfl {

// bf16 terms of a query and of a weight
template <int DT> struct Terms {
  static constexpr int Q = DT == VFL_FLOAT32 ? 3 : DT == VFL_FLOAT16 ? 2 : 1;
  static constexpr int P = DT == VFL_FLOAT32 ? 3 : 2;
};

using Bf16 = Mfma<VFL_BFLOAT16>;

// bf16 terms of four floats, largest first; f is left with the remainder.  Queries are cut, weights
// rounded: a cut term holds 8 bits and the next ones start behind it, so two hold all of fp16 and
// three all of fp32 either way, and the largest fp32 values, which would round to infinity,
// stay finite; of two or three terms that do not hold everything rounding leaves half as much.
template <bool ROUND> __device__ __forceinline__ uint2 take_bf16(float (&f)[4]) {
  uint2 w;
  if constexpr (ROUND) {
    w = make_uint2(Bf16::narrow2(f[0], f[1]), Bf16::narrow2(f[2], f[3]));
  } else {
    constexpr uint32_t HIGH_HALVES = 0x07060302u;
    w = make_uint2(
        __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), HIGH_HALVES),
        __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), HIGH_HALVES));
  }
  f[0] -= Bf16::widen_lo(w.x), f[1] -= Bf16::widen_hi(w.x);
  f[2] -= Bf16::widen_lo(w.y), f[3] -= Bf16::widen_hi(w.y);
  return w;
}

template <int DT>
__device__ __forceinline__ void store_result(typename Elem<DT>::T *p, float S, float o) {
  const float y = S > 0.f ? o / S : S == S ? 0.f : S;  // NaN scores stay NaN
  if constexpr (DT == VFL_FLOAT32) *p = y;
  else *p = (uint16_t)Mfma<DT>::narrow(y);
}

// What is added to a softmax when its context is split: [row][head][split].  The sums come first
// in the workspace: whole 64-byte pieces, 16-byte aligned for any number of parts.
struct SplitOut {
  float *acc;  // [D]
  float2 *ml;
};

// Bytes a (row, head) of one split takes in the workspace.
inline int64_t split_part_bytes(int head_dim) { return head_dim * 4 + 8; }

// Bytes of workspace that a launch takes at most.
constexpr int64_t MOST_WORKSPACE = 1LL << 27;

// A launch's rows and where their results go.
struct DecodeRows {
  void *out;
  const int32_t *group_start, *group_order;
  int64_t num_rows, num_groups;
  int H, D;
  float scale_log2;  // its magnitude: the query takes the sign
  int splits;
  SplitOut part;
};

constexpr int GROUP_ROWS = 8;  // rows of a group
constexpr float NO_SCORE = -3.402823466e38f;  // the least finite score

// |scale| in log2 units, finite and not 0, which would make NaN of an equal or a masked score (the
// least denormal in its place moves no weight by more than 2^-21).
inline float decode_scale_log2(float scale) {
  return fminf(fmaxf(fabsf(scale) * 1.4426950408889634f, __FLT_DENORM_MIN__), -NO_SCORE);
}

// Rows of the group at dispatch position `pos`, from row0 on (0: no such group).
__device__ __forceinline__ int group_rows(const DecodeRows &a, int64_t pos, int64_t &row0) {
  if (pos >= a.num_groups) return 0;
  int64_t g = pos;
  if (a.group_order) g = a.group_order[pos];
  if (g < 0 || g >= a.num_groups) return 0;
  row0 = g;
  int n = 1;
  if (a.group_start) {
    row0 = a.group_start[g];
    n = a.group_start[g + 1] - (int)row0;
  }
  if (row0 < 0 || row0 >= a.num_rows) return 0;
  return (int)min((int64_t)min(n, GROUP_ROWS), a.num_rows - row0);
}

// The splits of a (row, head) joined: a quarter of D threads, a team, take 4 dims each of
// every teams-th split, about a maximum of their own, so that maxima and sums come in one round
// trip; the teams meet in LDS.
constexpr int JOIN_NT = 256;
template <int DT>
__device__ __forceinline__ void join_splits(void *out, const SplitOut &part, int64_t at,
                                            int64_t out_at, int D, int splits, float scale_log2) {
  using T = typename Elem<DT>::T;
  __shared__ float4 s_o[JOIN_NT];
  __shared__ float2 s_ml[JOIN_NT];
  const int tid = threadIdx.x, quads = D / 4, teams = JOIN_NT / quads;
  const int team = tid / quads, quad = tid % quads;
  const float2 *ml = part.ml + at * splits;
  const float4 *acc = reinterpret_cast<const float4 *>(part.acc + at * splits * D) + quad;
  float M = NO_SCORE, S = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (team < teams) {
#pragma unroll 4
    for (int s = team; s < splits; s += teams) {
      const float2 x = ml[s];
      const float4 v = acc[(int64_t)s * quads];
      const float to = fmaxf(M, x.x);
      const float f = fast_exp2((M - to) * scale_log2), e = fast_exp2((x.x - to) * scale_log2);
      S = S * f + x.y * e;
      o.x = o.x * f + v.x * e, o.y = o.y * f + v.y * e;
      o.z = o.z * f + v.z * e, o.w = o.w * f + v.w * e;
      M = to;
    }
  }
  s_o[tid] = o;
  s_ml[tid] = make_float2(M, S);
  __syncthreads();
  for (int d = tid; d < D; d += JOIN_NT) {
    float top = NO_SCORE, sum = 0.f, y = 0.f;
    for (int t = 0; t < teams; ++t) top = fmaxf(top, s_ml[t * quads + d / 4].x);
    for (int t = 0; t < teams; ++t) {
      const float2 x = s_ml[t * quads + d / 4];
      const float e = fast_exp2((x.x - top) * scale_log2);
      sum = fmaf(x.y, e, sum);
      y = fmaf((&s_o[t * quads + d / 4].x)[d % 4], e, y);
    }
    store_result<DT>((T *)out + out_at + d, sum, y);
  }
}

// One workgroup a (group, head) and row of the group (blockIdx.y).
template <int DT> __global__ __launch_bounds__(JOIN_NT) void join_rows_kernel(DecodeRows a) {
  int64_t row0;
  if ((int)blockIdx.y >= group_rows(a, blockIdx.x / a.H, row0)) return;
  const int64_t at = (row0 + blockIdx.y) * a.H + blockIdx.x % a.H;
  join_splits<DT>(a.out, a.part, at, at * a.D, a.D, a.splits, a.scale_log2);
}

template <int DT> inline void launch_join_rows(const DecodeRows &a, hipStream_t stream) {
  const unsigned rows = a.group_start ? GROUP_ROWS : 1;
  join_rows_kernel<DT>
      <<<dim3((unsigned)(a.num_groups * a.H), rows), dim3(JOIN_NT), 0, stream>>>(a);
}

}  // namespace vfl
