// Paged decode attention over a cache held in e4m3 with a scale per (block, head) for K and
// one for V, gfx950:
//   out[r][h] = softmax_j(scale * ks_j <q[r][h], K8_j[h]>) (vs_j V8_j[h]),  j < seq_lens[r]
// with ks_j, vs_j the scales of token j's block, powers of two.  e4m3 times such a scale is
// exact in bf16 (one conversion per pair, which adds the exponent) on its way into the matrix
// cores.
//
// The rows of a group (a request's beams over one page list) sit in the 16 columns of the
// tiles.  A wave takes 32 tokens at a time, two 16-token parts:
//   S[tok][row]  = K[tok][:] . q[row][:]     v_mfma_f32_16x16x32, the head's dims in an order
//                  that gives a lane 16 consecutive bytes of its token's row per 64 dims
//   online softmax per row over the 32 tokens, fp32
//   O^T[d][row] += V^T[d][tok] . P[tok][row] v_mfma_f32_16x16x32 over the 32 tokens: a lane's
//                  scores are already that product's operand, and V's token-interleaved
//                  layout gives a lane 4 dims x 4 tokens per 16 bytes
// Queries go in as bf16 terms, which hold all of their bits: one of bf16, two of fp16, three of
// fp32.  Weights as two terms, 2^-17 relative, or three for fp32 outputs, 2^-25: below the
// output's rounding.  Their sum is the same product with a row of ones.
//
// What bounds it: HBM where there is enough to read (64 groups of 4 rows x 16 heads of 64, 2048
// tokens each: 46 us, 5.8 TB/s; 256 to 1024 tokens, 85 MB: 18.0 us, of which 5.1 are the launch
// and five dependent loads -- arguments, order, group, length and block ids, pages -- and the
// merge).  The vector units are busy for 7.2 us of these (about 147 operations per 32 tokens, 64
// dims: 32 conversions, 16 differences and products of the softmax, 8 exponentials, 24 that
// split the weights), the matrix units for 1.9 (cycles at 2.4 GHz).  What each step gave, us,
// the same 256 to 1024 tokens / 93 single rows to 1000 tokens, fp16 / 2 rows to 39999 tokens:
//   loads under conditions, each waited for        23.0 / 28.0 / 675
//   buffer loads one iteration ahead, splits       19.6 / 23.7 / 49
//   descriptors in scalar registers, a faster join 18.6 / 21.0 / 30.6
//   scales in the conversions, weights summed by
//   matrix products, non-temporal loads            18.0 / 21.6 / 27.0
//   weights from differences of unscaled scores    18.2 / 21.8 / 27.8
#include <math.h>
#include <stdio.h>

#include "e4m3.h"

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

__device__ __forceinline__ float lane_float(float x, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane));
}

// One lane's share of 32 tokens, two 16-token parts: per 64 dims, 16 dims of token l % 16 (K)
// and 4 dims x 4 tokens (V); and their blocks' scales.
template <int NS> struct Pair {
  uint4 k[2][NS], v[2][NS];
  float ks[2], vs[2];
  bool ok[2];  // holds tokens of the context
};

// The ids and scales of a wave's blocks, 64 at a time in a lane each.  Its i-th 32 tokens are
// the context's (first + i * step)-th: which blocks those are does not hang on the row's
// length, so the first ids are on their way together with it.  The next 64 ids and their
// scales are requested while the current ones are used: ids two refills ahead, scales
// (which need the id) one.
template <int BPP> struct BlockWalk {  // BPP: blocks per 32 tokens
  const int32_t *table;
  const float2 *scales;  // of the head, H apart
  int H, width, first, step;
  int64_t num_blocks;
  int64_t block_bytes;
  int base;        // of the current 64, counted in the wave's own blocks
  uint64_t inside; // lanes whose block lies in the pool
  uint64_t at;     // the block's first byte, of a lane's block
  float2 sc;
  int id1, id2;
  float2 sc1;

  __device__ __forceinline__ int fetch_id(int i) const {
    i += (int)__lane_id();
    const int64_t b = (first + (int64_t)(i / BPP) * step) * BPP + i % BPP;
    return table[min(b, (int64_t)width - 1)];
  }
  __device__ __forceinline__ float2 fetch_scale(int x) const {
    return scales[max(min((int64_t)x, num_blocks - 1), (int64_t)0) * H];
  }
  __device__ __forceinline__ void use(int x) {
    const bool in = x >= 0 && x < num_blocks;
    inside = __builtin_amdgcn_ballot_w64(in);
    at = (uint64_t)(in ? x : 0) * (uint64_t)block_bytes;
  }
  // start() requests, begin() takes what came
  __device__ __forceinline__ void start() {
    base = 0;
    id1 = fetch_id(0);
    id2 = fetch_id(64);
  }
  __device__ __forceinline__ void begin() {
    sc = fetch_scale(id1);
    sc1 = fetch_scale(id2);
    use(id1);
    id1 = id2;
    id2 = fetch_id(128);
  }
  __device__ __forceinline__ void advance() {
    base += 64;
    use(id1);
    sc = sc1;
    sc1 = fetch_scale(id2);
    id1 = id2;
    id2 = fetch_id(base + 128);
  }
};

// A descriptor of `bytes` bytes (wave-uniform) from p on; loads past them return 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_buffer(const uint8_t *p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, __builtin_amdgcn_readfirstlane(bytes),
                                           0x00020000);
}

// Pages are read once a launch: non-temporal loads (64 x 4 rows x 16 heads, 2048 tokens: 46.2
// against 53.7 us, 5.8 TB/s; up to 1024 tokens, 85 MB, no change).
__device__ __forceinline__ uint4 tile_load(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
  constexpr int NON_TEMPORAL = 2;
  return __builtin_bit_cast(uint4,
                            __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, NON_TEMPORAL));
}

// x limited to 0 .. 16, on the scalar unit (a median of three would go to the vector unit, and
// wait there for the registers of loads in flight).
__device__ __forceinline__ int clamp_scalar(int x) {
  int r;
  asm("s_max_i32 %0, %1, 0\n\ts_min_i32 %0, %0, 16" : "=s"(r) : "s"(x) : "scc");
  return r;
}

// What is added to a softmax when its context is split: [row][head][split].  The sums come first
// in the workspace: whole 64-byte pieces, 16-byte aligned for any number of parts.
struct SplitOut {
  float *acc;  // [D]
  float2 *ml;
};

struct Attn8Args {
  const void *q;
  int64_t q_st, q_sh;
  const uint8_t *kc, *vc;
  const float *scales;
  void *out;
  const int32_t *seq_lens, *bt;
  int64_t bt_stride;
  int width, room;  // entries of a table row (one at least), tokens it can list
  const int32_t *group_start, *group_order;
  int64_t num_rows, num_groups;
  int H, D;
  int64_t num_blocks;
  float scale_log2;  // its magnitude: the query takes the sign
  uint32_t q_sign;   // flips the sign of a word's elements
  bool q_vec;  // every 8 elements of a query are 16-byte aligned
  int splits;
  SplitOut part;
};

constexpr int ATTN8_COLS = 8;  // rows of a group
constexpr float NO_SCORE = -3.402823466e38f;  // the least finite score

// Maximum across the four 16-lane rows, a NaN passed on.
__device__ __forceinline__ float rows_maximum4(float x) {
  const auto a =
      __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_elementwise_maximum(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Rows of the group at dispatch position `pos`, from row0 on (0: no such group).
__device__ __forceinline__ int group_rows(const Attn8Args &a, int64_t pos, int64_t &row0) {
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
  return (int)min((int64_t)min(n, ATTN8_COLS), a.num_rows - row0);
}

// NS: ceil(D / 64).  PARTS: 16-token parts of a block.  NW waves split a context, and
// a.splits workgroups do where there are few rows (their sums then go to a.part).
template <int DT, int NS, int PARTS, int NW>
__global__ __launch_bounds__(64 * NW) void attention_8bit_kernel(Attn8Args a) {
  using T = typename Elem<DT>::T;
  constexpr int QT = Terms<DT>::Q, PT = Terms<DT>::P;
  constexpr int COLS = ATTN8_COLS;
  constexpr int BPP = 2 / PARTS;  // blocks per 32 tokens
  __shared__ float s_acc[NW][64 * NS][COLS + 1];
  __shared__ float s_ml[NW][2][COLS];

  // (known to be wave-uniform, so that descriptors live in scalar registers)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, rg = lane >> 4;
  const int H = a.H, D = a.D;
  int64_t pos;
  int h;
  xcd_position(blockIdx.x, (unsigned)H, pos, h);
  const int split = (int)(pos % a.splits);
  int64_t row0;
  const int nrows = group_rows(a, pos / a.splits, row0);
  if (nrows <= 0) return;

  BlockWalk<BPP> walk;
  walk.table = a.bt + row0 * a.bt_stride;
  walk.scales = reinterpret_cast<const float2 *>(a.scales) + h;
  walk.H = H;
  walk.width = a.width;
  walk.first = split * NW + wave;
  walk.step = a.splits * NW;
  walk.num_blocks = a.num_blocks;
  walk.block_bytes = (int64_t)H * 16 * PARTS * D;
  walk.start();
  const int L = min(max(a.seq_lens[row0], 0), a.room);
  const int pairs = (L + 31) / 32;
  const int first = split * NW + wave, step = a.splits * NW;
  const int count = first < pairs ? (pairs - first - 1) / step + 1 : 0;  // of this wave

  // Query: per 64 dims, dims 16 rg .. + 7 and + 8 .. + 15 of row `col`
  constexpr int QV = DT == VFL_FLOAT32 ? 2 : 1;  // 16-byte vectors of 8 elements
  uint4 qraw[NS][2][QV];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = 64 * s + 16 * rg + 8 * e;
      const bool in = col < nrows && d < D;
      const T *p = (const T *)a.q + (row0 + (in ? col : 0)) * a.q_st + h * a.q_sh + (in ? d : 0);
#pragma unroll
      for (int i = 0; i < QV; ++i) {
        if (a.q_vec) qraw[s][e][i] = reinterpret_cast<const uint4 *>(p)[i];
        else qraw[s][e][i] = load16_unaligned<DT>(p + 4 * i);
        uint4 &r = qraw[s][e][i];
        r = in ? make_uint4(r.x ^ a.q_sign, r.y ^ a.q_sign, r.z ^ a.q_sign, r.w ^ a.q_sign)
               : make_uint4(0, 0, 0, 0);
      }
    }

  floatx4_t acc[NS][4];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[s][c] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  // the sum of the weights, of the row `col`: the same products with a row of ones for V
  floatx4_t sum = {0.f, 0.f, 0.f, 0.f};
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  // A row's reference, an unscaled score; weights are exp2((score - m) * scale_log2).  (A product
  // m * scale_log2 would lose its units from 2^24 on, and exp2's whole range from 2^32.)
  float m = NEG_INF_F;  // the first score moves it

  // A part's tile is read through a buffer descriptor that ends with its last token: what lies
  // behind, or an id outside the pool, or dims past the head, reads as 0 without a branch.
  uint32_t k_off[NS], v_off[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    k_off[s] = 64 * s + 16 * rg < D ? col * D + 64 * s + 16 * rg : 0x7fffffffu;
    v_off[s] = 64 * s + 4 * col < D ? (rg * D + 64 * s + 4 * col) * 4 : 0x7fffffffu;
  }
  const uint8_t *kh = a.kc + (int64_t)h * 16 * PARTS * D, *vh = a.vc + (int64_t)h * 16 * PARTS * D;
  // the wave's i-th 32 tokens (nothing at and past `count`)
  auto load = [&](int i, Pair<NS> &x) {
    const int left = L - 32 * (first + i * step);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int from = (i * BPP + u / PARTS - walk.base) & 63;  // lane of the part's block
      const bool in = (walk.inside >> from) & 1;
      const int n = in ? clamp_scalar(left - 16 * u) : 0;  // the part's tokens
      const float ks = lane_float(walk.sc.x, from), vs = lane_float(walk.sc.y, from);
      x.ok[u] = n > 0;
      x.ks[u] = n > 0 ? ks : 1.f;
      x.vs[u] = n > 0 ? vs : 1.f;
      const uint64_t at =
          ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(walk.at >> 32), from) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)walk.at, from)) +
          (uint32_t)((u % PARTS) * 16 * D);
      const auto kr = tile_buffer(kh + at, n * D);
      const auto vr = tile_buffer(vh + at, (n + 3) / 4 * 4 * D);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        x.k[u][s] = tile_load(kr, k_off[s]);
        x.v[u][s] = tile_load(vr, v_off[s]);
      }
    }
  };

  auto consume = [&](int p, Pair<NS> &x, const uint4 (&qop)[NS][2][QT]) {
    floatx4_t y[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      y[u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const uint4 w = x.k[u][s];
        const uint2 k0 = e4m3_widen(w.x, x.ks[u]), k1 = e4m3_widen(w.y, x.ks[u]),
                    k2 = e4m3_widen(w.z, x.ks[u]), k3 = e4m3_widen(w.w, x.ks[u]);
#pragma unroll
        for (int t = QT - 1; t >= 0; --t) {
          y[u] = Bf16::qk(make_uint4(k0.x, k0.y, k1.x, k1.y), qop[s][0][t], y[u]);
          y[u] = Bf16::qk(make_uint4(k2.x, k2.y, k3.x, k3.y), qop[s][1][t], y[u]);
        }
      }
    }
    if (32 * p + 32 > L || !x.ok[0] || !x.ok[1]) {  // wave-uniform
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // what lies behind the last token must not meet a zero weight (0 * NaN)
        const int n = x.ok[u] ? L - (32 * p + 16 * u + 4 * rg) : 0;  // tokens of the lane's four
        const uint32_t keep = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j >= n) y[u][j] = NEG_INF_F;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const uint4 v = x.v[u][s];
          x.v[u][s] = make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep);
        }
      }
    }
    // (maxima that pass a NaN on: the others quiet their operands first, one by one)
    float mb = __builtin_elementwise_maximum(
        __builtin_elementwise_maximum(__builtin_elementwise_maximum(y[0][0], y[0][1]), y[0][2]),
        __builtin_elementwise_maximum(
            __builtin_elementwise_maximum(__builtin_elementwise_maximum(y[0][3], y[1][0]), y[1][1]),
            __builtin_elementwise_maximum(y[1][2], y[1][3])));
    mb = rows_maximum4(mb);
    const bool need = (mb - m) * a.scale_log2 > RESCALE_SLACK_LOG2;
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
      const float corr = need ? fast_exp2((m - mb) * a.scale_log2) : 1.f;
      sum *= corr;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[s][c] *= corr;
      m = need ? mb : m;
    }
    const float ref = __builtin_elementwise_maximum(m, NO_SCORE);  // (-inf - -inf is no score)
    float w[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) w[u][j] = fast_exp2((y[u][j] - ref) * a.scale_log2);
    uint4 pop[PT];
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      const uint2 p0 = take_bf16<true>(w[0]), p1 = take_bf16<true>(w[1]);
      pop[t] = make_uint4(p0.x, p0.y, p1.x, p1.y);
    }
#pragma unroll
    for (int t = PT - 1; t >= 0; --t) sum = Bf16::qk(ones, pop[t], sum);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint2 v0 = e4m3_widen((&x.v[0][s].x)[c], x.vs[0]);
        const uint2 v1 = e4m3_widen((&x.v[1][s].x)[c], x.vs[1]);
#pragma unroll
        for (int t = PT - 1; t >= 0; --t)
          acc[s][c] = Bf16::qk(make_uint4(v0.x, v0.y, v1.x, v1.y), pop[t], acc[s][c]);
      }
  };

  // the next 32 tokens' loads go out before the current ones are used
  uint4 qop[NS][2][QT];
  if (count > 0) {
    // (wider heads: a second buffer costs more waves than it hides latency, 64 x 4 rows x 8
    // heads of 128, 256 to 1024 tokens 20.4 against 21.4 us)
    constexpr bool AHEAD = NS <= 1;
    Pair<NS> x, y;
    walk.begin();
    load(0, x);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (DT == VFL_BFLOAT16) {
          qop[s][e][0] = qraw[s][e][0];
        } else {
          float f[8];
#pragma unroll
          for (int i = 0; i < QV; ++i) unpack16<DT>(qraw[s][e][i], f + 4 * i);
          float f0[4] = {f[0], f[1], f[2], f[3]}, f1[4] = {f[4], f[5], f[6], f[7]};
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            const uint2 lo = take_bf16<false>(f0), hi = take_bf16<false>(f1);
            qop[s][e][t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
        }
      }
    // (a load under a condition would make the waits before a use count on its absence)
    auto next = [&](int i, Pair<NS> &z) {
      if (i < count && i * BPP - walk.base >= 64) walk.advance();
      load(i, z);
    };
    for (int i = 0; i < count; i += AHEAD ? 2 : 1) {
      if constexpr (AHEAD) next(i + 1, y);
      consume(first + i * step, x, qop);
      if (i + 1 >= count) break;
      next(AHEAD ? i + 2 : i + 1, x);
      if constexpr (AHEAD) consume(first + (i + 1) * step, y, qop);
    }
  }
  // acc[s][c][j]: dim 64 s + 16 rg + 4 j + c of row `col`
  if (col < COLS) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s_acc[wave][64 * s + 16 * rg + 4 * j + c][col] = acc[s][c][j];
    if (rg == 0) s_ml[wave][0][col] = fmaxf(m, NO_SCORE), s_ml[wave][1][col] = sum[0];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * D; i += 64 * NW) {
    const int r = i / D, d = i % D;
    float M = NO_SCORE;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_ml[w][0][r]);
    float S = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = fast_exp2((s_ml[w][0][r] - M) * a.scale_log2);
      S = fmaf(s_ml[w][1][r], f, S);
      o = fmaf(s_acc[w][d][r], f, o);
    }
    const int64_t at = (row0 + r) * H + h;
    if (a.splits > 1) {
      a.part.acc[(at * a.splits + split) * D + d] = o;
      if (d == 0) a.part.ml[at * a.splits + split] = make_float2(M, S);
    } else {
      store_result<DT>((T *)a.out + at * D + d, S, o);
    }
  }
}

// The splits of a (row, head) joined: a quarter of D threads, a team, take 4 dims each of
// every teams-th split, about a maximum of their own, so that maxima and sums come in one round
// trip; the teams meet in LDS.
constexpr int ATTN8_JOIN_NT = 256;
template <int DT>
__global__ __launch_bounds__(ATTN8_JOIN_NT) void attention_8bit_join_kernel(Attn8Args a) {
  using T = typename Elem<DT>::T;
  __shared__ float4 s_o[ATTN8_JOIN_NT];
  __shared__ float2 s_ml[ATTN8_JOIN_NT];
  int64_t row0;
  if ((int)blockIdx.y >= group_rows(a, blockIdx.x / a.H, row0)) return;
  const int64_t at = (row0 + blockIdx.y) * a.H + blockIdx.x % a.H;
  const int tid = threadIdx.x, quads = a.D / 4, teams = ATTN8_JOIN_NT / quads;
  const int team = tid / quads, quad = tid % quads;
  const float2 *ml = a.part.ml + at * a.splits;
  const float4 *acc = reinterpret_cast<const float4 *>(a.part.acc + at * a.splits * a.D) + quad;
  float M = NO_SCORE, S = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (team < teams) {
#pragma unroll 4
    for (int s = team; s < a.splits; s += teams) {
      const float2 x = ml[s];
      const float4 v = acc[(int64_t)s * quads];
      const float to = fmaxf(M, x.x);
      const float f = fast_exp2((M - to) * a.scale_log2), e = fast_exp2((x.x - to) * a.scale_log2);
      S = S * f + x.y * e;
      o.x = o.x * f + v.x * e, o.y = o.y * f + v.y * e;
      o.z = o.z * f + v.z * e, o.w = o.w * f + v.w * e;
      M = to;
    }
  }
  s_o[tid] = o;
  s_ml[tid] = make_float2(M, S);
  __syncthreads();
  for (int d = tid; d < a.D; d += ATTN8_JOIN_NT) {
    float top = NO_SCORE, sum = 0.f, y = 0.f;
    for (int t = 0; t < teams; ++t) top = fmaxf(top, s_ml[t * quads + d / 4].x);
    for (int t = 0; t < teams; ++t) {
      const float2 x = s_ml[t * quads + d / 4];
      const float e = fast_exp2((x.x - top) * a.scale_log2);
      sum = fmaf(x.y, e, sum);
      y = fmaf((&s_o[t * quads + d / 4].x)[d % 4], e, y);
    }
    store_result<DT>((T *)a.out + at * a.D + d, sum, y);
  }
}

// Waves of a workgroup and workgroups of a context.  A workgroup a CU or fewer takes eight waves
// (eight against four, us: 12 of 590 tokens 5.6 / 6.4, 256 of 256 to 1024, fp32, 8.6 / 9.5; 384
// of 100 to 1000 9.4 / 9.0, 1024 of 256 to 1024 19.9 / 18.5); wide heads, whose waves hold more
// and are fewer on a CU, up to two (320 of 192 dims 21.4 / 26.5).  A context of more than 192 KB is
// split where four parts or more fill waves that the card would hold and leave each 64 tokens; the
// join costs 4.6 us (512 workgroups of 128 dims to 1024 tokens 24.9 in two parts, 20.5 whole; 16
// heads of 64, one group: 1024 tokens 8.8 split, 7.0 whole; 2048 8.8 / 10.3; 4096 9.1 / 16.4; 2
// rows of 17001 and 39999 tokens x 8 heads of 128 27.0 in 16 parts, 27.6 in 8, 28.6 in 32).
struct Attn8Plan {
  int waves, splits;
};

inline Attn8Plan attn8_plan(int64_t num_groups, int H, int D, int64_t max_tokens) {
  // waves of a launch that the card holds at once, by the registers that a head of D takes
  const int64_t resident = 256 * (D <= 128 ? 16 : D <= 192 ? 12 : D <= 256 ? 8 : 4);
  const int64_t wgs = num_groups * H;
  Attn8Plan p{D <= 256 && wgs <= (D <= 64 ? 256 : 512) ? 8 : 4, 1};
  const int64_t bytes = max_tokens * 2 * D;
  if (bytes > (192 << 10) && wgs * p.waves < resident) {
    const int64_t fill = resident / (wgs * p.waves);
    const int64_t most = max_tokens / 32 / (p.waves * 2);
    const int64_t parts = fill < most ? fill : most;
    if (parts >= 4) p.splits = (int)parts;
  }
  return p;
}

template <int DT, int NS, int PARTS>
static void launch_attention_8bit(const Attn8Args &a, int waves, hipStream_t stream) {
  const dim3 grid((unsigned)xcd_grid(a.num_groups * a.splits, a.H));
#define VFL_ATTN8(NW) \
  attention_8bit_kernel<DT, NS, PARTS, NW><<<grid, dim3(64 * NW), 0, stream>>>(a)
  if constexpr (NS == 8) VFL_ATTN8(4);
  else if (waves == 8) VFL_ATTN8(8);
  else VFL_ATTN8(4);
#undef VFL_ATTN8
}

template <int DT, int PARTS>
static int launch_attention_8bit_steps(const Attn8Args &a, int waves, hipStream_t stream) {
  switch ((a.D + 63) / 64) {
    case 1: launch_attention_8bit<DT, 1, PARTS>(a, waves, stream); break;
    case 2: launch_attention_8bit<DT, 2, PARTS>(a, waves, stream); break;
    case 3: launch_attention_8bit<DT, 3, PARTS>(a, waves, stream); break;
    case 4: launch_attention_8bit<DT, 4, PARTS>(a, waves, stream); break;
    default: launch_attention_8bit<DT, 8, PARTS>(a, waves, stream); break;  // head size 512
  }
  int st = launch_status("attention_with_kv_cache_8bit");
  if (st != VFL_OK || a.splits == 1) return st;
  const unsigned rows = a.group_start ? ATTN8_COLS : 1;
  attention_8bit_join_kernel<DT>
      <<<dim3((unsigned)(a.num_groups * a.H), rows), dim3(ATTN8_JOIN_NT), 0, stream>>>(a);
  return launch_status("attention_with_kv_cache_8bit");
}

}  // namespace vfl

using namespace vfl;

// Bytes a (row, head) of one split takes in the workspace.
static int64_t attn8_part_bytes(int head_dim) { return head_dim * 4 + 8; }

extern "C" int64_t vfl_attention_8bit_workspace(int64_t num_rows, int64_t num_groups,
                                                int num_heads, int head_dim, int block_size,
                                                int64_t max_blocks_per_seq) {
  if (num_rows <= 0 || num_groups <= 0 || num_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      max_blocks_per_seq <= 0)
    return 0;
  const Attn8Plan p =
      attn8_plan(num_groups, num_heads, head_dim, max_blocks_per_seq * block_size);
  return p.splits > 1 ? num_rows * num_heads * p.splits * attn8_part_bytes(head_dim) : 0;
}

extern "C" int vfl_attention_with_kv_cache_8bit(
    const void *query, int64_t query_stride_token, int64_t query_stride_head, const void *k_cache,
    const void *v_cache, const float *kv_scales, void *out, const int32_t *seq_lens,
    const int32_t *block_table, int64_t block_table_stride, int64_t max_blocks_per_seq,
    const int32_t *group_start, const int32_t *group_order, int64_t num_rows, int64_t num_groups,
    int num_heads, int head_dim, int block_size, int64_t num_blocks, float scale, int dtype,
    void *workspace, void *stream) {
  clear_error();
  const char *who = "attention_with_kv_cache_8bit";
  const int st = check_8bit_cache(who, dtype, num_heads, head_dim, block_size, num_blocks);
  if (st != VFL_OK) return st;
  if (num_rows < 0 || num_groups < 0 || num_groups > num_rows ||
      (!group_start && num_groups != num_rows) || max_blocks_per_seq < 0 ||
      max_blocks_per_seq > (1LL << 30) / block_size || block_table_stride < max_blocks_per_seq ||
      num_groups > (1LL << 31) || !grid_fits(xcd_grid(num_groups, num_heads), 256)) {
    set_error("%s: bad sizes (rows %lld groups %lld table %lld wide, stride %lld)", who,
              (long long)num_rows, (long long)num_groups, (long long)max_blocks_per_seq,
              (long long)block_table_stride);
    return VFL_E_INVALID;
  }
  if (!(fabsf(scale) < INFINITY)) {
    set_error("%s: scale %f", who, (double)scale);
    return VFL_E_INVALID;
  }
  if (num_rows == 0 || num_groups == 0) return VFL_OK;
  if (!query || !out || !seq_lens || (max_blocks_per_seq && !block_table) ||
      (num_blocks && (!k_cache || !v_cache || !kv_scales))) {
    set_error("%s: null pointer argument", who);
    return VFL_E_INVALID;
  }
  const int eb = elem_bytes(dtype);
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)kv_scales % 8 ||
      (uintptr_t)query % eb || (uintptr_t)out % eb || (uintptr_t)workspace % 16) {
    set_error("%s: misaligned pointer (caches and workspace 16 bytes, scales 8, others their "
              "element)",
              who);
    return VFL_E_INVALID;
  }
  // an empty pool holds nothing: every row is zero
  const int64_t table = num_blocks ? max_blocks_per_seq : 0;
  Attn8Args a{query, query_stride_token, query_stride_head, (const uint8_t *)k_cache,
              (const uint8_t *)v_cache, kv_scales, out, seq_lens, block_table,
              block_table_stride, (int)table, (int)table * block_size, group_start, group_order,
              num_rows, num_groups, num_heads, head_dim, num_blocks,
              // finite and not 0, which would make NaN of an equal or a masked score (the least
              // denormal in its place moves no weight by more than 2^-21)
              fminf(fmaxf(fabsf(scale) * 1.4426950408889634f, __FLT_DENORM_MIN__), -NO_SCORE),
              !(scale < 0.f) ? 0u : dtype == VFL_FLOAT32 ? 0x80000000u : 0x80008000u,
              (uintptr_t)query % 16 == 0 && query_stride_token % (16 / eb) == 0 &&
                  query_stride_head % (16 / eb) == 0,
              1, {nullptr, nullptr}};
  if (table == 0) a.bt = seq_lens, a.bt_stride = 0, a.width = 1;  // read, and not used
  const Attn8Plan plan = attn8_plan(num_groups, num_heads, head_dim, table * block_size);
  if (plan.splits > 1) {
    if (!workspace) {
      set_error("%s: null workspace", who);
      return VFL_E_INVALID;
    }
    a.splits = plan.splits;
    const int64_t parts = num_rows * num_heads * plan.splits;
    a.part.acc = (float *)workspace;
    a.part.ml = (float2 *)(a.part.acc + parts * head_dim);
  }
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return block_size == 16 ? launch_attention_8bit_steps<DT, 1>(a, plan.waves, s)
                            : launch_attention_8bit_steps<DT, 2>(a, plan.waves, s);
  };
  if (dtype == VFL_FLOAT32) return go(std::integral_constant<int, VFL_FLOAT32>{});
  if (dtype == VFL_BFLOAT16) return go(std::integral_constant<int, VFL_BFLOAT16>{});
  return go(std::integral_constant<int, VFL_FLOAT16>{});
}
