// Attention of packed runs of queries, each over its own run of keys and values (gfx950):
//   out[r][h] = softmax_j(scale * <q[r][h], k[j][h]>) v[j][h],  j over the keys of r's sequence
//
// Scores are computed transposed, S^T[key][query] = K Q^T (32x32x16 products), so a lane holds
// one query's column: the softmax reduces inside the lane plus one half-wave swap, the output
// O^T[dim][query] is rescaled by a lane scalar, and the weights are already in the second
// product's operand order: its k index runs over the keys in the order the first product left
// them (half-wave hf of step s holds keys 16 s + 4 hf + 0..3 and 16 s + 8 + 4 hf + 0..3).  V lies
// in LDS as it came, key by key, and is turned by the transposing reads.
//
// 16-bit inputs go in as they are, the weights rounded to that type (fp16's times 2^14, which keeps
// those down to 2^-28 of the largest clear of its subnormals; the others' times 2^-20).  fp32 goes in as three bf16 terms
// each, rounded, of whose nine products the six largest are taken: the others are 2^-26 of the whole
// or less.
#pragma once

#include <math.h>
#include <stdio.h>

#include <utility>

#include "split_softmax.h"

namespace vfl {

struct CrossArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  void *out;
  const int32_t *q_start, *k_start;  // [sequences + 1]
  int64_t num_queries, num_keys;     // rows of q and out, of k and v
  int sequences, H, D;
  int tiles;         // query tiles of a sequence in the launch (more run in turn)
  float scale_log2;  // its magnitude: the query takes the sign
  bool negative;
  bool vec;          // every 8 elements of q, k and v are 16-byte aligned
  bool out_vec;      // every 4 elements of out are aligned
  int splits;
  SplitOut part;
};

int launch_cross_f32(const CrossArgs &a, int ks, hipStream_t stream);
int launch_cross_bf16(const CrossArgs &a, int ks, hipStream_t stream);
int launch_cross_f16(const CrossArgs &a, int ks, hipStream_t stream);

// Key groups that a launch may take (their tiles have to fit the LDS).
inline int cross_most_groups(bool f32, int DG) { return !f32 || DG <= 2 ? 4 : DG <= 4 ? 2 : 1; }

#ifdef VFL_CROSS_KERNEL
namespace {

typedef float floatx16_t __attribute__((ext_vector_type(16)));

template <int DT> __device__ __forceinline__ floatx16_t mfma32(uint4 a, uint4 b, floatx16_t c) {
  if constexpr (DT == VFL_FLOAT16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a),
                                                  __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// A bf16 term of four floats, rounded, with the remainder left in f.  (In the first one, magnitudes
// that would round to infinity give the largest finite one, and their remainder the rest: so do
// an infinity and a NaN, which the second term then is.)
__device__ __forceinline__ uint2 take_rounded(float (&f)[4], bool first) {
  constexpr float MOST = 3.38953138925153547590e38f;
  float c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = first ? __builtin_amdgcn_fmed3f(f[i], -MOST, MOST) : f[i];
  const uint2 w = make_uint2(Bf16::narrow2(c[0], c[1]), Bf16::narrow2(c[2], c[3]));
  f[0] -= Bf16::widen_lo(w.x), f[1] -= Bf16::widen_hi(w.x);
  f[2] -= Bf16::widen_lo(w.y), f[3] -= Bf16::widen_hi(w.y);
  return w;
}

// The value of lane l ^ 32 and the lane's own, in some order.
__device__ __forceinline__ void half_pair(float x, float &a, float &b) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  a = __uint_as_float(s[0]);
  b = __uint_as_float(s[1]);
}

// Of 16 lanes, lane 4 i + c points to 4 elements of row i; lane n gets the four rows' element n
// of the 16 that the lanes point to.
__device__ __forceinline__ uint2 read_turned(const uint8_t *p) {
  typedef short4_t __attribute__((address_space(3))) *lds_t;
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(uint32_t)(uintptr_t)p));
}

// Shape of a launch: heads of up to 32 DG dims, KS key groups of 4 / KS waves.
template <int DT, int DG, int KS> struct CrossShape {
  static constexpr bool F32 = DT == VFL_FLOAT32;
  static constexpr int PLANES = F32 ? 3 : 1;   // bf16 terms
  static constexpr int KT = DG > 1 && (F32 || DG > 4 || (DG > 2 && KS > 1)) ? 32 : 64;  // keys of a tile
  static constexpr int STRIDE = DG * 64 + 16;  // bytes of a tile's row: rows on different banks
  static constexpr int PLANE = KT * STRIDE;
  static constexpr int TILE = 2 * PLANES * PLANE;  // K, then V
  static constexpr int BUFS = 2 * KS * TILE <= 160 * 1024 ? 2 : 1;
  static constexpr int GW = 4 / KS;            // waves of a key group
  static constexpr int QT = 32 * GW;           // queries of a workgroup
  static constexpr int GT = 64 * GW;           // threads of a key group
  static constexpr int PIECES = KT * DG * 4;   // of 8 elements, of K or V
  static constexpr int CH = (PIECES + GT - 1) / GT;  // a thread's
  static_assert(BUFS * KS * TILE <= 160 * 1024, "the tiles fit the LDS");
};

template <int DT, int DG, int KS>
__global__ __launch_bounds__(256) void cross_attention_kernel(CrossArgs a) {
  using S = CrossShape<DT, DG, KS>;
  using T = typename Elem<DT>::T;
  constexpr int PLANES = S::PLANES, KT = S::KT, STRIDE = S::STRIDE, GW = S::GW, GT = S::GT;
  constexpr int CH = S::CH, BUFS = S::BUFS, QT = S::QT;
  constexpr int KB = KT / 32;                        // 32-key blocks of a tile
  constexpr int RAW = S::F32 ? 2 : 1;                // 16-byte words of 8 elements
  constexpr int MDT = S::F32 ? VFL_BFLOAT16 : DT;    // the products' type
  constexpr int PART = 16 * DG + 2;                  // a lane's partial result
  // of a row's largest weight: fp16's small weights stay normal numbers; sums of up to 2^20 of the
  // other types' largest values stay finite
  constexpr float WEIGHT_LOG2 = DT == VFL_FLOAT16 ? 14.f : -20.f;
  __shared__ __align__(16) uint8_t s_tile[BUFS * KS * S::TILE];
  static_assert((KS - 1) * GW * 64 * PART * 4 <= (int)sizeof(s_tile),
                "the partial outputs fit the tile buffers");

  // A (sequence, head)'s query tiles run on one XCD, which then reads its K/V once: ids go to XCDs
  // round robin, so they are laid out as 8 pairs x tiles x splits.
  const int per = a.tiles * a.splits;
  const int64_t u = blockIdx.x;
  const int64_t pair = 8 * (u / 8 / per) + u % 8;
  if (pair >= (int64_t)a.sequences * a.H) return;
  const int within = (int)(u / 8 % per);
  const int split = within % a.splits;
  const int n = (int)(pair / a.H), h = (int)(pair % a.H);
  const int D = a.D;
  const int64_t qa = min(max((int64_t)a.q_start[n], (int64_t)0), a.num_queries);
  const int nq = (int)(min(max((int64_t)a.q_start[n + 1], qa), a.num_queries) - qa);
  const int64_t ka = min(max((int64_t)a.k_start[n], (int64_t)0), a.num_keys);
  const int nk = (int)(min(max((int64_t)a.k_start[n + 1], ka), a.num_keys) - ka);
  const T *k = (const T *)a.k + ka * a.k_st + h * a.k_sh;
  const T *v = (const T *)a.v + ka * a.v_st + h * a.v_sh;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int grp = wave / GW, gw = wave % GW;  // key group, wave within it
  const int gt = threadIdx.x % GT;
  const int col = lane & 31, hf = lane >> 5;
  uint8_t *tile0 = s_tile + grp * S::TILE;
  constexpr int BUF = KS * S::TILE;

  // this split's tiles
  const int all = (nk + KT - 1) / KT;
  const int tile_first = (int)((int64_t)all * split / a.splits);
  const int ntiles = (int)((int64_t)all * (split + 1) / a.splits) - tile_first;
  const int steps = (ntiles + KS - 1) / KS;

  uint4 kr[CH][RAW], vr[CH][RAW];
  auto read8 = [&](const T *p, bool in, uint4 (&r)[RAW]) {
#pragma unroll
    for (int i = 0; i < RAW; ++i) {
      r[i] = make_uint4(0, 0, 0, 0);
      if (in) {
        if (a.vec) r[i] = reinterpret_cast<const uint4 *>(p)[i];
        else r[i] = load16_unaligned<DT>(p + 4 * i);
      }
    }
  };
  auto load = [&](int t) {  // keys past the run and dims past the head are zeros
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int idx = gt + GT * i, d = 8 * (idx % (4 * DG));
      const int64_t key = (int64_t)(tile_first + t) * KT + idx / (4 * DG);
      const bool in = key < nk && d < D && idx < S::PIECES;
      read8(k + key * a.k_st + d, in, kr[i]);
      read8(v + key * a.v_st + d, in, vr[i]);
    }
  };
  auto put = [&](uint8_t *to, const uint4 (&r)[RAW]) {
    if constexpr (!S::F32) {
      *reinterpret_cast<uint4 *>(to) = r[0];
    } else {
      float f0[4], f1[4];
      unpack16<VFL_FLOAT32>(r[0], f0);
      unpack16<VFL_FLOAT32>(r[1], f1);
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        const uint2 lo = take_rounded(f0, p == 0), hi = take_rounded(f1, p == 0);
        *reinterpret_cast<uint4 *>(to + p * S::PLANE) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    }
  };
  auto store = [&](int buf) {
    uint8_t *kt = tile0 + buf * BUF, *vt = kt + PLANES * S::PLANE;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int idx = gt + GT * i, at = idx / (4 * DG) * STRIDE + idx % (4 * DG) * 16;
      if (S::PIECES % GT == 0 || idx < S::PIECES) {
        put(kt + at, kr[i]);
        put(vt + at, vr[i]);
      }
    }
  };

  for (int tile = within / a.splits; tile * QT < nq; tile += a.tiles) {
    const int query = tile * QT + 32 * gw + col;
    uint4 qop[2 * DG][PLANES];
#pragma unroll
    for (int kk = 0; kk < 2 * DG; ++kk) {
      const int d = 16 * kk + 8 * hf;
      const T *p = (const T *)a.q + (qa + min(query, nq - 1)) * a.q_st + h * a.q_sh + d;
      uint4 r[RAW];
      read8(p, d < D, r);
      if (a.negative) {
        const uint32_t sign = S::F32 ? 0x80000000u : 0x80008000u;
#pragma unroll
        for (int i = 0; i < RAW; ++i) r[i].x ^= sign, r[i].y ^= sign, r[i].z ^= sign, r[i].w ^= sign;
      }
      if constexpr (S::F32) {
        float f0[4], f1[4];
        unpack16<VFL_FLOAT32>(r[0], f0);
        unpack16<VFL_FLOAT32>(r[1], f1);
#pragma unroll
        for (int t = 0; t < PLANES; ++t) {
          const uint2 lo = take_rounded(f0, t == 0), hi = take_rounded(f1, t == 0);
          qop[kk][t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      } else {
        qop[kk][0] = r[0];
      }
    }

    floatx16_t o[DG];
#pragma unroll
    for (int b = 0; b < DG; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
    float m = NO_SCORE, l = 0.f;

    auto attend = [&](int t, int buf) {
      const uint8_t *kt = tile0 + buf * BUF, *vt = kt + PLANES * S::PLANE;
      floatx16_t s[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 2 * DG; ++kk) {
          const uint8_t *at = kt + (32 * b + col) * STRIDE + (2 * kk + hf) * 16;
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) {
            const uint4 kop = *reinterpret_cast<const uint4 *>(at + p * S::PLANE);
#pragma unroll
            for (int t = PLANES - 1 - p; t >= 0; --t) s[b] = mfma32<MDT>(kop, qop[kk][t], s[b]);
          }
        }
      }
      const int left = nk - (tile_first + t) * KT;
      if (left < KT) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * b + 8 * (i / 4) + 4 * hf + i % 4 >= left) s[b][i] = NEG_INF_F;
      }
      float mx = NO_SCORE;
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
      float ma, mb;
      half_pair(mx, ma, mb);
      mx = fmaxf(ma, mb);
      const bool need = mx > m;
      if (__builtin_amdgcn_ballot_w64(need) != 0) {
        const float corr = need ? fast_exp2((m - mx) * a.scale_log2) : 1.f;
        l *= corr;
#pragma unroll
        for (int b = 0; b < DG; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][i] *= corr;
        m = need ? mx : m;
      }
      const float ms = m * a.scale_log2 - WEIGHT_LOG2;
      // One operation a weight where the product m * scale keeps its units to 2^-8 (what it is
      // rounded by is the same for every weight of the row), two where it does not: by row, so
      // that none hangs on its neighbours
      const bool small = fabsf(ms) <= 65536.f;
      if (__builtin_amdgcn_ballot_w64(!small) == 0) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] = fast_exp2(fmaf(s[b][i], a.scale_log2, -ms));
      } else {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float one = fmaf(s[b][i], a.scale_log2, -ms);
            const float two = fmaf(s[b][i] - m, a.scale_log2, WEIGHT_LOG2);
            s[b][i] = fast_exp2(small ? one : two);
          }
      }
      float sum = 0.f;
#pragma unroll
      for (int st = 0; st < KT / 16; ++st) {
        const int e = 8 * (st & 1);
        float p0[4], p1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p0[i] = s[st >> 1][e + i], p1[i] = s[st >> 1][e + 4 + i];
        uint4 pop[PLANES];
        if constexpr (S::F32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += p0[i] + p1[i];
#pragma unroll
          for (int t = 0; t < PLANES; ++t) {
            const uint2 lo = take_bf16<true>(p0), hi = take_bf16<true>(p1);
            pop[t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
        } else {
          // the normaliser sums the weights as they are, which the product sees rounded
          pop[0] = make_uint4(Mfma<DT>::narrow2(p0[0], p0[1]), Mfma<DT>::narrow2(p0[2], p0[3]),
                              Mfma<DT>::narrow2(p1[0], p1[1]), Mfma<DT>::narrow2(p1[2], p1[3]));
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += p0[i] + p1[i];
        }
        // 16 lanes: four keys, 16 dims
        const int key = 16 * st + 4 * hf + (lane & 15) / 4;
        const uint8_t *vp = vt + key * STRIDE + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
#pragma unroll
        for (int b = 0; b < DG; ++b) {
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) {
            const uint2 v0 = read_turned(vp + p * S::PLANE + 64 * b);
            const uint2 v1 = read_turned(vp + p * S::PLANE + 64 * b + 8 * STRIDE);
            const uint4 vop = make_uint4(v0.x, v0.y, v1.x, v1.y);
#pragma unroll
            for (int t = PLANES - 1 - p; t >= 0; --t) o[b] = mfma32<MDT>(vop, pop[t], o[b]);
          }
        }
      }
      l += sum;
    };

    // Step t: the group's tile of step t is in buffer t % BUFS, the next one's rows in flight.
    load(grp);
    if constexpr (BUFS == 2) {
      store(0);
      if (steps > 1) load(KS + grp);
      __syncthreads();
      for (int t = 0; t < steps; ++t) {
        if (t + 1 < steps) {
          store((t + 1) & 1);
          if (t + 2 < steps) load((t + 2) * KS + grp);
        }
        if (t * KS + grp < ntiles) attend(t * KS + grp, t & 1);
        __syncthreads();
      }
    } else {
      for (int t = 0; t < steps; ++t) {
        store(0);
        __syncthreads();
        if (t + 1 < steps) load((t + 1) * KS + grp);
        if (t * KS + grp < ntiles) attend(t * KS + grp, 0);
        __syncthreads();
      }
    }
    // both halves of a column hold the same reference and other keys
    {
      float la, lb;
      half_pair(l, la, lb);
      l = la + lb;
    }

    if constexpr (KS > 1) {
      float *part = reinterpret_cast<float *>(s_tile);  // [wave - GW][PART][64]
      if (grp > 0) {
        float *dst = part + (wave - GW) * PART * 64 + lane;
#pragma unroll
        for (int b = 0; b < DG; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) dst[(16 * b + i) * 64] = o[b][i];
        dst[16 * DG * 64] = m;
        dst[(16 * DG + 1) * 64] = l;
      }
      __syncthreads();
      if (grp == 0) {
        float M = m;
#pragma unroll
        for (int g = 1; g < KS; ++g)
          M = fmaxf(M, part[(((g - 1) * GW + gw) * PART + 16 * DG) * 64 + lane]);
        const float f0 = fast_exp2((m - M) * a.scale_log2);
        l *= f0;
#pragma unroll
        for (int b = 0; b < DG; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][i] *= f0;
#pragma unroll
        for (int g = 1; g < KS; ++g) {
          const float *src = part + ((g - 1) * GW + gw) * PART * 64 + lane;
          const float f = fast_exp2((src[16 * DG * 64] - M) * a.scale_log2);
          l = fmaf(src[(16 * DG + 1) * 64], f, l);
#pragma unroll
          for (int b = 0; b < DG; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] = fmaf(src[(16 * b + i) * 64], f, o[b][i]);
        }
        m = M;
      }
      __syncthreads();  // the next tile's stores follow
    }
    if (grp == 0 && query < nq) {
      const int64_t at = (qa + query) * a.H + h;
      if (a.splits > 1) {
        float *dst = a.part.acc + (at * a.splits + split) * D;
#pragma unroll
        for (int b = 0; b < DG; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 32 * b + 8 * i + 4 * hf;
            if (d < D)
              *reinterpret_cast<float4 *>(dst + d) =
                  make_float4(o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]);
          }
        if (hf == 0) a.part.ml[at * a.splits + split] = make_float2(m, l);
      } else {
        T *dst = (T *)a.out + at * D;
        // no keys, or scores of -inf alone: 0; NaN scores stay NaN
        const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;
#pragma unroll
        for (int b = 0; b < DG; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 32 * b + 8 * i + 4 * hf;
            if (d >= D) continue;
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = o[b][4 * i + j] * inv;
            if constexpr (S::F32) {
              if (a.out_vec) *reinterpret_cast<float4 *>(dst + d) = make_float4(y[0], y[1], y[2], y[3]);
              else dst[d] = y[0], dst[d + 1] = y[1], dst[d + 2] = y[2], dst[d + 3] = y[3];
            } else {
              const uint32_t w0 = Mfma<DT>::narrow2(y[0], y[1]), w1 = Mfma<DT>::narrow2(y[2], y[3]);
              if (a.out_vec) {
                *reinterpret_cast<uint2 *>(dst + d) = make_uint2(w0, w1);
              } else {
                dst[d] = (uint16_t)w0, dst[d + 1] = (uint16_t)(w0 >> 16);
                dst[d + 2] = (uint16_t)w1, dst[d + 3] = (uint16_t)(w1 >> 16);
              }
            }
          }
      }
    }
  }
}

// One workgroup a (sequence, head) and query of the sequence.
template <int DT> __global__ __launch_bounds__(JOIN_NT) void cross_join_kernel(CrossArgs a) {
  const int n = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x % a.H);
  const int64_t qa = min(max((int64_t)a.q_start[n], (int64_t)0), a.num_queries);
  const int64_t qb = min(max((int64_t)a.q_start[n + 1], qa), a.num_queries);
  for (int64_t r = qa + blockIdx.y; r < qb; r += gridDim.y) {
    const int64_t at = r * a.H + h;
    join_splits<DT>(a.out, a.part, at, at * a.D, a.D, a.splits, a.scale_log2);
    __syncthreads();
  }
}

template <int DT, int DG, int KS> void launch_cross_shape(const CrossArgs &a, hipStream_t stream) {
  const int64_t pairs = (int64_t)a.sequences * a.H;
  const dim3 grid((unsigned)((pairs + 7) / 8 * 8 * a.tiles * a.splits));
  cross_attention_kernel<DT, DG, KS><<<grid, dim3(256), 0, stream>>>(a);
}

template <int DT, int DG> void launch_cross_groups(const CrossArgs &a, int ks, hipStream_t stream) {
  constexpr int MOST = DT != VFL_FLOAT32 || DG <= 2 ? 4 : DG <= 4 ? 2 : 1;  // cross_most_groups
  if constexpr (MOST >= 4) {
    if (ks == 4) return launch_cross_shape<DT, DG, 4>(a, stream);
  }
  if constexpr (MOST >= 2) {
    if (ks == 2) return launch_cross_shape<DT, DG, 2>(a, stream);
  }
  launch_cross_shape<DT, DG, 1>(a, stream);
}

template <int DT> int launch_cross(const CrossArgs &a, int ks, hipStream_t stream) {
  switch ((a.D + 31) / 32) {
    case 1: launch_cross_groups<DT, 1>(a, ks, stream); break;
    case 2: launch_cross_groups<DT, 2>(a, ks, stream); break;
    case 3: launch_cross_groups<DT, 3>(a, ks, stream); break;
    case 4: launch_cross_groups<DT, 4>(a, ks, stream); break;
    case 5:
    case 6: launch_cross_groups<DT, 6>(a, ks, stream); break;
    default: launch_cross_groups<DT, 8>(a, ks, stream); break;
  }
  const int st = launch_status("packed_cross_attention");
  if (st != VFL_OK || a.splits == 1) return st;
  const unsigned rows = (unsigned)min((int64_t)65535, (int64_t)a.num_queries);
  cross_join_kernel<DT>
      <<<dim3((unsigned)(a.sequences * a.H), rows), dim3(JOIN_NT), 0, stream>>>(a);
  return launch_status("packed_cross_attention");
}

}  // namespace
#endif

}  // namespace vfl
