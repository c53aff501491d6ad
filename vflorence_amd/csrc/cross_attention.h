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
// 16-bit inputs go in as they are, the weights rounded to that type (fp16's times 2^7, which
// keeps those down to 2^-20 of the reference clear of its subnormals; the others' times 2^-20).
// Their sum is that of the rounded weights.  An output is off by up to half an eps of its type times
// sum p |v| beside its own rounding: of random values 1.35 of that alone in the 2-norm (0.0023 for
// 0.0017 in bf16), where positive and negative ones cancel more.  A second term of a weight would
// take that away, at 2 to 16% (8 runs of 60 to 128 queries 13.5 / 15.7 us, 21 and 29 over 17001
// and 39999 keys 48.9 / 50.3).
// fp32 goes in as three bf16 terms each, rounded, of whose nine products the six largest are taken:
// the others are 2^-26 of the whole or less.  An infinity has no such terms and makes NaN of its
// scores or sums: those scores are taken again from the fp32 elements, and of those sums the
// infinite values alone count.
//
// What bounds it: long texts no unit alone (64 texts of 128 to 1024 tokens over 256 to 1024, 16
// heads of 64, bf16: 157 us, 94 GFLOP, 600 TFLOP/s of a large matrix product's 1205; vector units busy
// for 65 us, matrix units for 40, at 2.4 GHz, in three waves a SIMD; each operand read from LDS feeds
// one product, 3 GB in 12 reads for 8 products, 39 us at 128 bytes a clock, and 10 of bank conflicts.
// Copies that left work out: without loading tiles 134, nor storing them 118, nor exponentials 108).
// fp32 its six products (4 texts of 1024 over 1024 105 us, 980 TFLOP/s of bf16 products; 16 of 31 to
// 257 over 256 to 1024, whose workgroups are one round of unequal length, 67).  Few queries HBM: 64
// single tokens over 256 to 1024 keys 35 us, 4.8 TB/s; 21 and 29 over 17001 and 39999, heads of 128,
// fp16, 56 us, 4.1 TB/s (46 to 49 where the last call left some of the keys in the cache).
// What the steps gave, us, these long texts / fp32 / long keys in the cache / 9 over 590:
//   loads under conditions, maxima for every tile               242 / 88 / 61 / 12.4
//   no conditions, 32 keys at a time                            197 / 77 / 54
//   the last tile apart                                         175 / 71 / 50
//   workgroups found by the rows' offsets, no empty ones        168 / 72 / 49 / 9.1
//   weights about the references as they stand                  163 / 67
//   parts, groups and XCDs by the launch's size                 160 / 65 / 46 / 8.7
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
  float scale_log2;  // its magnitude: the query takes the sign
  bool negative;
  bool spread;       // workgroups go to any XCD
  bool out_vec;      // every 4 elements of out are aligned
  int splits;
  SplitOut part;
};

constexpr int CROSS_MAX_STRIDE = 1 << 22;  // elements between keys

int launch_cross_f32(const CrossArgs &a, int ks, hipStream_t stream);
int launch_cross_bf16(const CrossArgs &a, int ks, hipStream_t stream);
int launch_cross_f16(const CrossArgs &a, int ks, hipStream_t stream);

// Key groups that a launch may take (their tiles have to fit the LDS, and what the tiles' rows take
// on their way the registers).
constexpr int cross_most_groups(bool f32, int DG) {
  return f32 ? (DG <= 2 ? 4 : DG <= 4 ? 2 : 1) : (DG <= 4 ? 4 : 2);
}

// Workgroups of a launch.
inline int64_t cross_grid(int64_t num_queries, int64_t sequences, int H, int ks, int splits,
                          bool spread) {
  const int64_t places = num_queries / (128 / ks) + sequences;
  return places * (spread ? H : (H + XCDS - 1) / XCDS * XCDS) * splits;
}

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
// that would round to infinity give the largest finite one, and their remainder the rest.  An
// infinity has no three terms: its third is NaN, which the sums that meet it then are, and by which
// score_of and infinite_values' callers find them.)
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

// Two weights rounded to nearest even and packed, and the sum of a pair and c.
template <int DT> __device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (DT == VFL_FLOAT16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{a, b}, f16x2_t));
  else
    return Bf16::narrow2(a, b);
}
template <int DT> __device__ __forceinline__ float add_pair(uint32_t w, float c) {
  if constexpr (DT == VFL_FLOAT16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, w),
                                  __builtin_bit_cast(f16x2_t, 0x3c003c00u), c, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w),
                                           __builtin_bit_cast(bf16x2_t, 0x3f803f80u), c, false);
}

// Of 16 lanes, lane 4 i + c points to 4 elements of row i; lane n gets the four rows' element n
// of the 16 that the lanes point to.
__device__ __forceinline__ uint2 read_turned(const uint8_t *p) {
  typedef short4_t __attribute__((address_space(3))) *lds_t;
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(uint32_t)(uintptr_t)p));
}

// NaN where one of 16 registers is no finite number.
__device__ __forceinline__ float not_finite(const floatx16_t &x) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) t = fmaf(x[i], 0.f, t);
  return t;
}
// Which of 16 registers are NaN.
__device__ __forceinline__ uint32_t nan_places(const floatx16_t &x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m |= (x[i] != x[i] ? 1u : 0u) << i;
  return m;
}

// The score of a query and a key from their fp32 elements, as the definition has it for infinities.
// (One at a time: it is rare, and registers that it takes are all waves'.)
__device__ __forceinline__ float score_of(const CrossArgs &a, const float *q, const float *k) {
  float s = 0.f;
#pragma unroll 1
  for (int d = 0; d < a.D; ++d) s = fmaf(q[d], k[d], s);
  return a.negative ? -s : s;
}

// The sum of one dim of `keys` values, among them infinities or NaN, beside which the finite ones
// do not count: weighted by a score of -inf they are 0 * inf.  (0: there are none.)
__device__ __forceinline__ float infinite_values(const CrossArgs &a, const float *q, const float *k,
                                                 const float *v, int keys) {
  constexpr int AT_ONCE = 8;
  float r = 0.f;
#pragma unroll 1
  for (int j = 0; j < keys; j += AT_ONCE) {
    float x[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) x[i] = v[min(j + i, keys - 1) * a.v_st];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) finite = finite && fabsf(x[i]) < INFINITY;
    if (finite) continue;
#pragma unroll 1
    for (int i = j; i < min(j + AT_ONCE, keys); ++i) {
      const float y = v[i * a.v_st];
      if (fabsf(y) < INFINITY) continue;
      r += score_of(a, q, k + i * a.k_st) == NEG_INF_F ? NAN : y;
    }
  }
  return r;
}

// Shape of a launch: heads of up to 32 DG dims, KS key groups of 4 / KS waves.
constexpr int WAVES = 4;
template <int DT, int DG, int KS> struct CrossShape {
  static constexpr bool F32 = DT == VFL_FLOAT32;
  static constexpr int PLANES = F32 ? 3 : 1;   // bf16 terms
  static constexpr int KT = DG > 1 && (F32 || DG > 4 || (DG > 2 && KS > 1)) ? 32 : 64;  // keys of a tile
  static constexpr int STRIDE = DG * 64 + 16;  // bytes of a tile's row: rows on different banks
  static constexpr int PLANE = KT * STRIDE;
  static constexpr int TILE = 2 * PLANES * PLANE;  // K, then V
  static constexpr int BUFS = 2 * KS * TILE <= 160 * 1024 ? 2 : 1;
  static constexpr int NW = WAVES;
  static constexpr int GW = NW / KS;           // waves of a key group
  static constexpr int QT = 32 * GW;           // queries of a workgroup
  static constexpr int GT = 64 * GW;           // threads of a key group
  static constexpr int PIECES = KT * DG * 4;   // of 8 elements, of K or V
  static constexpr int CH = (PIECES + GT - 1) / GT;  // a thread's
  // waves of a SIMD at least: three of heads of up to 64 (long texts 162 us; four, which spill, 173);
  // fp32's heads of 96 two, which the LDS leaves them (those of up to 64 have them anyway)
  static constexpr int OCC = KS > 1 ? 1 : F32 ? (DG == 3 ? 2 : 1) : DG <= 2 ? 3 : 1;
  static_assert(BUFS * KS * TILE <= 160 * 1024, "the tiles fit the LDS");
};

// A tile of queries: from `first` on of sequence n's nq (nq: none), which begin at row qa
// and see the nk keys from row ka on.
struct Tile {
  int n, first, nq, nk;
  int64_t qa, ka;
};

// Sequence n's tiles take the launch's places from floor(its first row / QT) + n on, as many as
// there are to the next one's: never fewer than its queries fill, and no more than one to a
// sequence beyond the rows' own.  A wave looks 64 sequences up at a time.
template <int QT> __device__ __forceinline__ Tile find_tile(const CrossArgs &a, int place) {
  const int lane = __lane_id();
  const int rows = (int)a.num_queries, keys = (int)a.num_keys;
  int lo = 0, span = a.sequences;
  while (span > 63) {
    const int step = (span + 63) / 64, n = lo + lane * step;
    const bool in = lane * step < span;
    const int q = min(max(a.q_start[in ? n : lo], 0), rows);
    const uint64_t below = __builtin_amdgcn_ballot_w64(in && q / QT + n <= place);
    const int i = max((int)__builtin_popcountll(below) - 1, 0);
    lo += i * step;
    span = min(step, span - i * step);
  }
  const int n = min(lo + lane, a.sequences);
  const int q = min(max(a.q_start[n], 0), rows), k = min(max(a.k_start[n], 0), keys);
  const uint64_t below = __builtin_amdgcn_ballot_w64(lane < span && q / QT + n <= place);
  const int i = max((int)__builtin_popcountll(below) - 1, 0);  // (span is 63 at most)
  const int qa = __builtin_amdgcn_readlane(q, i), qb = __builtin_amdgcn_readlane(q, i + 1);
  const int ka = __builtin_amdgcn_readlane(k, i), kb = __builtin_amdgcn_readlane(k, i + 1);
  const int nq = max(qb - qa, 0);
  const int64_t first = (int64_t)(place - (qa / QT + lo + i)) * QT;
  return Tile{lo + i, first < 0 || first >= nq ? nq : (int)first, nq, max(kb - ka, 0), qa, ka};
}

template <int DT, int DG, int KS>
__global__ __launch_bounds__(64 * WAVES, (CrossShape<DT, DG, KS>::OCC)) void cross_attention_kernel(
    CrossArgs a) {
  using S = CrossShape<DT, DG, KS>;
  using T = typename Elem<DT>::T;
  constexpr int PLANES = S::PLANES, KT = S::KT, STRIDE = S::STRIDE, GW = S::GW, GT = S::GT;
  constexpr int CH = S::CH, BUFS = S::BUFS, QT = S::QT;
  constexpr int KB = KT / 32;                        // 32 keys' worth of a tile
  constexpr int RAW = S::F32 ? 2 : 1;                // 16-byte words of 8 elements
  constexpr int MDT = S::F32 ? VFL_BFLOAT16 : DT;    // the products' type
  constexpr int PART = 16 * DG + 2;                  // a lane's partial result
  // of the weight of a row's reference: fp16's small weights stay normal numbers, those that pass
  // the reference by the slack finite; sums of up to 2^12 of the other types' largest values stay
  // finite
  constexpr float WEIGHT_LOG2 = DT == VFL_FLOAT16 ? 15.f - RESCALE_SLACK_LOG2 : -20.f;
  // a lane's sum at which a reference moves (a weight that fp16 does not hold is infinite)
  constexpr float MOST_SUM = DT == VFL_FLOAT16 ? 0x1p15f : 0x1p-12f;
  static_assert(RESCALE_SLACK_LOG2 == 8.f, "MOST_SUM is 2^(WEIGHT_LOG2 + slack)");
  __shared__ __align__(16) uint8_t s_tile[BUFS * KS * S::TILE];
  static_assert((KS - 1) * GW * 64 * PART * 4 <= (int)sizeof(s_tile),
                "the partial outputs fit the tile buffers");

  // A (sequence, head)'s query tiles run on one XCD, which then reads its K/V once: ids go to XCDs
  // round robin, and XCD x takes the heads h of sequence n with (n H + h) % 8 = x.  A launch that
  // the card holds at once goes anywhere: its heads may not fill the XCDs evenly.
  const int lane = threadIdx.x & 63;
  const unsigned ways = a.spread ? 1 : XCDS;
  const unsigned heads = (a.H + ways - 1) / ways;
  const unsigned item = blockIdx.x / ways;
  const int split = (int)(item % a.splits);
  const Tile at = find_tile<QT>(a, (int)(item / a.splits / heads));
  const int h = (int)((blockIdx.x - (unsigned)at.n * (unsigned)a.H) % ways
                      + item / a.splits % heads * ways);
  if (at.first >= at.nq || h >= a.H) return;
  const int D = a.D, nq = at.nq, nk = at.nk;
  const int64_t qa = at.qa, ka = at.ka;
  const T *k = (const T *)a.k + ka * a.k_st + h * a.k_sh;
  const T *v = (const T *)a.v + ka * a.v_st + h * a.v_sh;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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

  // Pieces of rows past the run or of dims past the head are read from the last row's or the head's
  // first ones, so that no load stands under a condition, and stored as zeros.
  uint4 kr[CH][RAW], vr[CH][RAW];
  auto load = [&](int t) {
    const int first = min((tile_first + t) * KT, nk - 1);
    const T *kt = k + first * a.k_st, *vt = v + first * a.v_st;
    const unsigned most = (unsigned)(nk - 1 - first);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const unsigned idx = gt + GT * i, row = min(idx / (4 * DG), most);
      const unsigned d = 8 * (idx % (4 * DG)) < (unsigned)D ? 8 * (idx % (4 * DG)) : 0;
      const uint4 *kp = reinterpret_cast<const uint4 *>(kt + (row * (unsigned)a.k_st + d));
      const uint4 *vp = reinterpret_cast<const uint4 *>(vt + (row * (unsigned)a.v_st + d));
#pragma unroll
      for (int j = 0; j < RAW; ++j) kr[i][j] = kp[j], vr[i][j] = vp[j];
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
  auto store = [&](int t, int buf) {
    uint8_t *kt = tile0 + buf * BUF, *vt = kt + PLANES * S::PLANE;
    const int left = nk - (tile_first + t) * KT;  // rows of the tile that are keys
    if (left < KT || D != 32 * DG) {  // uniform
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int idx = gt + GT * i;
        if (idx / (4 * DG) >= left || 8 * (idx % (4 * DG)) >= D)
#pragma unroll
          for (int j = 0; j < RAW; ++j) kr[i][j] = vr[i][j] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int idx = gt + GT * i, at = idx / (4 * DG) * STRIDE + idx % (4 * DG) * 16;
      if (S::PIECES % GT == 0 || idx < S::PIECES) {
        put(kt + at, kr[i]);
        put(vt + at, vr[i]);
      }
    }
  };

  {
    const int query = at.first + 32 * gw + col;
    const bool active = at.first + 32 * gw < nq;  // (of the wave) some query is one
    const T *qp = (const T *)a.q + (qa + min(query, nq - 1)) * a.q_st + h * a.q_sh;
    auto read_query = [&](int kk, uint4 (&to)[PLANES]) {  // dims 16 kk + 8 hf .. + 7
      const int d = 16 * kk + 8 * hf;
      uint4 r[RAW];
#pragma unroll
      for (int i = 0; i < RAW; ++i) {
        r[i] = make_uint4(0, 0, 0, 0);
        if (16 * kk < D) r[i] = reinterpret_cast<const uint4 *>(qp + d)[i];  // uniform
      }
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
          to[t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      } else {
        to[0] = r[0];
      }
    };
    // (wide fp32 queries' terms would not fit the registers: they are read again for each tile)
    constexpr bool HOLD = !S::F32 || DG <= 4;
    uint4 qop[HOLD ? 2 * DG : 1][PLANES];
    if constexpr (HOLD) {
#pragma unroll
      for (int kk = 0; kk < 2 * DG; ++kk) read_query(kk, qop[kk]);
    }

    floatx16_t o[DG];
#pragma unroll
    for (int b = 0; b < DG; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
    // A row's reference m is a score; weights are 2^(score scale - ms), ms the whole number next to
    // m scale, less WEIGHT_LOG2: exact up to WHOLE, so that weights about different references,
    // key groups' and parts' too, are apart by a power of two.  Where it is larger, they are
    // 2^((score - m) scale + WEIGHT_LOG2).
    constexpr float WHOLE = 65536.f;
    float m = NO_SCORE, l = 0.f;
    float ms = INFINITY;
    bool fresh = true;  // (of the wave) no row has one yet
    bool wide = false;  // (of the wave) some row's ms is past WHOLE
    // log2 of what weights are above those about m itself
    auto above = [&](float m, float ms) {
      return fabsf(ms) <= WHOLE ? fmaf(m, a.scale_log2, -(ms + WEIGHT_LOG2)) : 0.f;
    };

    // 32 keys, the run's from `key0` on, from row 32 b of the buffer on; ragged: `left` of them
    auto attend_block = [&](int key0, int left, int b, int buf, auto ragged) {
      const uint8_t *kt = tile0 + buf * BUF + 32 * b * STRIDE, *vt = kt + PLANES * S::PLANE;
      auto scores = [&]() {
        floatx16_t s;
        if constexpr (S::F32) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 2 * DG; ++kk) {
          const uint8_t *at = kt + col * STRIDE + (2 * kk + hf) * 16;
          if constexpr (!HOLD) read_query(kk, qop[0]);
          const auto &qk = qop[HOLD ? kk : 0];
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) {
            const uint4 kop = *reinterpret_cast<const uint4 *>(at + p * S::PLANE);
#pragma unroll
            for (int t = PLANES - 1 - p; t >= 0; --t) s = mfma32<MDT>(kop, qk[t], s);
          }
        }
        if constexpr (S::F32) __builtin_amdgcn_s_setprio(0);
        if (decltype(ragged)::value && left < 32) {  // uniform
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[i] = 8 * (i / 4) + i % 4 < left - 4 * hf ? s[i] : NEG_INF_F;
        }
        return s;
      };
      // a lane's weights as the second product takes them, and their sum as it sees them
      uint4 pop[2][PLANES];
      float sum;
      auto take = [&](floatx16_t &s) {
        sum = 0.f;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          float p0[4], p1[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) p0[i] = s[8 * st + i], p1[i] = s[8 * st + 4 + i];
          if constexpr (S::F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += p0[i] + p1[i];
#pragma unroll
            for (int t = 0; t < PLANES; ++t) {
              const uint2 lo = take_bf16<true>(p0), hi = take_bf16<true>(p1);
              pop[st][t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
          } else {
            pop[st][0] = make_uint4(narrow2<DT>(p0[0], p0[1]), narrow2<DT>(p0[2], p0[3]),
                                    narrow2<DT>(p1[0], p1[1]), narrow2<DT>(p1[2], p1[3]));
            sum = add_pair<DT>(pop[st][0].x, sum);
            sum = add_pair<DT>(pop[st][0].y, sum);
            sum = add_pair<DT>(pop[st][0].z, sum);
            sum = add_pair<DT>(pop[st][0].w, sum);
          }
        }
      };
      // Weights about the references as they stand, without a look at the scores' maxima: a weight
      // that passes its reference by more than the slack shows in its lane's sum.
      // One operation a weight where the reference is a whole number, two where it is not: by row,
      // so that none hangs on its neighbours.
      auto weights = [&](floatx16_t &s) {
        if (__builtin_expect(!wide, 1)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], a.scale_log2, -ms));
        } else {
          const bool one = fabsf(ms) <= WHOLE;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = fmaf(s[i], a.scale_log2, -ms);
            const float y = fmaf(s[i] - m, a.scale_log2, WEIGHT_LOG2);
            s[i] = fast_exp2(one ? x : y);
          }
        }
        take(s);
      };
      if (__builtin_expect(!fresh, 1)) {
        floatx16_t s = scores();
        weights(s);
      }
      if (__builtin_expect(fresh || __builtin_amdgcn_ballot_w64(!(sum <= MOST_SUM)) != 0, 0)) {
        // rows whose own sums pass the slack move, whatever stands beside them
        bool need = true;
        if (!fresh) {
          float sa, sb;
          half_pair(sum, sa, sb);
          need = !(sa <= MOST_SUM && sb <= MOST_SUM);
        }
        floatx16_t s = scores();
        if constexpr (S::F32) {  // (a NaN weight always comes here)
          const float t = not_finite(s);
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(t != t) != 0, 0)) {
            const uint32_t lost = nan_places(s);
#pragma unroll 1
            for (int n = 0; n < 16; ++n) {
              if (!(lost >> n & 1)) continue;
              const int key = key0 + 8 * (n / 4) + n % 4 + 4 * hf;
              const float x = score_of(a, qp, k + key * a.k_st);
#pragma unroll
              for (int i = 0; i < 16; ++i) s[i] = i == n ? x : s[i];
            }
          }
        }
        float mx = m;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
        float ma, mb;
        half_pair(mx, ma, mb);
        mx = fmaxf(ma, mb);
        const float to = rintf(mx * a.scale_log2) - WEIGHT_LOG2;
        if (!fresh) {
          const float corr =
              need ? fast_exp2((m - mx) * a.scale_log2 + (above(mx, to) - above(m, ms))) : 1.f;
          l *= corr;
#pragma unroll
          for (int d = 0; d < DG; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= corr;
        }
        m = need ? mx : m;
        ms = need ? to : ms;
        fresh = false;
        wide = __builtin_amdgcn_ballot_w64(!(fabsf(ms) <= WHOLE)) != 0;
        weights(s);
      }
      l += sum;
      // (waves in their products go first, so that others' vector work runs beside them: fp32, whose
      // products take most of the time, 68 against 65 us)
      if constexpr (S::F32) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        // 16 lanes: four keys, 16 dims
        const int key = 16 * st + 4 * hf + (lane & 15) / 4;
        const uint8_t *vp = vt + key * STRIDE + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
#pragma unroll
        for (int d = 0; d < DG; ++d) {
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) {
            const uint2 v0 = read_turned(vp + p * S::PLANE + 64 * d);
            const uint2 v1 = read_turned(vp + p * S::PLANE + 64 * d + 8 * STRIDE);
            const uint4 vop = make_uint4(v0.x, v0.y, v1.x, v1.y);
#pragma unroll
            for (int t = PLANES - 1 - p; t >= 0; --t) o[d] = mfma32<MDT>(vop, pop[st][t], o[d]);
          }
        }
      }
      if constexpr (S::F32) __builtin_amdgcn_s_setprio(0);
    };

    auto attend = [&](int t, int buf) {
      const int key0 = (tile_first + t) * KT;
#pragma unroll
      for (int b = 0; b < KB; ++b) attend_block(key0 + 32 * b, 32, b, buf, std::false_type{});
    };
    auto attend_last = [&](int t, int buf) {  // of the run's last tile some rows may be no keys
      const int key0 = (tile_first + t) * KT, left = nk - key0;
#pragma unroll
      for (int b = 0; b < KB; ++b)
        if (left > 32 * b)
          attend_block(key0 + 32 * b, left - 32 * b, b, buf, std::true_type{});
    };

    // Step t: the group's tile of step t is in buffer t % BUFS, the next one's rows in flight.
    // (all but the last step's are whole tiles of every group)
    if (steps > 0) load(grp);
    if constexpr (BUFS == 2) {
      if (steps > 0) store(grp, 0);
      if (steps > 1) load(KS + grp);
      __syncthreads();
#pragma unroll 1
      for (int t = 0; t < steps - 1; ++t) {
        store((t + 1) * KS + grp, (t + 1) & 1);
        if (t + 2 < steps) load((t + 2) * KS + grp);
        if (active) attend(t * KS + grp, t & 1);
        __syncthreads();
      }
    } else {
#pragma unroll 1
      for (int t = 0; t < steps; ++t) {
        store(t * KS + grp, 0);
        __syncthreads();
        if (t + 1 >= steps) break;
        load((t + 1) * KS + grp);
        if (active) attend(t * KS + grp, 0);
        __syncthreads();
      }
    }
    const int last = (steps - 1) * KS + grp;
    if (active && steps > 0 && last < ntiles) attend_last(last, BUFS == 2 ? (steps - 1) & 1 : 0);
    __syncthreads();
    // both halves of a column hold the same reference and other keys
    {
      float la, lb;
      half_pair(l, la, lb);
      l = la + lb;
    }
    if (KS > 1 || a.splits > 1) {  // parts meet about m itself
      const float f = fast_exp2(-above(m, ms));
      l *= f;
#pragma unroll
      for (int b = 0; b < DG; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= f;
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
    }
    if constexpr (S::F32) {
      // Sums that met an infinite value are NaN, whatever its weights: such dims are looked at again.
      // (Before any of the row's results is written, which may be where its query is.)
      const int key0 = tile_first * KT, keys = min(ntiles * KT, nk - key0);
#pragma unroll
      for (int b = 0; b < DG; ++b) {
        const float t = not_finite(o[b]);
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(t != t) == 0, 1)) continue;
        const uint32_t lost = grp == 0 && query < nq && l == l ? nan_places(o[b]) : 0;
#pragma unroll 1
        for (int n = 0; n < 16; ++n) {
          if (!(lost >> n & 1)) continue;  // (a NaN sum has keys; dims past the head are 0)
          const int d = 32 * b + 8 * (n / 4) + n % 4 + 4 * hf;
          const float r = infinite_values(a, qp, k + key0 * a.k_st, v + key0 * a.v_st + d, keys);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][i] = i == n && r != 0.f ? r : o[b][i];
        }
      }
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
        T *dst = (T *)a.out + at * D + 4 * hf;
        // no keys, or scores of -inf alone: 0; NaN scores stay NaN
        const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;
        auto write = [&](auto aligned) {
#pragma unroll
          for (int b = 0; b < DG; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i >= 2 && 32 * b + 16 >= D) continue;  // (head sizes are multiples of 16; uniform)
              if (32 * b >= D) continue;
              T *to = dst + 32 * b + 8 * i;
              float y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] = o[b][4 * i + j] * inv;
              if constexpr (S::F32) {
                if constexpr (decltype(aligned)::value)
                  *reinterpret_cast<float4 *>(to) = make_float4(y[0], y[1], y[2], y[3]);
                else to[0] = y[0], to[1] = y[1], to[2] = y[2], to[3] = y[3];
              } else {
                const uint32_t w0 = narrow2<DT>(y[0], y[1]), w1 = narrow2<DT>(y[2], y[3]);
                if constexpr (decltype(aligned)::value) {
                  *reinterpret_cast<uint2 *>(to) = make_uint2(w0, w1);
                } else {
                  to[0] = (uint16_t)w0, to[1] = (uint16_t)(w0 >> 16);
                  to[2] = (uint16_t)w1, to[3] = (uint16_t)(w1 >> 16);
                }
              }
            }
        };
        if (a.out_vec) write(std::true_type{});
        else write(std::false_type{});
      }
    }
  }
}

// Whether a row is one of a sequence's.
__device__ __forceinline__ bool in_sequence(const CrossArgs &a, int row) {
  int lo = 0, hi = a.sequences;  // the last sequence that begins at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.q_start[mid] <= row) lo = mid;
    else hi = mid;
  }
  return row >= a.q_start[lo] && row < a.q_start[lo + 1];
}

// The splits of each (query, head) joined: of many a workgroup takes one (query, head), of few a
// thread four dims.  (With the attention, us: 60 queries x 8 heads of 128 in 32 parts 31.3 / 45.0, 8
// runs of 20 to 32 x 16 of 64 in four 21.9 / 20.0, 590 x 12 in two, fp32, 25.6 / 20.7.)
constexpr int CROSS_JOIN_NT = 256;
constexpr int CROSS_JOIN_FEW = 8;
template <int DT> __global__ __launch_bounds__(JOIN_NT) void cross_join_many_kernel(CrossArgs a) {
  const int64_t at = blockIdx.x;
  if (!in_sequence(a, (int)(at / a.H))) return;
  join_splits<DT>(a.out, a.part, at, at * a.D, a.D, a.splits, a.scale_log2);
}
template <int DT> __global__ __launch_bounds__(CROSS_JOIN_NT) void cross_join_few_kernel(CrossArgs a) {
  using T = typename Elem<DT>::T;
  const int quads = a.D / 4;
  const int64_t i = (int64_t)blockIdx.x * CROSS_JOIN_NT + threadIdx.x;
  const int64_t at = i / quads;  // query * H + head
  const int row = (int)(at / a.H), d = (int)(i % quads) * 4;
  if (row >= a.num_queries || !in_sequence(a, row)) return;
  const float2 *ml = a.part.ml + at * a.splits;
  const float *acc = a.part.acc + at * a.splits * a.D + d;
  float2 x[CROSS_JOIN_FEW];
  float4 v[CROSS_JOIN_FEW];
#pragma unroll
  for (int s = 0; s < CROSS_JOIN_FEW; ++s) {
    const int at_split = min(s, a.splits - 1);
    x[s] = ml[at_split];
    v[s] = *reinterpret_cast<const float4 *>(acc + (int64_t)at_split * a.D);
  }
  float M = x[0].x;
#pragma unroll
  for (int s = 1; s < CROSS_JOIN_FEW; ++s) M = fmaxf(M, x[s].x);
  float S = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < CROSS_JOIN_FEW; ++s) {
    if (s >= a.splits) break;
    const float e = fast_exp2((x[s].x - M) * a.scale_log2);
    S = fmaf(x[s].y, e, S);
    o[0] = fmaf(v[s].x, e, o[0]), o[1] = fmaf(v[s].y, e, o[1]);
    o[2] = fmaf(v[s].z, e, o[2]), o[3] = fmaf(v[s].w, e, o[3]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) store_result<DT>((T *)a.out + at * a.D + d + j, S, o[j]);
}

template <int DT, int DG, int KS> void launch_cross_shape(const CrossArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)cross_grid(a.num_queries, a.sequences, a.H, KS, a.splits, a.spread));
  cross_attention_kernel<DT, DG, KS><<<grid, dim3(64 * WAVES), 0, stream>>>(a);
}

template <int DT, int DG> void launch_cross_groups(const CrossArgs &a, int ks, hipStream_t stream) {
  constexpr int MOST = cross_most_groups(DT == VFL_FLOAT32, DG);
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
  const int64_t units = a.num_queries * a.H;
  if (a.splits > CROSS_JOIN_FEW) {
    cross_join_many_kernel<DT><<<dim3((unsigned)units), dim3(JOIN_NT), 0, stream>>>(a);
  } else {
    const int64_t threads = units * (a.D / 4);
    cross_join_few_kernel<DT><<<dim3((unsigned)((threads + CROSS_JOIN_NT - 1) / CROSS_JOIN_NT)),
                                dim3(CROSS_JOIN_NT), 0, stream>>>(a);
  }
  return launch_status("packed_cross_attention");
}

}  // namespace
#endif

}  // namespace vfl
