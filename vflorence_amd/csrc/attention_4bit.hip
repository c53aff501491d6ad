// Paged decode attention over a cache held in e2m1 with a scale per token, head and 32 dims
// (e2m1.h), gfx950:
//   out[r][h] = softmax_j(scale * <q[r][h], K4_j[h]>) V4_j[h],  j < seq_lens[r]
//
// The rows of a group (a request's beams over one page list) are few, so the products are the
// 4x4x4 ones of 16 blocks, which waste nothing on four rows, and one operand of which can be one
// block's for all:
//   S[row][tok]  = q[row][:] . K[tok][:]   a lane is a token; the q of 64 dims takes two registers,
//                  a block each 4 dims, and step c hands block c's to all of them.  K's codes times
//                  their scale are exact in bf16: one conversion a pair, which adds the exponent
//   online softmax per row over 64 tokens, fp32, a register a row
//   O[row][d]   += (P[row][tok] vs[tok]) . V[tok][d]   a lane is two dims of its row of lanes'
//                  16 tokens.  A group's V scales go to the weights: 64 tokens' V codes are
//                  converted by a constant, four tokens to a block's operand
// Queries go in as bf16 terms, which hold all of their bits: one of bf16, two of fp16, three of
// fp32.  Weights as two terms, 2^-17 relative, or three for fp32 outputs, 2^-25: below the
// output's rounding.  Their sum is taken in fp32.
//
// What bounds it: HBM, after the launch and five dependent loads (arguments, order, group, length
// and block ids, pages) that every workgroup waits for.  64 groups of 4 rows x 16 heads of 64, 256 to
// 1024 tokens: 13.8 us for 45.5 MB, which a large copy moves in 8.9; 93 single rows to 1000 tokens,
// fp16, 15.0 us for 51 MB; 2 rows of 17001 and 39999 tokens x 8 heads of 128 18.2 us for 62 MB, 3.8 of
// them the join.  Nearly all of a launch's pages are on their way at once (16 waves a CU of two
// buffers of 4.3 KB: 36 MB), so what is left is the chain and the contexts' unequal lengths: four
// steps of 64 tokens a wave for the longest, 2.5 on average.  The vector units are busy for 8.3 us of
// the first (5.09 M quad cycles over 1024 SIMDs at 2.4 GHz: about 64 conversions, 32 operations that
// pair V's tokens, 8 exponentials a 64 tokens of 64 dims, a third of what 16-column tiles would take
// with 12 columns empty), the matrix units for 1.7.
// Pages are read once a launch: non-temporal loads (13.6 against 14.8 us).
#include <math.h>
#include <stdio.h>

#include <algorithm>
#include <utility>

#include "e2m1.h"
#include "split_softmax.h"

namespace vfl {

namespace {

template <typename F, int... I>
__device__ __forceinline__ void call_each(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void static_for(F f) {
  call_each(f, std::make_integer_sequence<int, N>{});
}

// D[i][j] += sum_k A[i][k] B[k][j] in 16 blocks: lane 4 b + i holds A's row i and 4 b + j B's
// column j of block b, four bf16 each; lane 4 b + j register i of D is D[i][j].  A's block is
// block BLOCK of each 2^LOG blocks.
template <int LOG, int BLOCK>
__device__ __forceinline__ floatx4_t blocks4x4(uint2 a, uint2 b, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(__builtin_bit_cast(short4_t, a),
                                                __builtin_bit_cast(short4_t, b), c, LOG, BLOCK, 0);
}

// One lane's share of 64 tokens: its token's dims of K, 16 tokens of two dims of V in each group,
// and the scales of four tokens, K's [group] then V's.
template <int G> struct Chunk {
  uint4 k[G], v[G];
  uint32_t s[2 * G];
  bool ok;  // the lane's token is one of the context
};

struct Attn4Args : DecodeRows {
  const void *q;
  int64_t q_st, q_sh;
  const uint8_t *cache;
  const int32_t *seq_lens, *bt;
  int64_t bt_stride;
  int width, room;  // entries of a table row (one at least), tokens it can list
  int shift;        // 16 << shift tokens a block
  int64_t num_blocks;
  float sign;  // the query's factor
};

template <typename U> __device__ __forceinline__ U load_once(const uint8_t *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const U *>(p));
}
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint4 load16_once(const uint8_t *p) {
  const u32x4_t x = load_once<u32x4_t>(p);
  return make_uint4(x[0], x[1], x[2], x[3]);
}

template <int CTRL> __device__ __forceinline__ float quad(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF,
                                                               true));
}

// What is summed is taken down by 2^-20, so that sums of 2^12 tokens of the largest values (6 *
// 2^125), whose weights pass their reference by the slack, are finite: a weight by 2^-6, which with
// its V scale is 2^127 at most then, V's codes by 2^-14, the weights' own sum by both.  A weight of
// the least scale, 2^-100, keeps its terms above 2^-134: 2^-28 of that scale.  (A smaller slack in
// place of the first costs up to 5% of the time, this up to 1.)
constexpr float WEIGHT_FACTOR = 0x1p-6f, CODE_FACTOR = 0x1p-14f;
static_assert(RESCALE_SLACK_LOG2 <= 8.f, "2^(125 + slack - 6) is finite");

// Four registers to the one of each row of 16 lanes (row q: register q), each summed over the rows.
__device__ __forceinline__ float rows_scatter4(const floatx4_t &x) {
  auto half = [](float a, float b) {  // lanes 0 .. 31: a's sum of halves, 32 .. 63: b's
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                    false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
  };
  const float a = half(x[0], x[2]), b = half(x[1], x[3]);
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                  false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Waves of a workgroup at most: wide heads take more registers than eight leave.
template <int G> constexpr int attn4_threads() { return G > 8 ? 256 : 512; }

// G: groups of 32 dims.  ROWS: 1, 4 or 8, rows of a group taken together (more run in turn).
// blockDim.x / 64 waves split a context, and a.splits workgroups do where there are few rows
// (their sums then go to a.part).
template <int DT, int G, int ROWS>
__global__ __launch_bounds__(attn4_threads<G>()) void attention_4bit_kernel(Attn4Args a) {
  using T = typename Elem<DT>::T;
  constexpr int QT = Terms<DT>::Q, PT = Terms<DT>::P;
  constexpr int QUADS = (ROWS + 3) / 4, QR = ROWS < 4 ? ROWS : 4;  // rows of a quad that are used
  constexpr int NQ = (G + 1) / 2;  // 64 dims' registers of q
  constexpr int DP = 32 * G + 16;  // (rows of the sums on different banks)
  extern __shared__ float s_mem[];
  const int NW = blockDim.x >> 6;
  float *s_acc = s_mem;                         // [NW][4 QUADS][DP]
  float *s_m = s_mem + NW * 4 * QUADS * DP;     // [NW][4 QUADS]
  float *s_l = s_m + NW * 4 * QUADS;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int p16 = lane & 15, rg = lane >> 4;
  const int H = a.H, D = a.D;
  int64_t pos;
  int h;
  xcd_position(blockIdx.x, (unsigned)H, pos, h);
  // (a launch has fewer than 2^32 threads: positions divide in 32 bits)
  const unsigned parts = (unsigned)a.splits, place = (unsigned)pos / parts;
  const int split = (int)((unsigned)pos - place * parts);
  int64_t row0;
  const int nrows = group_rows(a, place, row0);
  if (nrows <= 0) return;

  const int first = split * NW + wave, step = a.splits * NW;
  const int32_t *table = a.bt + row0 * a.bt_stride;
  auto fetch_id = [&](int i) {  // of the lane's part of the wave's i-th 64 tokens
    const int64_t part = (first + (int64_t)i * step) * 4 + rg;
    return table[min(part >> a.shift, (int64_t)a.width - 1)];
  };
  const int id0 = fetch_id(0), id1 = fetch_id(1);
  const int L = min(max(a.seq_lens[row0], 0), a.room);
  const int chunks = (L + 63) / 64;
  const int count = first < chunks ? (chunks - first - 1) / step + 1 : 0;  // of this wave

  const E2m1Layout lay(H, G, 1 << a.shift);
  const uint8_t *kh = a.cache + lay.keys(h, 0), *sh = a.cache + lay.scales(h, 0);
  const int64_t half = lay.half, block_bytes = lay.block_bytes;
  const int sub_mask = (1 << a.shift) - 1;
  // the wave's i-th 64 tokens, whose block (of the lane's part) is `id`: blocks that hold nothing
  // of the context are read as block 0 and not used
  auto load = [&](int i, int id, Chunk<G> &x) {
    const int64_t c = first + (int64_t)i * step;
    const int tok = (int)(c * 64) + lane;
    const bool in = i < count && 64 * c + 16 * rg < L && id >= 0 && id < a.num_blocks;
    x.ok = in && tok < L;
    const int64_t at = (int64_t)(in ? id : 0) * block_bytes;
    const int sub = (int)((c * 4 + rg) & sub_mask);
    const uint8_t *k = kh + at + sub * (G * 256) + p16 * 16;
    const uint8_t *v = k + half;
    const uint8_t *s = sh + at + sub * (G * 32) + (p16 >> 2) * (G * 8);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      x.k[g] = load16_once(k + g * 256);
      x.v[g] = load16_once(v + g * 256);
    }
    if constexpr (G % 2 == 0) {
#pragma unroll
      for (int g = 0; g < G / 2; ++g) {
        const uint4 w = load16_once(s + 16 * g);
        x.s[4 * g] = w.x, x.s[4 * g + 1] = w.y, x.s[4 * g + 2] = w.z, x.s[4 * g + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const u32x2_t w = load_once<u32x2_t>(s + 8 * g);
        x.s[2 * g] = w[0], x.s[2 * g + 1] = w[1];
      }
    }
  };

  for (int r0 = 0; r0 < nrows; r0 += ROWS) {  // (workgroup-uniform)
    // q: lane 4 b + r has dims 64 n + 4 b .. + 3 of row r of each quad
    uint2 q[QUADS][NQ][QT];
#pragma unroll
    for (int u = 0; u < QUADS; ++u)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int r = r0 + 4 * u + (lane & 3), d = 64 * n + 4 * (lane >> 2);
        const bool in = r < nrows && (ROWS > 1 || (lane & 3) == 0) && d < D;
        const T *p = (const T *)a.q + (row0 + (in ? r : 0)) * a.q_st + h * a.q_sh + (in ? d : 0);
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (DT == VFL_FLOAT32) f[i] = p[i];
          else f[i] = Mfma<DT>::widen(p[i]);
          f[i] = in ? f[i] * a.sign : 0.f;
        }
#pragma unroll
        for (int t = 0; t < QT; ++t) q[u][n][t] = take_bf16<false>(f);
      }

    floatx4_t acc[QUADS][G][2];
    float m[QUADS][QR], l[QUADS][QR];
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) acc[u][g][e] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < QR; ++r) m[u][r] = NO_SCORE, l[u][r] = 0.f;
    }

    auto consume = [&](bool begin, const Chunk<G> &x) {
      const int byte = 8 * (lane & 3);  // of the lane's token in a word of scales
      floatx4_t y[QUADS];
#pragma unroll
      for (int u = 0; u < QUADS; ++u) y[u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
      static_for<G>([&](auto g) {
        const float ks = e2m1_scale((x.s[g] >> byte) & 255u);
        const uint32_t w[4] = {x.k[g].x, x.k[g].y, x.k[g].z, x.k[g].w};
        static_for<4>([&](auto i) {
          const uint2 b0 = make_uint2(e2m1_bf16x2<0>(w[i], ks), e2m1_bf16x2<1>(w[i], ks));
          const uint2 b1 = make_uint2(e2m1_bf16x2<2>(w[i], ks), e2m1_bf16x2<3>(w[i], ks));
          constexpr int c = 8 * g + 2 * i;  // of 4 dims
#pragma unroll
          for (int u = 0; u < QUADS; ++u)
#pragma unroll
            for (int t = QT - 1; t >= 0; --t) {
              y[u] = blocks4x4<4, c % 16>(q[u][c / 16][t], b0, y[u]);
              y[u] = blocks4x4<4, c % 16 + 1>(q[u][c / 16][t], b1, y[u]);
            }
        });
      });
      float e[QUADS][QR], most = NO_SCORE;
#pragma unroll
      for (int u = 0; u < QUADS; ++u)
#pragma unroll
        for (int r = 0; r < QR; ++r) {
          y[u][r] = x.ok ? y[u][r] : NEG_INF_F;
          e[u][r] = (y[u][r] - m[u][r]) * a.scale_log2;
          most = fmaxf(most, e[u][r]);
        }
      // the first scores move a row's reference, others only by more than the slack (each row by
      // its own scores, whatever stands beside it)
      if (begin || __builtin_amdgcn_ballot_w64(most > RESCALE_SLACK_LOG2) != 0) {
#pragma unroll
        for (int u = 0; u < QUADS; ++u)
#pragma unroll
          for (int r = 0; r < QR; ++r) {
            if (!begin && __builtin_amdgcn_ballot_w64(e[u][r] > RESCALE_SLACK_LOG2) == 0) continue;
            const float to = fmaxf(wave_max64(y[u][r]), m[u][r]);
            const float corr = fast_exp2((m[u][r] - to) * a.scale_log2);
            m[u][r] = to;
            l[u][r] *= corr;
#pragma unroll
            for (int g = 0; g < G; ++g) acc[u][g][0][r] *= corr, acc[u][g][1][r] *= corr;
            e[u][r] = (y[u][r] - to) * a.scale_log2;
          }
      }
#pragma unroll
      for (int u = 0; u < QUADS; ++u)
#pragma unroll
        for (int r = 0; r < QR; ++r) {
          e[u][r] = fast_exp2(e[u][r]);
          l[u][r] += e[u][r];
        }
      static_for<G>([&](auto g) {
        // (a masked token's scale may be anything)
        const float vs =
            x.ok ? e2m1_scale((x.s[G + g] >> byte) & 255u) * WEIGHT_FACTOR : 0.f;
        uint2 pop[QUADS][PT];
#pragma unroll
        for (int u = 0; u < QUADS; ++u) {
          // tokens to registers: lane 4 b + r has the weights of row r for tokens 4 b + 1, 0, 3, 2
          float p[4];
          if constexpr (QR == 1) {
            const float w = e[u][0] * vs;
            p[0] = quad<0x55>(w), p[1] = quad<0x00>(w), p[2] = quad<0xff>(w), p[3] = quad<0xaa>(w);
          } else {
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = e[u][r] * vs;
            // (the exchanges take all lanes: none may stand under a condition)
            const bool o1 = lane & 1, o2 = lane & 2;
            const float n0 = quad<DPP_QUAD_XOR1>(w[0]), n1 = quad<DPP_QUAD_XOR1>(w[1]);
            const float n2 = quad<DPP_QUAD_XOR1>(w[2]), n3 = quad<DPP_QUAD_XOR1>(w[3]);
            const float a0 = o1 ? n1 : w[0], a1 = o1 ? w[1] : n0;  // rows 0 and 1
            const float b0 = o1 ? n3 : w[2], b1 = o1 ? w[3] : n2;  // rows 2 and 3
            const float fa0 = quad<DPP_QUAD_XOR2>(a0), fa1 = quad<DPP_QUAD_XOR2>(a1);
            const float fb0 = quad<DPP_QUAD_XOR2>(b0), fb1 = quad<DPP_QUAD_XOR2>(b1);
            p[1] = o2 ? fb0 : a0;  // token 0
            p[0] = o2 ? fb1 : a1;  // 1
            p[3] = o2 ? b0 : fa0;  // 2
            p[2] = o2 ? b1 : fa1;  // 3
          }
#pragma unroll
          for (int t = 0; t < PT; ++t) pop[u][t] = take_bf16<true>(p);
        }
        const uint32_t w[4] = {x.v[g].x, x.v[g].y, x.v[g].z, x.v[g].w};
        static_for<4>([&](auto i) {  // tokens 4 i .. + 3 of the part: low halves dim p16, high + 16
          // byte 1 of lo: tokens 1 and 0, byte 3: 3 and 2; of hi bytes 0 and 2
          const uint32_t lo = (w[i] << 12 & 0xf000f000u) | (w[i] & 0x0fff0fffu);
          const uint32_t hi = (w[i] >> 12 & 0x000f000fu) | (w[i] & 0xfff0fff0u);
          const uint2 b0 = make_uint2(e2m1_bf16x2<1>(lo, CODE_FACTOR),
                                      e2m1_bf16x2<3>(lo, CODE_FACTOR));
          const uint2 b1 = make_uint2(e2m1_bf16x2<0>(hi, CODE_FACTOR),
                                      e2m1_bf16x2<2>(hi, CODE_FACTOR));
#pragma unroll
          for (int u = 0; u < QUADS; ++u)
#pragma unroll
            for (int t = PT - 1; t >= 0; --t) {
              acc[u][g][0] = blocks4x4<2, i>(pop[u][t], b0, acc[u][g][0]);
              acc[u][g][1] = blocks4x4<2, i>(pop[u][t], b1, acc[u][g][1]);
            }
        });
      });
    };

    // the next 64 tokens' loads go out before the current ones are used, but for wide heads, whose
    // second buffer does not fit the registers (64 rows x 8 heads of 256 23.7 us, with it 32.6)
    constexpr bool AHEAD = G <= 4;
    if (count > 0) {
      Chunk<G> x;
      load(0, id0, x);
      int id = id1;
      for (int i = 0; i < count; ++i) {
        const int after = fetch_id(i + 2);
        if constexpr (AHEAD) {
          Chunk<G> y;
          load(i + 1, id, y);
          consume(i == 0, x);
          x = y;
        } else {
          consume(i == 0, x);
          if (i + 1 < count) load(i + 1, id, x);
        }
        id = after;
      }
    }

    if (r0) __syncthreads();  // the previous rows' sums have been read
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      float *to = s_acc + (wave * QUADS + u) * 4 * DP;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          to[rg * DP + 32 * g + 16 * e + p16] = rows_scatter4(acc[u][g][e]);
#pragma unroll
      for (int r = 0; r < QR; ++r) {
        const float sum = group_sum<64>(l[u][r]) * (WEIGHT_FACTOR * CODE_FACTOR);
        if (lane == 0) {
          s_m[(wave * QUADS + u) * 4 + r] = m[u][r];
          s_l[(wave * QUADS + u) * 4 + r] = sum;
        }
      }
    }
    __syncthreads();
    const int rows = min(ROWS, nrows - r0);
    for (int i = threadIdx.x; i < rows * D; i += blockDim.x) {
      const int r = i / D, d = i % D;
      float M = NO_SCORE;
      for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w * 4 * QUADS + r]);
      float S = 0.f, o = 0.f;
      for (int w = 0; w < NW; ++w) {
        const float f = fast_exp2((s_m[w * 4 * QUADS + r] - M) * a.scale_log2);
        S = fmaf(s_l[w * 4 * QUADS + r], f, S);
        o = fmaf(s_acc[(w * 4 * QUADS + r) * DP + d], f, o);
      }
      const int64_t at = (row0 + r0 + r) * H + h;
      if (a.splits > 1) {
        a.part.acc[(at * a.splits + split) * D + d] = o;
        if (d == 0) a.part.ml[at * a.splits + split] = make_float2(M, S);
      } else {
        store_result<DT>((T *)a.out + at * D + d, S, o);
      }
    }
  }
}

// Waves of a workgroup and workgroups of a context.  A context is split where four parts or more
// fill eight waves a CU and leave each wave 128 tokens; more waves than that, or eight to a
// workgroup, were the slower ones (2 rows of 17001 and 39999 tokens x 8 heads of 128, us: workgroups
// of four waves, 4 / 8 / 12 / 16 a CU 18.9 / 17.8 / 19.4 / 20.5, of eight 25.2 / 19.4 / 22.5 / 21.6;
// one row of 40000 x 16 of 64 16.8 / 14.9 / 15.6 / 15.4).  What is not split takes eight waves where
// there is a workgroup a CU or fewer (eight / four: 16 rows of 2000 to 4000 tokens x 16 heads 14.7 /
// 17.6, of 400 to 1000 6.3 / 6.1, 32 x 8 heads of 256 15.5 / 16.4; 384 workgroups of 64 dims 8.3 / 8.0,
// 512 of 128 dims 15.9 / 12.9, of 256 dims 29.9 / 26.9, 1536 of 64 dims 18.6 / 14.9).
// A call's rows all take a place for each part, also those of no group: parts that would need more
// than 128 MB (the rows of a launch's own groups take 4.3 at most) are not made.
struct Attn4Plan {
  int waves, splits;
};

inline Attn4Plan attn4_plan(int64_t num_rows, int64_t num_groups, int H, int D,
                            int64_t max_tokens) {
  const int64_t wgs = num_groups * H;
  const int64_t fill = 256 * (D <= 256 ? 8 : 4) / (wgs * 4), most = max_tokens / (4 * 128);
  const int64_t room = MOST_WORKSPACE / H / split_part_bytes(D) / num_rows;
  const int64_t parts = std::min({fill, most, room});
  if (parts >= 4) return Attn4Plan{4, (int)parts};
  return Attn4Plan{D <= 256 && wgs <= 256 ? 8 : 4, 1};
}

template <int DT, int G, int ROWS>
void launch_attention_4bit(const Attn4Args &a, int waves, hipStream_t stream) {
  constexpr int QUADS = (ROWS + 3) / 4;
  const dim3 grid((unsigned)xcd_grid(a.num_groups * a.splits, a.H));
  const size_t lds = (size_t)waves * 4 * QUADS * (32 * G + 16 + 2) * 4;
  attention_4bit_kernel<DT, G, ROWS><<<grid, dim3(64 * waves), lds, stream>>>(a);
}

// Rows taken together: as many as the caller says that a group has, but four of wide heads (more
// read the pages again).
template <int DT, int G>
void launch_attention_4bit_rows(const Attn4Args &a, int rows, int waves, hipStream_t stream) {
  if (rows == 1) launch_attention_4bit<DT, G, 1>(a, waves, stream);
  else if (rows <= 4 || G > 4) launch_attention_4bit<DT, G, 4>(a, waves, stream);
  else if constexpr (G <= 4) launch_attention_4bit<DT, G, 8>(a, waves, stream);
}

template <int DT>
int launch_attention_4bit_groups(const Attn4Args &a, int rows, int waves, hipStream_t stream) {
  switch (e2m1_groups(a.D)) {
    case 1: launch_attention_4bit_rows<DT, 1>(a, rows, waves, stream); break;
    case 2: launch_attention_4bit_rows<DT, 2>(a, rows, waves, stream); break;
    case 3: launch_attention_4bit_rows<DT, 3>(a, rows, waves, stream); break;
    case 4: launch_attention_4bit_rows<DT, 4>(a, rows, waves, stream); break;
    case 5: launch_attention_4bit_rows<DT, 5>(a, rows, waves, stream); break;
    case 6: launch_attention_4bit_rows<DT, 6>(a, rows, waves, stream); break;
    case 7: launch_attention_4bit_rows<DT, 7>(a, rows, waves, stream); break;
    case 8: launch_attention_4bit_rows<DT, 8>(a, rows, waves, stream); break;
    default: launch_attention_4bit_rows<DT, 16>(a, rows, waves, stream); break;  // head size 512
  }
  const int st = launch_status("attention_with_kv_cache_4bit");
  if (st != VFL_OK || a.splits == 1) return st;
  launch_join_rows<DT>(a, stream);
  return launch_status("attention_with_kv_cache_4bit");
}

}  // namespace

}  // namespace vfl

using namespace vfl;

extern "C" int64_t vfl_attention_4bit_workspace(int64_t num_rows, int64_t num_groups,
                                                int num_heads, int head_dim, int block_size,
                                                int64_t max_blocks_per_seq) {
  if (num_rows <= 0 || num_groups <= 0 || num_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      max_blocks_per_seq <= 0)
    return 0;
  const Attn4Plan p =
      attn4_plan(num_rows, num_groups, num_heads, head_dim, max_blocks_per_seq * block_size);
  return p.splits > 1 ? num_rows * num_heads * p.splits * split_part_bytes(head_dim) : 0;
}

extern "C" int vfl_attention_with_kv_cache_4bit(
    const void *query, int64_t query_stride_token, int64_t query_stride_head, const void *cache,
    void *out, const int32_t *seq_lens, const int32_t *block_table, int64_t block_table_stride,
    int64_t max_blocks_per_seq, const int32_t *group_start, const int32_t *group_order,
    int64_t num_rows, int64_t num_groups, int max_group_size, int num_heads, int head_dim,
    int block_size, int64_t num_blocks, float scale, int dtype, void *workspace, void *stream) {
  clear_error();
  const char *who = "attention_with_kv_cache_4bit";
  const int st = check_4bit_cache(who, dtype, num_heads, head_dim, block_size, num_blocks);
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
  if (max_group_size < 1 || max_group_size > GROUP_ROWS) {
    set_error("%s: groups of up to %d rows (1 to %d)", who, max_group_size, GROUP_ROWS);
    return VFL_E_INVALID;
  }
  if (!(fabsf(scale) < INFINITY)) {
    set_error("%s: scale %f", who, (double)scale);
    return VFL_E_INVALID;
  }
  if (num_rows == 0 || num_groups == 0) return VFL_OK;
  if (!query || !out || !seq_lens || (max_blocks_per_seq && !block_table) ||
      (num_blocks && !cache)) {
    set_error("%s: null pointer argument", who);
    return VFL_E_INVALID;
  }
  const int eb = elem_bytes(dtype);
  if ((uintptr_t)cache % 16 || (uintptr_t)query % eb || (uintptr_t)out % eb ||
      (uintptr_t)workspace % 16) {
    set_error("%s: misaligned pointer (cache and workspace 16 bytes, others their element)", who);
    return VFL_E_INVALID;
  }
  // an empty pool holds nothing: every row is zero
  const int64_t table = num_blocks ? max_blocks_per_seq : 0;
  Attn4Args a;
  a.out = out;
  a.group_start = group_start, a.group_order = group_order;
  a.num_rows = num_rows, a.num_groups = num_groups;
  a.H = num_heads, a.D = head_dim;
  a.scale_log2 = decode_scale_log2(scale);
  a.splits = 1, a.part = {nullptr, nullptr};
  a.q = query, a.q_st = query_stride_token, a.q_sh = query_stride_head;
  a.cache = (const uint8_t *)cache;
  a.seq_lens = seq_lens, a.bt = block_table, a.bt_stride = block_table_stride;
  a.width = (int)table, a.room = (int)table * block_size;
  a.shift = block_shift(block_size);
  a.num_blocks = num_blocks;
  a.sign = scale < 0.f ? -1.f : 1.f;
  if (table == 0) a.bt = seq_lens, a.bt_stride = 0, a.width = 1;  // read, and not used
  const Attn4Plan plan = attn4_plan(num_rows, num_groups, num_heads, head_dim, table * block_size);
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
  const int rows = group_start ? max_group_size : 1;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == VFL_FLOAT32)
    return launch_attention_4bit_groups<VFL_FLOAT32>(a, rows, plan.waves, s);
  if (dtype == VFL_BFLOAT16)
    return launch_attention_4bit_groups<VFL_BFLOAT16>(a, rows, plan.waves, s);
  return launch_attention_4bit_groups<VFL_FLOAT16>(a, rows, plan.waves, s);
}
