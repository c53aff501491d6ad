// Paged decode attention over a cache held in e4m3 with a scale per (block, head) for K and
// one for V, gfx950:
//   out[r][h] = softmax_j(scale * ks_j <q[r][h], K8_j[h]>) (vs_j V8_j[h]),  j < seq_lens[r]
// with ks_j, vs_j the scales of token j's block.  The K scale multiplies a block's scores and
// the V scale its weights, so no element is dequantised in memory: e4m3 widens to 16 bits
// exactly (one conversion per pair) on its way into the matrix cores.
//
// The rows of a group (a request's beams over one page list) sit in the 16 columns of the
// tiles.  A wave takes 32 tokens at a time, two 16-token parts:
//   S[tok][row]  = K[tok][:] . q[row][:]     v_mfma_f32_16x16x32, the head's dims in an order
//                  that gives a lane 16 consecutive bytes of its token's row per 64 dims
//   online softmax per row over the 32 tokens, fp32
//   O^T[d][row] += V^T[d][tok] . P[tok][row] v_mfma_f32_16x16x32 over the 32 tokens: a lane's
//                  scores are already that product's operand, and V's token-interleaved
//                  layout gives a lane 4 dims x 4 tokens per 16 bytes
// Queries: 16-bit ones as they are; fp32 ones as three bf16 terms, which hold all 24 bits.
// Weights go through the second product in bf16 (whose range holds any scale) as a sum of
// two terms, 2^-17 relative, or three for fp32 outputs, 2^-25: below the output's rounding.
#include <stdio.h>

#include "e4m3.h"

namespace vfl {

// 16-bit type K is widened to, and terms of a query and of a weight
template <int DT> struct Terms {
  static constexpr int KT = DT == VFL_FLOAT16 ? VFL_FLOAT16 : VFL_BFLOAT16;
  static constexpr int Q = DT == VFL_FLOAT32 ? 3 : 1;
  static constexpr int P = DT == VFL_FLOAT32 ? 3 : 2;
};

using Bf16 = Mfma<VFL_BFLOAT16>;

// bf16 terms of four floats, largest first; f is left with the remainder.
__device__ __forceinline__ uint2 take_bf16(float (&f)[4]) {
  const uint2 w = make_uint2(Bf16::narrow2(f[0], f[1]), Bf16::narrow2(f[2], f[3]));
  f[0] -= Bf16::widen_lo(w.x), f[1] -= Bf16::widen_hi(w.x);
  f[2] -= Bf16::widen_lo(w.y), f[3] -= Bf16::widen_hi(w.y);
  return w;
}

// One lane's share of a 16-token part: per 64 dims, 16 dims of token l % 16 (K) and 4 dims x
// 4 tokens (V).
template <int NS> struct Part {
  uint4 k[NS], v[NS];
};

// NS: ceil(D / 64).  PARTS: 16-token parts of a block.  NW waves split a context.
template <int DT, int NS, int PARTS, int NW>
__global__ __launch_bounds__(64 * NW) void attention_8bit_kernel(
    const typename Elem<DT>::T *__restrict__ q, int64_t q_st, int64_t q_sh,
    const uint8_t *__restrict__ kc, const uint8_t *__restrict__ vc,
    const float *__restrict__ scales, typename Elem<DT>::T *__restrict__ out,
    const int32_t *__restrict__ seq_lens, const int32_t *__restrict__ bt, int64_t bt_stride,
    int max_blocks, const int32_t *__restrict__ group_start,
    const int32_t *__restrict__ group_order, int64_t num_rows, int64_t num_groups, int H, int D,
    int64_t num_blocks, float scale_log2) {
  using T = typename Elem<DT>::T;
  constexpr int KT = Terms<DT>::KT, QT = Terms<DT>::Q, PT = Terms<DT>::P;
  constexpr int COLS = 8;  // rows of a group
  constexpr int BPP = 2 / PARTS;  // blocks per 32 tokens
  __shared__ float s_acc[NW][64 * NS][COLS + 1];
  __shared__ float s_ml[NW][2][COLS];

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = lane & 15, rg = lane >> 4;
  int64_t pos;
  int h;
  xcd_position(blockIdx.x, (unsigned)H, pos, h);
  if (pos >= num_groups) return;
  int64_t g = pos;
  if (group_order) g = group_order[pos];
  if (g < 0 || g >= num_groups) return;
  int64_t row0 = g;
  int nrows = 1;
  if (group_start) {
    row0 = group_start[g];
    nrows = group_start[g + 1] - (int)row0;
  }
  if (row0 < 0 || row0 >= num_rows) return;
  nrows = (int)min((int64_t)min(nrows, COLS), num_rows - row0);
  if (nrows <= 0) return;

  const int64_t room = (int64_t)max_blocks * 16 * PARTS;  // tokens the table can list
  const int L = (int)min((int64_t)max(seq_lens[row0], 0), room);
  const int pairs = (L + 31) / 32;
  const int chunk = (pairs + NW - 1) / NW;
  const int p0 = min(pairs, wave * chunk), p1 = min(pairs, p0 + chunk);

  // Q operand: per 64 dims, dims 16 rg .. + 7 and + 8 .. + 15 of row `col`
  uint4 qop[NS][2][QT];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = 64 * s + 16 * rg + 8 * e;
      const bool in = col < nrows && d < D;
      const T *p = q + (row0 + col) * q_st + h * q_sh + d;
      if constexpr (DT != VFL_FLOAT32) {
        qop[s][e][0] = make_uint4(0, 0, 0, 0);
        if (in) qop[s][e][0] = load16_unaligned<DT>(p);
      } else {
        float f[2][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i / 4][i % 4] = in ? p[i] : 0.f;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const uint2 a = take_bf16(f[0]), b = take_bf16(f[1]);
          qop[s][e][t] = make_uint4(a.x, a.y, b.x, b.y);
        }
      }
    }

  floatx4_t acc[NS][4];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[s][c] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF_F, l = 0.f;

  const int32_t *table = bt + row0 * bt_stride;
  const int64_t block_bytes = (int64_t)H * 16 * PARTS * D;
  const int head_off = h * 16 * PARTS * D;
  for (int p = p0; p < p1; ++p) {
    Part<NS> part[2];
    bool ok[2];
    float ks[2], vs[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int b = p * BPP + u / PARTS;  // the part's block
      const int tok = 32 * p + 16 * u;    // its first token
      int id = -1;
      if (tok < L) id = table[b];
      ok[u] = id >= 0 && id < num_blocks;
      ks[u] = vs[u] = 0.f;
      if (ok[u]) {
        const float *sc = scales + 2 * ((int64_t)id * H + h);
        ks[u] = sc[0] * scale_log2, vs[u] = sc[1];
      }
      const int64_t base =
          (ok[u] ? (int64_t)id : 0) * block_bytes + head_off + (u % PARTS) * 16 * D;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        part[u].k[s] = part[u].v[s] = make_uint4(0, 0, 0, 0);
        if (ok[u] && 64 * s + 16 * rg < D && tok + col < L)
          part[u].k[s] = *reinterpret_cast<const uint4 *>(kc + base + col * D + 64 * s + 16 * rg);
        if (ok[u] && 64 * s + 4 * col < D && tok + 4 * rg < L)
          part[u].v[s] =
              *reinterpret_cast<const uint4 *>(vc + base + (rg * D + 64 * s + 4 * col) * 4);
      }
    }
    float sv[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      floatx4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const uint4 w = part[u].k[s];
        const uint2 a = e4m3_widen<KT>(w.x), b = e4m3_widen<KT>(w.y), c = e4m3_widen<KT>(w.z),
                    d = e4m3_widen<KT>(w.w);
#pragma unroll
        for (int t = QT - 1; t >= 0; --t) {
          x = Mfma<KT>::qk(make_uint4(a.x, a.y, b.x, b.y), qop[s][0][t], x);
          x = Mfma<KT>::qk(make_uint4(c.x, c.y, d.x, d.y), qop[s][1][t], x);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sv[u][j] = ok[u] && 32 * p + 16 * u + 4 * rg + j < L ? x[j] * ks[u] : NEG_INF_F;
    }
    float mb = NEG_INF_F;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) mb = fmaxf(mb, sv[u][j]);
    mb = rows_max4(mb);
    const bool need = mb > m + RESCALE_SLACK_LOG2;
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
      const float corr = need ? fast_exp2(m - mb) : 1.f;
      l *= corr;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[s][c] *= corr;
      m = need ? mb : m;
    }
    const float ms = m == NEG_INF_F ? 0.f : m;
    float w[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = fast_exp2(sv[u][j] - ms);
        l += e;
        w[u][j] = e * vs[u];
      }
    uint4 pop[PT];
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      const uint2 a = take_bf16(w[0]), b = take_bf16(w[1]);
      pop[t] = make_uint4(a.x, a.y, b.x, b.y);
    }
    // what lies behind the last token must not meet a zero weight (0 * NaN)
    if (32 * p + 32 > L) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int n = L - (32 * p + 16 * u + 4 * rg);  // tokens of the lane's four
        const uint32_t keep = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          uint4 &v = part[u].v[s];
          v = make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint2 a = e4m3_widen<VFL_BFLOAT16>((&part[0].v[s].x)[c]);
        const uint2 b = e4m3_widen<VFL_BFLOAT16>((&part[1].v[s].x)[c]);
#pragma unroll
        for (int t = PT - 1; t >= 0; --t)
          acc[s][c] = Bf16::qk(make_uint4(a.x, a.y, b.x, b.y), pop[t], acc[s][c]);
      }
  }
  l = rows_sum4(l);

  // acc[s][c][j]: dim 64 s + 16 rg + 4 j + c of row `col`
  if (col < COLS) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s_acc[wave][64 * s + 16 * rg + 4 * j + c][col] = acc[s][c][j];
    if (rg == 0) s_ml[wave][0][col] = m, s_ml[wave][1][col] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * D; i += 64 * NW) {
    const int r = i / D, d = i % D;
    float M = NEG_INF_F;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_ml[w][0][r]);
    const float Ms = M == NEG_INF_F ? 0.f : M;
    float S = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = fast_exp2(s_ml[w][0][r] - Ms);
      S = fmaf(s_ml[w][1][r], f, S);
      o = fmaf(s_acc[w][d][r], f, o);
    }
    const float y = S > 0.f ? o / S : S == S ? 0.f : S;  // NaN scores stay NaN
    if constexpr (DT == VFL_FLOAT32) out[((row0 + r) * H + h) * D + d] = y;
    else out[((row0 + r) * H + h) * D + d] = (T)Mfma<DT>::narrow(y);
  }
}

struct Attn8Args {
  const void *q;
  int64_t q_st, q_sh;
  const uint8_t *kc, *vc;
  const float *scales;
  void *out;
  const int32_t *seq_lens, *bt;
  int64_t bt_stride;
  int max_blocks;
  const int32_t *group_start, *group_order;
  int64_t num_rows, num_groups;
  int H, D;
  int64_t num_blocks;
  float scale_log2;
};

template <int DT, int NS, int PARTS>
static void launch_attention_8bit(const Attn8Args &a, hipStream_t stream) {
  using T = typename Elem<DT>::T;
  constexpr int NW = NS >= 8 ? 2 : NS >= 4 ? 4 : 4;
  attention_8bit_kernel<DT, NS, PARTS, NW>
      <<<dim3((unsigned)xcd_grid(a.num_groups, a.H)), dim3(64 * NW), 0, stream>>>(
          (const T *)a.q, a.q_st, a.q_sh, a.kc, a.vc, a.scales, (T *)a.out, a.seq_lens, a.bt,
          a.bt_stride, a.max_blocks, a.group_start, a.group_order, a.num_rows, a.num_groups, a.H,
          a.D, a.num_blocks, a.scale_log2);
}

template <int DT, int PARTS>
static int launch_attention_8bit_steps(const Attn8Args &a, hipStream_t stream) {
  switch ((a.D + 63) / 64) {
    case 1: launch_attention_8bit<DT, 1, PARTS>(a, stream); break;
    case 2: launch_attention_8bit<DT, 2, PARTS>(a, stream); break;
    case 3: launch_attention_8bit<DT, 3, PARTS>(a, stream); break;
    case 4: launch_attention_8bit<DT, 4, PARTS>(a, stream); break;
    default: launch_attention_8bit<DT, 8, PARTS>(a, stream); break;  // head size 512
  }
  return launch_status("attention_with_kv_cache_8bit");
}

}  // namespace vfl

using namespace vfl;

extern "C" int vfl_attention_with_kv_cache_8bit(
    const void *query, int64_t query_stride_token, int64_t query_stride_head, const void *k_cache,
    const void *v_cache, const float *kv_scales, void *out, const int32_t *seq_lens,
    const int32_t *block_table, int64_t block_table_stride, int64_t max_blocks_per_seq,
    const int32_t *group_start, const int32_t *group_order, int64_t num_rows, int64_t num_groups,
    int num_heads, int head_dim, int block_size, int64_t num_blocks, float scale, int dtype,
    void *stream) {
  clear_error();
  const char *who = "attention_with_kv_cache_8bit";
  const int st = check_8bit_cache(who, dtype, num_heads, head_dim, block_size, num_blocks);
  if (st != VFL_OK) return st;
  if (num_rows < 0 || num_groups < 0 || num_groups > num_rows ||
      (!group_start && num_groups != num_rows) || max_blocks_per_seq < 0 ||
      max_blocks_per_seq * block_size > 2147483647LL - 64 ||
      block_table_stride < max_blocks_per_seq ||
      (num_groups + XCDS) * (int64_t)num_heads > 2147483647LL) {
    set_error("%s: bad sizes (rows %lld groups %lld table %lld wide, stride %lld)", who,
              (long long)num_rows, (long long)num_groups, (long long)max_blocks_per_seq,
              (long long)block_table_stride);
    return VFL_E_INVALID;
  }
  if (num_rows == 0 || num_groups == 0) return VFL_OK;
  if (!query || !out || !seq_lens || (max_blocks_per_seq && !block_table) ||
      (num_blocks && (!k_cache || !v_cache || !kv_scales))) {
    set_error("%s: null pointer argument", who);
    return VFL_E_INVALID;
  }
  const int eb = elem_bytes(dtype);
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)kv_scales % 4 ||
      (uintptr_t)query % eb || (uintptr_t)out % eb) {
    set_error("%s: misaligned pointer (caches 16 bytes, others their element)", who);
    return VFL_E_INVALID;
  }
  const Attn8Args a{query, query_stride_token, query_stride_head, (const uint8_t *)k_cache,
                    (const uint8_t *)v_cache, kv_scales, out, seq_lens, block_table,
                    block_table_stride, (int)max_blocks_per_seq, group_start, group_order,
                    num_rows, num_groups, num_heads, head_dim, num_blocks,
                    scale * 1.4426950408889634f};
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return block_size == 16 ? launch_attention_8bit_steps<DT, 1>(a, s)
                            : launch_attention_8bit_steps<DT, 2>(a, s);
  };
  if (dtype == VFL_FLOAT32) return go(std::integral_constant<int, VFL_FLOAT32>{});
  if (dtype == VFL_BFLOAT16) return go(std::integral_constant<int, VFL_BFLOAT16>{});
  return go(std::integral_constant<int, VFL_FLOAT16>{});
}
