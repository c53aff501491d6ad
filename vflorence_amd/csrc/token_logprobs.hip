// Log probabilities of given tokens, each row's entropy and its best alternatives (gfx950).
// Per row x of the logits, with m = max x:
//   S = sum exp(x - m),  W = sum (x - m) exp(x - m)
//   logprob(t) = (x_t - m) - log S,   entropy = -sum p log p = log S - W / S
// and the k best (value, id), best first, equal values by the lower id, with their logprobs.
// Sums and statistics are fp32.  A value of -inf has weight 0 and adds nothing to W.  A row
// that holds a NaN or +inf, or nothing above -inf, has no distribution: its figures are NaN,
// its alternatives' ids -1.
#include <math.h>
#include <stdio.h>

#include "common.h"
#include "mfma_ops.h"

namespace vfl {

constexpr int TLP_MAX_K = 20;
constexpr int TLP_MAX_VOCAB = 1 << 20;
constexpr int TLP_CAP = 512;        // candidates for the alternatives kept in LDS
constexpr int TLP_MAX_SEGMENTS = 64;
constexpr float TLP_FLOOR = -1e4f;  // exp() is 0 long before

template <int DT> __device__ __forceinline__ float logit(typename Elem<DT>::T v) {
  if constexpr (DT == VFL_FLOAT32) return v;
  else return Mfma<DT>::widen(v);
}
// Element j of a 16-byte vector (j a constant after unrolling).
template <int DT> __device__ __forceinline__ float logit_of(const uint4 &u, int j) {
  if constexpr (DT == VFL_FLOAT32) return __uint_as_float((&u.x)[j]);
  else return j % 2 ? Mfma<DT>::widen_hi((&u.x)[j / 2]) : Mfma<DT>::widen_lo((&u.x)[j / 2]);
}

template <int DT> __device__ __forceinline__ float vector_max(const uint4 &u) {
  float v = logit_of<DT>(u, 0);
#pragma unroll
  for (int j = 1; j < Elem<DT>::VEC; ++j) v = fmaxf(v, logit_of<DT>(u, j));
  return v;
}

// Keeps the compiler from holding a vector's widened elements in registers from one pass over
// it to the next (57 to 69 of them spilled).
__device__ __forceinline__ void opaque(uint4 &u) {
  asm volatile("" : "+v"(u.x), "+v"(u.y), "+v"(u.z), "+v"(u.w));
}

// (value, id) order: higher value first, then lower id.
__device__ __forceinline__ bool ahead(float a, int ia, float b, int ib) {
  return a > b || (a == b && ia < ib);
}

// One segment's statistics, kept for the join.
struct Partial {
  float m, s, w, unused;
};

// Where a workgroup's results go: a row's final figures, or a segment's for the join.
struct LogprobOut {
  const int64_t *tokens;
  int num_tokens, k;
  float *logprobs, *entropy, *top;
  int64_t *ids;
  Partial *part;    // [rows][segments]
  float *cand;      // [rows][segments][k]
  int32_t *cand_id;
};

// A row, or with SPLIT one segment of it, lives in the registers of NT threads, NV vectors
// of 16 bytes each, read once.
//
// The alternatives: the k-th largest of the maxima of 64 groups of threads, tau, bounds the
// k-th value from below (k groups hold a value >= tau); every value >= tau (24 of a random
// row at k = 20) goes to LDS, and its rank is the number of candidates ahead of it.  Rows
// without a bound (fewer than k groups hold a value above -inf) or with more than TLP_CAP
// candidates (ties) pick the next best k times, reading the row again.
template <int DT, int NT, int NV, int OCC, bool SPLIT>
__global__ __launch_bounds__(NT, OCC) void token_logprobs_kernel(
    const typename Elem<DT>::T *__restrict__ logits, int64_t stride, int vocab, int segment,
    LogprobOut o) {
  using T = typename Elem<DT>::T;
  constexpr int NWAVE = NT / 64, VE = Elem<DT>::VEC;
  constexpr int GL = NT / 64;  // lanes of a group
  __shared__ float s_group[64], s_cv[TLP_CAP], s_red[2][NWAVE], s_tau, s_bv[NWAVE];
  __shared__ int s_ci[TLP_CAP], s_count, s_bi[NWAVE];

  const int64_t row = blockIdx.x;
  const int base = SPLIT ? blockIdx.y * segment : 0;  // first id
  const int n = SPLIT ? min(segment, vocab - base) : vocab;
  const T *x = logits + row * stride + base;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int k = o.k;

  // whole 16-byte vectors from the first aligned address, and one scalar per thread of the
  // few values before (threads 0..) and after them (threads 8..); absent values are -inf
  const int head = min(n, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
  const int nvec = (n - head) / VE;
  const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
  constexpr uint32_t NI = DT == VFL_FLOAT32    ? 0xff800000u
                          : DT == VFL_BFLOAT16 ? 0xff80ff80u
                                               : 0xfc00fc00u;
  uint4 u[NV];
#pragma unroll
  for (int r = 0; r < NV; ++r) {
    u[r] = make_uint4(NI, NI, NI, NI);
    if (tid + r * NT < nvec) u[r] = xv[tid + r * NT];
  }
  int xi = -1;  // the scalar's place
  if (tid < head) xi = tid;
  else if (tid >= 8 && head + nvec * VE + tid - 8 < n) xi = head + nvec * VE + tid - 8;
  const float xs = xi >= 0 ? logit<DT>(x[xi]) : NEG_INF_F;
  // the row's first given tokens, on their way during the rest
  float given = 0.f;
  bool inside = false;
  if constexpr (!SPLIT) {
    if (tid < o.num_tokens) {
      const int64_t t = o.tokens[row * o.num_tokens + tid];
      inside = t >= 0 && t < vocab;
      if (inside) given = logit<DT>(x[t]);
    }
  }
  if (tid == 0) s_count = 0;

  float tmax = fmaxf(NEG_INF_F, xs);  // (a NaN bounds nothing)
#pragma unroll
  for (int r = 0; r < NV; ++r)
    if (r * NT < nvec) tmax = fmaxf(tmax, vector_max<DT>(u[r]));  // workgroup-uniform
  float g = tmax;
  if constexpr (GL >= 4) {
    g = fmaxf(g, dpp<DPP_QUAD_XOR1>(g));
    g = fmaxf(g, dpp<DPP_QUAD_XOR2>(g));
  }
  if constexpr (GL >= 16) {
    g = fmaxf(g, dpp<DPP_ROW_HALF_MIRROR>(g));
    g = fmaxf(g, dpp<DPP_ROW_MIRROR>(g));
  }
  if (tid % GL == 0) s_group[tid / GL] = g;
  __syncthreads();
  g = s_group[lane];
  const float mx = wave_max64(g);
  if (wave == 0 && k > 0) {
    float tau = mx;
    if (k > 1) {
      int rank = 0;
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        const float og = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), j));
        rank += og > g || (og == g && j < lane);
      }
      const uint64_t at = __builtin_amdgcn_ballot_w64(rank == k - 1);
      tau = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), __builtin_ctzll(at)));
    }
    if (lane == 0) s_tau = tau;
  }

  // S and W.  t = x - max first, then its product with log2 e: one fused step would round
  // max * log2 e, an error common to every term.  exp(-inf) = 0 must not meet its -inf.
  constexpr float LOG2E_F = 1.4426950408889634f;
  const float ref = mx == NEG_INF_F ? 0.f : mx;
  float s4[4] = {0.f, 0.f, 0.f, 0.f}, w4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < NV; ++r) {
    if (r * NT >= nvec) continue;
    opaque(u[r]);
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float t = logit_of<DT>(u[r], j) - ref, e = fast_exp2(t * LOG2E_F);
      s4[j % 4] += e;
      w4[j % 4] = fmaf(fmaxf(t, TLP_FLOOR), e, w4[j % 4]);
    }
  }
  {
    const float t = xs - ref, e = fast_exp2(t * LOG2E_F);
    s4[0] += e;
    w4[0] = fmaf(fmaxf(t, TLP_FLOOR), e, w4[0]);
  }
  const float ws = group_sum<64>((s4[0] + s4[1]) + (s4[2] + s4[3]));
  const float ww = group_sum<64>((w4[0] + w4[1]) + (w4[2] + w4[3]));
  if (lane == 0) s_red[0][wave] = ws, s_red[1][wave] = ww;
  __syncthreads();
  float S = 0.f, W = 0.f;
#pragma unroll
  for (int w = 0; w < NWAVE; ++w) S += s_red[0][w], W += s_red[1][w];
  // a NaN, +inf or an empty row leaves S NaN or 0
  const bool bad = !SPLIT && !(S > 0.f);
  const float log_s = SPLIT ? 0.f : logf(S);
  const int64_t seg = SPLIT ? row * gridDim.y + blockIdx.y : row;
  if constexpr (SPLIT) {
    if (tid == 0) o.part[seg] = Partial{mx, S, W, 0.f};
  } else {
    if (tid == 0) o.entropy[row] = bad ? NAN : log_s - W / S;
    for (int i = tid; i < o.num_tokens; i += NT) {
      if (i != tid) {
        const int64_t t = o.tokens[row * o.num_tokens + i];
        inside = t >= 0 && t < vocab;
        if (inside) given = logit<DT>(x[t]);
      }
      o.logprobs[row * o.num_tokens + i] = bad || !inside ? NAN : (given - mx) - log_s;
    }
  }
  if (k == 0) return;

  auto put = [&](int rank, float v, int id) {
    if constexpr (SPLIT) {
      o.cand[seg * k + rank] = v;
      o.cand_id[seg * k + rank] = id;
    } else {
      o.top[row * k + rank] = bad ? NAN : (v - mx) - log_s;
      o.ids[row * k + rank] = bad ? -1 : id;
    }
  };
  const float tau = s_tau;
  const bool bounded = tau != NEG_INF_F;
  if (bounded && tmax >= tau) {
    auto keep = [&](float v, int i) {
      if (v >= tau) {
        const int slot = atomicAdd(&s_count, 1);
        if (slot < TLP_CAP) s_cv[slot] = v, s_ci[slot] = base + i;
      }
    };
    if (xi >= 0) keep(xs, xi);
#pragma unroll
    for (int r = 0; r < NV; ++r) {
      opaque(u[r]);
      if (r * NT >= nvec || !(vector_max<DT>(u[r]) >= tau)) continue;
#pragma unroll
      for (int j = 0; j < VE; ++j) keep(logit_of<DT>(u[r], j), head + (tid + r * NT) * VE + j);
    }
  }
  __syncthreads();
  const int count = s_count;
  if (bounded && count <= TLP_CAP) {
    for (int c = tid; c < count; c += NT) {
      const float v = s_cv[c];
      const int id = s_ci[c];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += ahead(s_cv[j], s_ci[j], v, id);
      if (rank < k) put(rank, v, id);
    }
    return;
  }
  float last = INFINITY;
  int last_id = -1;
  for (int r = 0; r < k; ++r) {
    float bv = NEG_INF_F;
    int bi = INT32_MAX;
#pragma nounroll
    for (int i = tid; i < n; i += NT) {
      const float v = logit<DT>(x[i]);
      if (ahead(last, last_id, v, base + i) && ahead(v, base + i, bv, bi)) bv = v, bi = base + i;
    }
    for (int d = 1; d < 64; d *= 2) {
      const float ov = __shfl_xor(bv, d);
      const int oi = __shfl_xor(bi, d);
      if (ahead(ov, oi, bv, bi)) bv = ov, bi = oi;
    }
    __syncthreads();  // the previous round's best have been read
    if (lane == 0) s_bv[wave] = bv, s_bi[wave] = bi;
    __syncthreads();
    for (int w = 0; w < NWAVE; ++w)
      if (ahead(s_bv[w], s_bi[w], bv, bi)) bv = s_bv[w], bi = s_bi[w];
    last = bv, last_id = bi;
    if (tid == 0) put(r, bv, bi);
  }
}

// A row's segments joined: their sums rescaled to the common maximum, and the best of their
// best by rank.
constexpr int TLP_JOIN_NT = 256;
template <int DT>
__global__ __launch_bounds__(TLP_JOIN_NT) void token_logprobs_join_kernel(
    const typename Elem<DT>::T *__restrict__ logits, int64_t stride, int vocab, int segments,
    LogprobOut o) {
  __shared__ float s_cv[TLP_MAX_SEGMENTS * TLP_MAX_K];
  __shared__ int s_ci[TLP_MAX_SEGMENTS * TLP_MAX_K];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, k = o.k, count = segments * k;
  for (int i = tid; i < count; i += TLP_JOIN_NT)
    s_cv[i] = o.cand[row * count + i], s_ci[i] = o.cand_id[row * count + i];
  Partial p{NEG_INF_F, 0.f, 0.f, 0.f};
  if (lane < segments) p = o.part[row * segments + lane];
  const float mx = wave_max64(p.m);
  // W about the common maximum: sum (x - M) e = f (W + (m - M) S).  A segment of weight 0 adds
  // nothing (0 times an m - M past fp32's range), but hands on its NaN.
  const float dm = p.m - mx, f = p.m == NEG_INF_F ? 0.f : expf(dm);
  const float S = group_sum<64>(p.m == NEG_INF_F ? p.s : f * p.s);
  const float W = group_sum<64>(f == 0.f ? 0.f : f * (p.w + dm * p.s));
  const bool bad = !(S > 0.f);
  const float log_s = logf(S);
  if (tid == 0) o.entropy[row] = bad ? NAN : log_s - W / S;
  const typename Elem<DT>::T *x = logits + row * stride;
  for (int i = tid; i < o.num_tokens; i += TLP_JOIN_NT) {
    const int64_t t = o.tokens[row * o.num_tokens + i];
    o.logprobs[row * o.num_tokens + i] =
        bad || t < 0 || t >= vocab ? NAN : (logit<DT>(x[t]) - mx) - log_s;
  }
  __syncthreads();
  for (int c = tid; c < count; c += TLP_JOIN_NT) {
    const float v = s_cv[c];
    const int id = s_ci[c];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += ahead(s_cv[j], s_ci[j], v, id);
    if (rank < k) {
      o.top[row * k + rank] = bad ? NAN : (v - mx) - log_s;
      o.ids[row * k + rank] = bad ? -1 : id;
    }
  }
}

// Values that a workgroup of 1024 threads holds, and so the longest row of one launch.
constexpr int tlp_capacity(int dtype) { return dtype == VFL_FLOAT32 ? 1024 * 14 * 4 : 1024 * 8 * 8; }
constexpr int TLP_SEGMENT_BYTES = 1024 * 8 * 16;

// Segments of a row that does not fit (0: it does), of equal length, a multiple of 8.
inline int tlp_segments(int vocab, int dtype, int *segment) {
  if (vocab <= tlp_capacity(dtype)) return 0;
  const int most = TLP_SEGMENT_BYTES / elem_bytes(dtype);
  const int parts = (vocab + most - 1) / most;
  *segment = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  return (vocab + *segment - 1) / *segment;
}

template <int DT>
static int launch_token_logprobs(const void *logits, int64_t stride, int64_t rows, int vocab,
                                 LogprobOut o, void *workspace, hipStream_t s) {
  using T = typename Elem<DT>::T;
  const T *x = (const T *)logits;
  constexpr int VE = Elem<DT>::VEC;
  int segment = 0;
  const int segments = tlp_segments(vocab, DT, &segment);
  if (segments) {
    o.part = (Partial *)workspace;
    o.cand = (float *)(o.part + rows * segments);
    o.cand_id = (int32_t *)(o.cand + rows * segments * o.k);
    token_logprobs_kernel<DT, 1024, 8, 8, true>
        <<<dim3((unsigned)rows, (unsigned)segments), dim3(1024), 0, s>>>(x, stride, vocab, segment,
                                                                         o);
    const int st = launch_status("token_logprobs");
    if (st != VFL_OK) return st;
    token_logprobs_join_kernel<DT><<<dim3((unsigned)rows), dim3(TLP_JOIN_NT), 0, s>>>(
        x, stride, vocab, segments, o);
    return launch_status("token_logprobs");
  }
#define VFL_TLP(NT, NV, OCC)                                                       \
  token_logprobs_kernel<DT, NT, NV, OCC, false><<<dim3((unsigned)rows), dim3(NT), 0, s>>>( \
      x, stride, vocab, 0, o)
  if (vocab <= 64 * 8 * VE) VFL_TLP(64, 8, 8);
  else if (vocab <= 256 * 8 * VE) VFL_TLP(256, 8, 8);
  else if (vocab <= 1024 * 8 * VE) VFL_TLP(1024, 8, 8);
  else if constexpr (DT == VFL_FLOAT32) VFL_TLP(1024, 14, 4);
#undef VFL_TLP
  return launch_status("token_logprobs");
}

}  // namespace vfl

using namespace vfl;

extern "C" int64_t vfl_token_logprobs_workspace(int vocab, int dtype, int k) {
  if (vocab <= 0 || vocab > TLP_MAX_VOCAB || k < 0 || k > TLP_MAX_K) return 0;
  int segment = 0;
  return (int64_t)tlp_segments(vocab, dtype, &segment) * (int64_t)(sizeof(Partial) + 8 * k);
}

extern "C" int vfl_token_logprobs(const void *logits, int64_t row_stride, int64_t rows, int vocab,
                                  int dtype, const int64_t *tokens, int num_tokens, int k,
                                  float *logprobs, float *entropy, float *top_logprobs,
                                  int64_t *top_ids, void *workspace, void *stream) {
  clear_error();
  if (dtype != VFL_FLOAT32 && dtype != VFL_BFLOAT16 && dtype != VFL_FLOAT16) {
    set_error("token_logprobs: unsupported dtype code %d", dtype);
    return VFL_E_INVALID;
  }
  if (rows < 0 || rows > 2147483647LL || vocab <= 0 || vocab > TLP_MAX_VOCAB ||
      row_stride < vocab || k < 0 || k > TLP_MAX_K || k > vocab || num_tokens < 0) {
    set_error("token_logprobs: need 0 <= k <= min(%d, vocab), vocab up to %d and row_stride >= "
              "vocab (k %d, vocab %d, stride %lld, rows %lld)",
              TLP_MAX_K, TLP_MAX_VOCAB, k, vocab, (long long)row_stride, (long long)rows);
    return VFL_E_INVALID;
  }
  if (rows == 0) return VFL_OK;
  if (!logits || !entropy || (num_tokens && (!tokens || !logprobs)) ||
      (k && (!top_logprobs || !top_ids)) ||
      (!workspace && vfl_token_logprobs_workspace(vocab, dtype, k))) {
    set_error("token_logprobs: null pointer argument");
    return VFL_E_INVALID;
  }
  if ((uintptr_t)logits % elem_bytes(dtype) || (uintptr_t)workspace % 16) {
    set_error("token_logprobs: logits not aligned to their element, or workspace to 16 bytes");
    return VFL_E_INVALID;
  }
  hipStream_t s = (hipStream_t)stream;
  const LogprobOut o{tokens, num_tokens, k, logprobs, entropy, top_logprobs, top_ids,
                     nullptr, nullptr, nullptr};
  if (dtype == VFL_FLOAT32)
    return launch_token_logprobs<VFL_FLOAT32>(logits, row_stride, rows, vocab, o, workspace, s);
  if (dtype == VFL_BFLOAT16)
    return launch_token_logprobs<VFL_BFLOAT16>(logits, row_stride, rows, vocab, o, workspace, s);
  return launch_token_logprobs<VFL_FLOAT16>(logits, row_stride, rows, vocab, o, workspace, s);
}
