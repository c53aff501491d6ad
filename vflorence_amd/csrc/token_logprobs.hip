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

#include "e4m3.h"

namespace vfl {

constexpr int TLP_MAX_K = 20;
constexpr int TLP_MAX_VOCAB = 1 << 20;
constexpr int TLP_CAP = 512;        // candidates for the alternatives kept in LDS
constexpr int TLP_MAX_SEGMENTS = 64;
constexpr float TLP_FLOOR = -1e4f;  // exp2() is 0 long before
// A thread's reference is max * log2 e, rounded: every term carries that rounding, 2^-8 at most up
// to this maximum, and the step to differences from the maximum itself takes it off again.  Rows
// (or segments) whose maximum lies further from 0 would carry more, exp2's whole range from
// 2^32 on: they are summed in a second read, from the differences.
constexpr float TLP_FAR = 65536.f;
constexpr float TLP_NONE = -1e5f;  // a thread's first reference: below every such maximum's
// log2 units a reference may lag behind.  A thread's terms are up to 2^16, its sum of up to 57
// below 2^22; about the maximum a row's 2^20 terms sum to 2^20 at most.
constexpr float TLP_SLACK = 16.f;
constexpr float LOG2E_F = 1.4426950408889634f, LN2_F = 0.6931471805599453f;

// A thread's sums of exp2(x log2 e - c) and of its product with the exponent.
struct Sums {
  float c, s, w;

  // Move the reference to `to` (or stay, where to == c).
  __device__ __forceinline__ void move(float to) {
    const float d = c - to, f = d == 0.f ? 1.f : fast_exp2(d);
    w = f == 0.f ? 0.f : f * (w + d * s);
    s *= f;
    c = to;
  }
};

// The same of exp2((x - r) log2 e), r a value no less than any of the x.
struct Stats {
  float r, s, w;

  // A thread's sums about r: divided by the term that r has in them (or would have), so that
  // its own term becomes 1.
  __device__ __forceinline__ Stats(const Sums &a, float r) : r(r), s(a.s), w(a.w) {
    if (s == 0.f) return;  // (no value: the reference is none)
    const float t = fmaf(r, LOG2E_F, -a.c), e = fast_exp2(t);
    w = e < INFINITY ? fmaf(-t, s, w) / e : 0.f;
    s /= e;
  }
  __device__ __forceinline__ Stats(float r, float s, float w) : r(r), s(s), w(w) {}

  __device__ __forceinline__ void move(float to) {
    if (s == 0.f) return;  // (nothing: r may be -inf)
    const float d = (r - to) * LOG2E_F, f = fast_exp2(d);
    w = f == 0.f ? 0.f : f * fmaf(d, s, w);
    s *= f;
    r = to;
  }
};

// Sum over the wave, the first lane's for every lane: a product before the first addition is
// fused into it, which then rounds differently on the two lanes of a pair.
__device__ __forceinline__ float wave_total(float x) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(group_sum<64>(x))));
}

// A row's normaliser, about its maximum, and what it makes of a value.
struct Normaliser {
  float mx, log2_s;

  __device__ __forceinline__ float logprob(float x) const {
    return fmaf(-LN2_F, log2_s, x - mx);
  }
};

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

// Whether an element of the vector may reach tau (a NaN may seem to).  16-bit patterns order
// like their values where they are positive, and against it where negative: packed maxima
// of signed, or minima of unsigned patterns (which take 0 as -0), instead of eight widened
// elements.
template <int DT> __device__ __forceinline__ bool may_reach(const uint4 &u, float tau) {
  if constexpr (DT == VFL_FLOAT32) {
    return vector_max<DT>(u) >= tau;
  } else {
    typedef short s2_t __attribute__((ext_vector_type(2)));
    typedef unsigned short u2_t __attribute__((ext_vector_type(2)));
    const uint32_t bits = Mfma<DT>::narrow(tau == 0.f ? -0.f : tau);
    if (tau > 0.f) {
      const s2_t m = __builtin_elementwise_max(
          __builtin_elementwise_max(__builtin_bit_cast(s2_t, u.x), __builtin_bit_cast(s2_t, u.y)),
          __builtin_elementwise_max(__builtin_bit_cast(s2_t, u.z), __builtin_bit_cast(s2_t, u.w)));
      return max(m.x, m.y) >= (short)bits;
    }
    const u2_t m = __builtin_elementwise_min(
        __builtin_elementwise_min(__builtin_bit_cast(u2_t, u.x), __builtin_bit_cast(u2_t, u.y)),
        __builtin_elementwise_min(__builtin_bit_cast(u2_t, u.z), __builtin_bit_cast(u2_t, u.w)));
    return min(m.x, m.y) <= (unsigned short)bits;
  }
}

// The k best of `count` candidates in LDS: a wave takes every waves-th one and counts those
// ahead of it, 64 at a time.  put(rank, value, id) runs on one lane.
template <typename F>
__device__ __forceinline__ void rank_candidates(const float *cv, const int *ci, int count,
                                                int wave, int waves, int k, F &&put) {
  const int lane = __lane_id();
  for (int c = wave; c < count; c += waves) {
    const float v = cv[c];
    const int id = ci[c];
    int rank = 0;
    for (int j = 0; j < count; j += 64) {
      const bool over = j + lane < count && ahead(cv[j + lane], ci[j + lane], v, id);
      rank += __builtin_popcountll(__builtin_amdgcn_ballot_w64(over));
    }
    if (lane == 0 && rank < k) put(rank, v, id);
  }
}

// One segment's maximum and sums about it, kept for the join.
struct alignas(16) Partial {
  float mx, s, w;
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
// What bounds it: many rows the vector work, 17 operations a value with k = 5 (one of them
// the exponential, at a quarter of their rate), two workgroups of 64 VGPRs a CU overlapping
// it with the other's loads; few rows their own chain of loads,
// exponentials and picks.  Device time, us: 4096 x 50265 bf16 k = 5 92 (4.5 TB/s), k = 0 81
// (5.1); 256 x 50265 k = 0 8.2; 4 x 51289 k = 8 8.5; 93 x 51289 fp32 k = 20 10.6.  What
// the steps gave (the same cases): loads that no condition holds back 106 -> 93, 10.4 ->
// 8.5; ranks by ballot and packed compares for the alternatives k = 8 10.0 -> 8.5, k = 20
// 13.1 -> 10.7.
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
  __shared__ float s_group[64], s_cv[TLP_CAP], s_red[3][NWAVE], s_tau, s_bv[NWAVE];
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
  const __amdgpu_buffer_rsrc_t xv =
      __builtin_amdgcn_make_buffer_rsrc((void *)(x + head), 0, nvec * 16, 0x00020000);
  constexpr uint32_t NI = DT == VFL_FLOAT32    ? 0xff800000u
                          : DT == VFL_BFLOAT16 ? 0xff80ff80u
                                               : 0xfc00fc00u;
  // No load under a condition, whose branch would wait for it before the next one goes out:
  // buffer loads return 0 past the row's last vector.  The given token of this thread first:
  // its logit follows while the row is on its way.
  int64_t token = 0;
  if constexpr (!SPLIT) {
    if (o.num_tokens > 0) token = o.tokens[row * o.num_tokens + min(tid, o.num_tokens - 1)];
  }
  uint4 u[NV];
#pragma unroll
  for (int r = 0; r < NV; ++r)
    u[r] = __builtin_bit_cast(
        uint4, __builtin_amdgcn_raw_buffer_load_b128(xv, (tid + r * NT) * 16, 0, 0));
  int xi = -1;  // the scalar's place
  if (tid < head) xi = tid;
  else if (tid >= 8 && head + nvec * VE + tid - 8 < n) xi = head + nvec * VE + tid - 8;
  const T xraw = x[max(xi, 0)];
  bool inside = token >= 0 && token < vocab;
  T graw = 0;
  if constexpr (!SPLIT) graw = x[inside ? token : 0];
  if (tid == 0) s_count = 0, s_tau = NEG_INF_F;

  // Each thread's sums about a reference of its own, moved only when a vector's maximum
  // exceeds it by TLP_SLACK, so that the first vectors are summed while the last ones
  // are on their way.
  Sums sums{TLP_NONE, 0.f, 0.f};
  float tmax = NEG_INF_F;  // (a NaN bounds nothing)
  auto refer = [&](float v) {  // v: the maximum of what comes next
    tmax = fmaxf(tmax, v);
    const float to = v * LOG2E_F;
    const bool need = to > sums.c + TLP_SLACK;
    if (__builtin_amdgcn_ballot_w64(need) != 0) sums.move(need ? to : sums.c);
  };
  auto add = [&](float v, float &s, float &w) {
    // one fused step: what c lost in rounding every term carries alike.  exp2(-inf) = 0 must
    // not meet its -inf.
    const float t = fmaf(v, LOG2E_F, -sums.c), e = fast_exp2(t);
    s += e;
    w = fmaf(fmaxf(t, TLP_FLOOR), e, w);
  };
#pragma unroll
  for (int r = 0; r < NV; ++r) {
    if (r * NT >= nvec) continue;  // workgroup-uniform
    if (__builtin_expect(r * NT + NT > nvec, 0)) {
      if (tid + r * NT >= nvec) u[r] = make_uint4(NI, NI, NI, NI);
      opaque(u[r]);
    }
    refer(vector_max<DT>(u[r]));
    float s2 = 0.f, w2 = 0.f;
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
      add(logit_of<DT>(u[r], j), sums.s, sums.w);
      add(logit_of<DT>(u[r], j + 1), s2, w2);
    }
    sums.s += s2, sums.w += w2;
    opaque(u[r]);
  }
  const float xs = xi >= 0 ? logit<DT>(xraw) : NEG_INF_F;
  refer(xs);
  add(xs, sums.s, sums.w);

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
  const float wmx = wave_max64(tmax);
  const Stats own(sums, wmx);
  const float ws = group_sum<64>(own.s), ww = group_sum<64>(own.w);
  if (lane == 0) s_red[0][wave] = wmx, s_red[1][wave] = ws, s_red[2][wave] = ww;
  __syncthreads();
  g = s_group[lane];
  const float mx = wave_max64(g);
  // tau: one wave takes the best k - 1 groups away, several waves rank their shares of them
  // (4096 x 3000, k = 5: 13.0 against 17.6 us with ranks for both)
  if (NWAVE == 1 && k > 0) {
    float tau = mx;
    for (int r = k; r > 1; --r) {
      const uint64_t top = __builtin_amdgcn_ballot_w64(g == tau);
      if (lane == __builtin_ctzll(top | (1ull << 63))) g = NEG_INF_F;
      tau = wave_max64(g);
    }
    if (lane == 0) s_tau = tau;
  } else if (k > 0) {
#pragma unroll
    for (int j = 0; j < 64 / NWAVE; ++j) {
      const int at = wave * (64 / NWAVE) + j;
      const float og = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), at));
      const uint64_t over = __builtin_amdgcn_ballot_w64(g > og);
      const uint64_t level = __builtin_amdgcn_ballot_w64(g == og) & ((1ull << at) - 1);
      if (__builtin_popcountll(over) + __builtin_popcountll(level) == k - 1 && lane == 0)
        s_tau = og;
    }
  }
  // the waves' sums, joined by every wave for itself
  Stats all{mx, 0.f, 0.f};
  if (lane < NWAVE) all = Stats{s_red[0][lane], s_red[1][lane], s_red[2][lane]};
  all.move(mx);
  float S = wave_total(all.s), W = wave_total(all.w);
  if (fabsf(mx) > TLP_FAR && fabsf(mx) < INFINITY) {  // workgroup-uniform
    float s = 0.f, w = 0.f;
#pragma nounroll
    for (int i = tid; i < n; i += NT) {
      const float t = (logit<DT>(x[i]) - mx) * LOG2E_F, e = fast_exp2(t);
      s += e;
      w = fmaf(fmaxf(t, TLP_FLOOR), e, w);
    }
    s = group_sum<64>(s), w = group_sum<64>(w);
    __syncthreads();  // the waves' sums have been read
    if (lane == 0) s_red[1][wave] = s, s_red[2][wave] = w;
    __syncthreads();
    S = wave_total(lane < NWAVE ? s_red[1][lane] : 0.f);
    W = wave_total(lane < NWAVE ? s_red[2][lane] : 0.f);
  }
  // a NaN, +inf or an empty row leaves S NaN or 0
  const bool bad = !SPLIT && !(S > 0.f);
  const Normaliser norm{mx, log2f(S)};
  const int64_t seg = SPLIT ? row * gridDim.y + blockIdx.y : row;
  if constexpr (SPLIT) {
    if (tid == 0) o.part[seg] = Partial{mx, S, W};
  } else {
    if (tid == 0) o.entropy[row] = bad ? NAN : LN2_F * (norm.log2_s - W / S);
    for (int i = tid; i < o.num_tokens; i += NT) {
      if (i != tid) {
        token = o.tokens[row * o.num_tokens + i];
        inside = token >= 0 && token < vocab;
        graw = x[inside ? token : 0];
      }
      o.logprobs[row * o.num_tokens + i] =
          bad || !inside ? NAN : norm.logprob(logit<DT>(graw));
    }
  }
  if (k == 0) return;
  __syncthreads();  // s_tau

  auto put = [&](int rank, float v, int id) {
    if constexpr (SPLIT) {
      o.cand[seg * k + rank] = v;
      o.cand_id[seg * k + rank] = id;
    } else {
      o.top[row * k + rank] = bad ? NAN : norm.logprob(v);
      o.ids[row * k + rank] = bad ? -1 : id;
    }
  };
  const float tau = s_tau;
  const bool bounded = tau != NEG_INF_F;
  if (bounded) {
    auto keep = [&](float v, int i) {
      if (v >= tau) {
        const int slot = atomicAdd(&s_count, 1);
        if (slot < TLP_CAP) s_cv[slot] = v, s_ci[slot] = base + i;
      }
    };
    if (xi >= 0) keep(xs, xi);
    uint32_t hits = 0;  // vectors of this thread that may hold one
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if (r * NT < nvec && may_reach<DT>(u[r], tau)) hits |= 1u << r;
    if (!(tmax >= tau)) hits = 0;
    // one copy of the search for all of them: the code runs once a row, from a cold
    // instruction cache
    while (hits) {
      const int r = __builtin_ctz(hits);
      hits &= hits - 1;
      uint4 h = u[0];
#pragma unroll
      for (int q = 1; q < NV; ++q)
        if (r == q) h = u[q];
#pragma unroll
      for (int j = 0; j < VE; ++j) keep(logit_of<DT>(h, j), head + (tid + r * NT) * VE + j);
    }
  }
  __syncthreads();
  const int count = s_count;
  if (bounded && count <= TLP_CAP) {
    rank_candidates(s_cv, s_ci, count, wave, NWAVE, k, put);
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
  Partial p{NEG_INF_F, 0.f, 0.f};
  if (lane < segments) p = o.part[row * segments + lane];
  const float mx = wave_max64(p.mx);
  Stats all{p.mx, p.s, p.w};
  all.move(mx);
  const float S = wave_total(all.s), W = wave_total(all.w);
  const bool bad = !(S > 0.f);
  const Normaliser norm{mx, log2f(S)};
  if (tid == 0) o.entropy[row] = bad ? NAN : LN2_F * (norm.log2_s - W / S);
  const typename Elem<DT>::T *x = logits + row * stride;
  for (int i = tid; i < o.num_tokens; i += TLP_JOIN_NT) {
    const int64_t t = o.tokens[row * o.num_tokens + i];
    o.logprobs[row * o.num_tokens + i] =
        bad || t < 0 || t >= vocab ? NAN : norm.logprob(logit<DT>(x[t]));
  }
  if (bad) {  // (its segments may have fewer than k candidates, whose ranks leave gaps)
    if (tid < k) o.top[row * k + tid] = NAN, o.ids[row * k + tid] = -1;
    return;
  }
  __syncthreads();
  rank_candidates(s_cv, s_ci, count, tid >> 6, TLP_JOIN_NT / 64, k, [&](int rank, float v, int id) {
    o.top[row * k + rank] = norm.logprob(v);
    o.ids[row * k + rank] = id;
  });
}

// Values that a workgroup of 1024 threads holds, and so the longest row of one launch.
constexpr int TLP_CAPACITY = 1024 * 7 * 8;
constexpr int TLP_SEGMENT_BYTES = 1024 * 7 * 16;

// Segments of a row that does not fit (0: it does), of equal length, a multiple of 8.
inline int tlp_segments(int vocab, int dtype, int *segment) {
  if (vocab <= TLP_CAPACITY) return 0;
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
    token_logprobs_kernel<DT, 1024, 7, 8, true>
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
  if (vocab <= 64 * 7 * VE) VFL_TLP(64, 7, 8);
  else if (vocab <= 256 * 7 * VE) VFL_TLP(256, 7, 8);
  else if (vocab <= 1024 * 7 * VE) VFL_TLP(1024, 7, 8);
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
  if (rows < 0 || !grid_fits(rows, 1024) || vocab <= 0 || vocab > TLP_MAX_VOCAB ||
      (row_stride != 0 && row_stride < vocab) || k < 0 || k > TLP_MAX_K || k > vocab ||
      num_tokens < 0) {
    set_error("token_logprobs: need 0 <= k <= min(%d, vocab), vocab up to %d, fewer than 2^22 rows "
              "and row_stride 0 or at least vocab (k %d, vocab %d, stride %lld, rows %lld)",
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
