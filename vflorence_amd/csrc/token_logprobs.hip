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
constexpr int TLP_NT = 512;

template <int DT> __device__ __forceinline__ float logit(typename Elem<DT>::T v) {
  if constexpr (DT == VFL_FLOAT32) return v;
  else return Mfma<DT>::widen(v);
}

// (value, id) order: higher value first, then lower id.
__device__ __forceinline__ bool ahead(float a, int ia, float b, int ib) {
  return a > b || (a == b && ia < ib);
}

template <int DT>
__global__ __launch_bounds__(TLP_NT) void token_logprobs_kernel(
    const typename Elem<DT>::T *__restrict__ logits, int64_t stride, int vocab,
    const int64_t *__restrict__ tokens, int num_tokens, int k, float *__restrict__ logprobs,
    float *__restrict__ entropy, float *__restrict__ top, int64_t *__restrict__ ids) {
  __shared__ float s_v[TLP_NT], s_w[TLP_NT];
  __shared__ int s_i[TLP_NT];
  const int64_t row = blockIdx.x;
  const typename Elem<DT>::T *x = logits + row * stride;
  const int tid = threadIdx.x;

  float m = NEG_INF_F;
  bool bad = false;
  for (int i = tid; i < vocab; i += TLP_NT) {
    const float v = logit<DT>(x[i]);
    bad |= !(v < INFINITY);
    m = fmaxf(m, v);
  }
  s_v[tid] = m;
  bad = __syncthreads_or(bad);
  for (int n = TLP_NT / 2; n > 0; n /= 2) {
    if (tid < n) s_v[tid] = fmaxf(s_v[tid], s_v[tid + n]);
    __syncthreads();
  }
  m = s_v[0];
  bad |= m == NEG_INF_F;
  __syncthreads();
  float S = 0.f, W = 0.f;
  for (int i = tid; i < vocab; i += TLP_NT) {
    const float t = logit<DT>(x[i]) - m, e = expf(t);
    S += e;
    if (e > 0.f) W += t * e;
  }
  s_v[tid] = S, s_w[tid] = W;
  __syncthreads();
  for (int n = TLP_NT / 2; n > 0; n /= 2) {
    if (tid < n) s_v[tid] += s_v[tid + n], s_w[tid] += s_w[tid + n];
    __syncthreads();
  }
  S = s_v[0], W = s_w[0];
  const float log_s = logf(S);
  if (tid == 0) entropy[row] = bad ? NAN : log_s - W / S;
  for (int i = tid; i < num_tokens; i += TLP_NT) {
    const int64_t t = tokens[row * num_tokens + i];
    logprobs[row * num_tokens + i] =
        bad || t < 0 || t >= vocab ? NAN : (logit<DT>(x[t]) - m) - log_s;
  }
  float last = INFINITY;
  int last_id = -1;
  for (int r = 0; r < k; ++r) {
    float bv = NEG_INF_F;
    int bi = INT32_MAX;
    for (int i = tid; i < vocab; i += TLP_NT) {
      const float v = logit<DT>(x[i]);
      if (ahead(last, last_id, v, i) && ahead(v, i, bv, bi)) bv = v, bi = i;
    }
    __syncthreads();
    s_v[tid] = bv, s_i[tid] = bi;
    __syncthreads();
    for (int n = TLP_NT / 2; n > 0; n /= 2) {
      if (tid < n && ahead(s_v[tid + n], s_i[tid + n], s_v[tid], s_i[tid]))
        s_v[tid] = s_v[tid + n], s_i[tid] = s_i[tid + n];
      __syncthreads();
    }
    last = s_v[0], last_id = s_i[0];
    if (tid == 0) {
      top[row * k + r] = bad ? NAN : (last - m) - log_s;
      ids[row * k + r] = bad ? -1 : last_id;
    }
  }
}

}  // namespace vfl

using namespace vfl;

extern "C" int vfl_token_logprobs(const void *logits, int64_t row_stride, int64_t rows, int vocab,
                                  int dtype, const int64_t *tokens, int num_tokens, int k,
                                  float *logprobs, float *entropy, float *top_logprobs,
                                  int64_t *top_ids, void *stream) {
  clear_error();
  if (dtype != VFL_FLOAT32 && dtype != VFL_BFLOAT16 && dtype != VFL_FLOAT16) {
    set_error("token_logprobs: unsupported dtype code %d", dtype);
    return VFL_E_INVALID;
  }
  if (rows < 0 || rows > 2147483647LL || vocab <= 0 || row_stride < vocab || k < 0 ||
      k > TLP_MAX_K || k > vocab || num_tokens < 0) {
    set_error("token_logprobs: need 0 <= k <= min(%d, vocab) and row_stride >= vocab (k %d, vocab "
              "%d, stride %lld, rows %lld)",
              TLP_MAX_K, k, vocab, (long long)row_stride, (long long)rows);
    return VFL_E_INVALID;
  }
  if (rows == 0) return VFL_OK;
  if (!logits || !entropy || (num_tokens && (!tokens || !logprobs)) ||
      (k && (!top_logprobs || !top_ids))) {
    set_error("token_logprobs: null pointer argument");
    return VFL_E_INVALID;
  }
  if ((uintptr_t)logits % elem_bytes(dtype)) {
    set_error("token_logprobs: logits are not aligned to their element");
    return VFL_E_INVALID;
  }
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    token_logprobs_kernel<DT><<<dim3((unsigned)rows), dim3(TLP_NT), 0, s>>>(
        (const typename Elem<DT>::T *)logits, row_stride, vocab, tokens, num_tokens, k, logprobs,
        entropy, top_logprobs, top_ids);
    return launch_status("token_logprobs");
  };
  if (dtype == VFL_FLOAT32) return go(std::integral_constant<int, VFL_FLOAT32>{});
  if (dtype == VFL_BFLOAT16) return go(std::integral_constant<int, VFL_BFLOAT16>{});
  return go(std::integral_constant<int, VFL_FLOAT16>{});
}
