// The C entry of packed cross-attention: argument checks and the shape of the launch (the kernels
// are cross_attention.h's).
#include "cross_attention.h"

#include <algorithm>

namespace vfl {

namespace {

// Key groups of a workgroup and workgroups of a run of keys.
struct CrossPlan {
  int ks, splits;
  bool spread;
};

// us, 16 heads of 64 over 256 to 1024 keys if not said otherwise, bf16:
// - more key groups are the faster ones where tiles of 128 queries are few or would stay mostly
//   empty.  One / two / four groups: 8 runs of 60 to 128 queries 19.7 / 13.4 / 18.1, 590 queries x 12
//   heads over 590 keys 13.8 / 10.1 / 16.7, 64 runs of 40 to 64 45.0 / 39.8 / 74.8; yet 64 of 60 to
//   128 49.1 / 54.4 / 124, 16 of 31 to 257 26.5 / 28.8 / 48.5; 9 queries x 12 heads over 590 keys
//   12.6 / 9.4 / 8.9.  fp32, whose tiles take a CU's LDS in two groups: 8 runs of 60 to 128 56.8 / 38.3
//   / 48.1, but 64 of 20 to 32 110 / 128 / 120, 16 of 31 to 257 67.8 / 86.4 / 116.
// - runs of keys are split where that leaves no more workgroups than two a CU (fp32: one): 8 runs
//   of 20 to 32 queries over 1000 to 2000 keys whole 22.9, in four parts 17.9, in eight 20.7; fp32 4
//   of 60 to 64 whole 63.6, in four 26.6, in eight 30.4; 60 queries x 8 heads of 128 over 30000 keys
//   in 16 parts 48.0, in 32 35.5 (21 and 29 over 17001 and 39999 57.6 / 58.0).  A call's rows all take
//   a place for each part, also those of no sequence: parts that would need more than 128 MB, twice
//   what a launch's own queries ever take, are not made.
// - launches of up to two workgroups a CU go to any XCD: 12 heads, fp32, 590 queries in two parts
//   21.2, a head to an XCD 33.6.
constexpr int64_t MOST_ROWS = 2147483647LL - 1024;  // (a tile past the last is counted in 32 bits)

CrossPlan cross_plan(int64_t num_queries, int64_t sequences, int H, int D, bool f32,
                     int64_t max_queries, int64_t max_keys) {
  const int DG = (D + 31) / 32;
  max_queries = std::min(max_queries, num_queries);
  CrossPlan p{1, 1, false};
  auto workgroups = [&](int ks) {  // that hold queries, at most
    const int64_t qt = 128 / ks, tiles = (max_queries + qt - 1) / qt;
    const int64_t by_length = sequences * (tiles > 1 ? tiles : 1);
    const int64_t by_rows = num_queries / qt + sequences;
    return (by_length < by_rows ? by_length : by_rows) * H;
  };
  if (max_queries <= 32 && workgroups(1) <= 64) p.ks = 4;
  else if ((!f32 && max_queries <= 64) || workgroups(1) <= 256) p.ks = 2;
  const int most = cross_most_groups(f32, DG);
  if (p.ks > most) p.ks = most;
  while (p.ks > 1 && 64 * (p.ks / 2) >= max_keys) p.ks /= 2;
  const int64_t wgs = workgroups(p.ks);
  const int64_t fill = (f32 ? 256 : 512) / wgs, parts = max_keys / (f32 ? 64 : 256 * p.ks);
  const int64_t room = MOST_WORKSPACE / (num_queries * H * split_part_bytes(D));
  const int64_t most_parts = std::min({fill, parts, room, (int64_t)32});
  if (most_parts >= 2) p.splits = (int)most_parts;
  p.spread = wgs * p.splits <= 512;
  return p;
}

}  // namespace

}  // namespace vfl

using namespace vfl;

extern "C" int64_t vfl_packed_cross_attention_workspace(int64_t num_queries, int64_t num_sequences,
                                                        int num_heads, int head_dim,
                                                        int64_t max_query_len,
                                                        int64_t max_key_len, int dtype) {
  if (num_queries <= 0 || num_sequences <= 0 || num_heads <= 0 || head_dim <= 0 ||
      num_queries > MOST_ROWS || num_heads > 65535 || num_sequences > MOST_ROWS / num_heads ||
      head_dim > 256)
    return 0;  // nothing to do, or refused
  const CrossPlan p = cross_plan(num_queries, num_sequences, num_heads, head_dim,
                                 dtype == VFL_FLOAT32, max_query_len, max_key_len);
  return p.splits > 1 ? num_queries * num_heads * p.splits * split_part_bytes(head_dim) : 0;
}

extern "C" int vfl_packed_cross_attention(
    const void *query, int64_t query_stride_token, int64_t query_stride_head, const void *key,
    int64_t key_stride_token, int64_t key_stride_head, const void *value,
    int64_t value_stride_token, int64_t value_stride_head, void *out,
    const int32_t *query_start_loc, const int32_t *key_start_loc, int64_t num_queries,
    int64_t num_keys, int64_t num_sequences, int num_heads, int head_dim, int64_t max_query_len,
    int64_t max_key_len, float scale, int dtype, void *workspace, void *stream) {
  clear_error();
  const char *who = "packed_cross_attention";
  if (dtype != VFL_FLOAT32 && dtype != VFL_BFLOAT16 && dtype != VFL_FLOAT16) {
    set_error("%s: unsupported dtype code %d", who, dtype);
    return VFL_E_INVALID;
  }
  if (!vfl_get_isa(dtype, 16, head_dim) || head_dim > 256) {
    set_error("%s: no kernel for head_dim %d", who, head_dim);
    return VFL_E_UNSUPPORTED;
  }
  if (num_queries < 0 || num_keys < 0 || num_queries > MOST_ROWS || num_keys > MOST_ROWS ||
      num_sequences < 0 || num_heads <= 0 || num_heads > 65535 || max_query_len < 0 ||
      max_key_len < 0 || max_query_len > 2147483647LL || num_sequences > 2147483647LL / num_heads) {
    set_error("%s: bad sizes (queries %lld keys %lld sequences %lld heads %d longest %lld %lld)", who,
              (long long)num_queries, (long long)num_keys, (long long)num_sequences, num_heads,
              (long long)max_query_len, (long long)max_key_len);
    return VFL_E_INVALID;
  }
  if (!(fabsf(scale) < INFINITY)) {
    set_error("%s: scale %f", who, (double)scale);
    return VFL_E_INVALID;
  }
  if (num_queries == 0 || num_sequences == 0) return VFL_OK;
  if (!query || !out || !query_start_loc || !key_start_loc || (num_keys && (!key || !value))) {
    set_error("%s: null pointer argument", who);
    return VFL_E_INVALID;
  }
  const int eb = elem_bytes(dtype);
  if (((uintptr_t)query | (uintptr_t)key | (uintptr_t)value | (uintptr_t)workspace) % 16 ||
      (uintptr_t)out % eb ||
      (query_stride_token | query_stride_head | key_stride_token | key_stride_head |
       value_stride_token | value_stride_head) % (16 / eb)) {
    set_error("%s: misaligned rows (query, key, value, their strides and workspace 16 bytes, out "
              "its element)", who);
    return VFL_E_INVALID;
  }
  // (a tile's rows are addressed by 32-bit offsets)
  if (key_stride_token < 0 || value_stride_token < 0 || key_stride_token > CROSS_MAX_STRIDE ||
      value_stride_token > CROSS_MAX_STRIDE) {
    set_error("%s: key and value token strides %lld, %lld (0 to %d)", who,
              (long long)key_stride_token, (long long)value_stride_token, CROSS_MAX_STRIDE);
    return VFL_E_INVALID;
  }
  const CrossPlan plan = cross_plan(num_queries, num_sequences, num_heads, head_dim,
                                    dtype == VFL_FLOAT32, max_query_len, max_key_len);
  if (!grid_fits(cross_grid(num_queries, num_sequences, num_heads, plan.ks, plan.splits, plan.spread),
                 256)) {
    set_error("%s: %lld queries of %lld sequences x %d heads exceed a launch", who,
              (long long)num_queries, (long long)num_sequences, num_heads);
    return VFL_E_INVALID;
  }
  CrossArgs a;
  a.q = query, a.k = key, a.v = value;
  a.q_st = query_stride_token, a.q_sh = query_stride_head;
  a.k_st = key_stride_token, a.k_sh = key_stride_head;
  a.v_st = value_stride_token, a.v_sh = value_stride_head;
  a.out = out;
  a.q_start = query_start_loc, a.k_start = key_start_loc;
  a.num_queries = num_queries, a.num_keys = num_keys;
  a.sequences = (int)num_sequences, a.H = num_heads, a.D = head_dim;
  a.scale_log2 = decode_scale_log2(scale);
  a.negative = scale < 0.f, a.spread = plan.spread;
  a.out_vec = (uintptr_t)out % (4 * eb) == 0;
  a.splits = plan.splits, a.part = {nullptr, nullptr};
  if (plan.splits > 1) {
    if (!workspace) {
      set_error("%s: null workspace", who);
      return VFL_E_INVALID;
    }
    a.part.acc = (float *)workspace;
    a.part.ml = (float2 *)(a.part.acc + num_queries * num_heads * plan.splits * head_dim);
  }
  hipStream_t s = (hipStream_t)stream;
  if (dtype == VFL_FLOAT32) return launch_cross_f32(a, plan.ks, s);
  if (dtype == VFL_BFLOAT16) return launch_cross_bf16(a, plan.ks, s);
  return launch_cross_f16(a, plan.ks, s);
}
