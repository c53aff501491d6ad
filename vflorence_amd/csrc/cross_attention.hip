// The C entry of packed cross-attention: argument checks and the shape of the launch (the kernels
// are cross_attention.h's).
#include "cross_attention.h"

namespace vfl {

namespace {

// Key groups of a workgroup and workgroups of a run of keys.
struct CrossPlan {
  int ks, tiles, splits;
};

CrossPlan cross_plan(int64_t sequences, int H, int D, bool f32, int64_t max_queries,
                     int64_t max_keys) {
  const int DG = (D + 31) / 32;
  CrossPlan p{1, 1, 1};
  if (max_queries < 1) max_queries = 1;
  const int64_t wide = sequences * H * ((max_queries + 127) / 128);
  p.ks = max_queries <= 32 || wide <= 32 ? 4 : max_queries <= 64 || wide <= 192 ? 2 : 1;
  const int most = cross_most_groups(f32, DG);
  if (p.ks > most) p.ks = most;
  while (p.ks > 1 && 64 * (p.ks / 2) >= max_keys) p.ks /= 2;
  const int64_t qt = 128 / p.ks;
  p.tiles = (int)((max_queries + qt - 1) / qt);
  const int64_t wgs = sequences * H * p.tiles;
  if (wgs < 256 && max_keys > 2048) {
    const int64_t fill = 512 / wgs, parts = max_keys / (256 * p.ks);
    const int64_t s = fill < parts ? fill : parts;
    if (s >= 2) p.splits = (int)s;
  }
  return p;
}

}  // namespace

}  // namespace vfl

using namespace vfl;

extern "C" int64_t vfl_packed_cross_attention_workspace(int64_t num_queries, int64_t num_sequences,
                                                        int num_heads, int head_dim,
                                                        int64_t max_query_len,
                                                        int64_t max_key_len, int dtype) {
  if (num_queries <= 0 || num_sequences <= 0 || num_heads <= 0 || head_dim <= 0) return 0;
  const CrossPlan p = cross_plan(num_sequences, num_heads, head_dim, dtype == VFL_FLOAT32,
                                 max_query_len, max_key_len);
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
  if (num_queries < 0 || num_keys < 0 || num_queries > 2147483647LL || num_keys > 2147483647LL ||
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
  if ((uintptr_t)query % eb || (uintptr_t)key % eb || (uintptr_t)value % eb ||
      (uintptr_t)out % eb || (uintptr_t)workspace % 16) {
    set_error("%s: misaligned pointer (workspace 16 bytes, others their element)", who);
    return VFL_E_INVALID;
  }
  const CrossPlan plan = cross_plan(num_sequences, num_heads, head_dim, dtype == VFL_FLOAT32,
                                    max_query_len, max_key_len);
  if (!grid_fits((num_sequences * num_heads + 7) / 8 * 8 * plan.tiles * plan.splits, 256)) {
    set_error("%s: %lld sequences x %d heads x %d tiles exceed a launch", who,
              (long long)num_sequences, num_heads, plan.tiles);
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
  a.tiles = plan.tiles;
  a.scale_log2 = decode_scale_log2(scale);
  a.negative = scale < 0.f;
  const int64_t vec = 16 / eb;
  a.vec = ((uintptr_t)query | (uintptr_t)key | (uintptr_t)value) % 16 == 0 &&
          (a.q_st | a.q_sh | a.k_st | a.k_sh | a.v_st | a.v_sh) % vec == 0;
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
