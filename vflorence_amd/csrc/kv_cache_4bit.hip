// Writing keys and values to a paged cache held in 4 bits, and reading them back by their slots
// (gfx950); the format is e2m1.h's.
//
// Per token, head and group of 32 dims, for K and for V:
//   a = max |x|,  scale = the smallest power of two with a / scale <= 6,  code = rne(x / scale)
// The division by a power of two is exact, so a value is rounded once.  A group that holds an
// infinity or a NaN has no such scale: its byte is 255 and every value reads as NaN.
//
// A pair of lanes takes a group, 16 dims each.  A wave takes 32 groups: in a step those of a
// token, in a prompt two groups of 16 tokens.  K's bytes of a group lie together.  V's lie 16
// apart, one for each two dims, beside the part's other tokens: a wave whose 16 tokens fill a part
// turns them in LDS and moves 16 bytes at a time, other tokens move bytes.  No byte holds two
// tokens' values, so nothing is read back, nothing is ordered, and a call's bytes are the same on
// every run.
//
// What bounds it: prompts HBM (64 of 256 to 1024 tokens x 16 heads of 64, bf16, written 36.1 us, read
// back 35.9 on tensors that the last call left in the 256 MB of last-level cache, 46 and 41 on
// other caches, read back into rows that were not written lately 65: 213 MB either way, which a large
// copy moves in 41.7; the counters show 166 MB fetched and 44 written by the append).  Steps their chain of slots, rows and stores: 256 rows x 16 heads 3.6
// and 3.2 us, 4 x 12 2.8 both.
#include <stdio.h>

#include "e2m1.h"

namespace vfl {

int check_4bit_cache(const char *who, int dtype, int num_heads, int head_dim, int block_size,
                     int64_t num_blocks) {
  if (dtype != VFL_FLOAT32 && dtype != VFL_BFLOAT16 && dtype != VFL_FLOAT16) {
    set_error("%s: unsupported dtype code %d", who, dtype);
    return VFL_E_INVALID;
  }
  if (num_heads <= 0 || num_heads > 65535 || num_blocks < 0 || num_blocks > 2147483647LL) {
    set_error("%s: bad sizes (heads %d blocks %lld)", who, num_heads, (long long)num_blocks);
    return VFL_E_INVALID;
  }
  if (!vfl_get_isa(dtype, block_size, head_dim)) {
    set_error("%s: no kernel for block_size %d, head_dim %d", who, block_size, head_dim);
    return VFL_E_UNSUPPORTED;
  }
  return VFL_OK;
}

namespace {

struct Cache4Args {
  const void *x[2];  // K's and V's rows (append: read, gather: written)
  int64_t st[2], sh[2];
  uint8_t *cache;
  const int64_t *slots;
  int T, H, D, G, shift;  // 16 << shift tokens a block
  int64_t num_blocks;
};

// 16 elements as words of memory.
template <int DT, bool ALIGNED>
__device__ __forceinline__ void load16(const typename Elem<DT>::T *p,
                                       uint32_t (&w)[16 * sizeof(typename Elem<DT>::T) / 4]) {
  constexpr int WORDS = 16 * sizeof(typename Elem<DT>::T) / 4;
  constexpr int PER = Elem<DT>::VEC;
#pragma unroll
  for (int i = 0; i < WORDS / 4; ++i) {
    const uint4 u = ALIGNED ? reinterpret_cast<const uint4 *>(p)[i]
                            : load16_unaligned<DT>(p + PER * i);
    w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
  }
}
template <int DT, bool ALIGNED>
__device__ __forceinline__ void store16(typename Elem<DT>::T *p,
                                        const uint32_t (&w)[16 * sizeof(typename Elem<DT>::T) / 4]) {
  constexpr int WORDS = 16 * sizeof(typename Elem<DT>::T) / 4;
  constexpr int PER = Elem<DT>::VEC;
#pragma unroll
  for (int i = 0; i < WORDS / 4; ++i) {
    const uint4 u = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    if constexpr (ALIGNED) reinterpret_cast<uint4 *>(p)[i] = u;
    else store16_unaligned<DT>(p + PER * i, u);
  }
}

// Magnitudes are compared as patterns without their sign, which order like the values, an
// infinity and then NaN above them all; 16-bit ones two at a time.
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
template <int DT> struct Magnitude {
  static constexpr bool PAIRS = DT != VFL_FLOAT32;
  static constexpr uint32_t INF = DT == VFL_FLOAT32    ? 0x7f800000u
                                  : DT == VFL_BFLOAT16 ? 0x7f80u
                                                       : 0x7c00u;
  static __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) {
    if constexpr (!PAIRS) return max(a, b);
    else
      return __builtin_bit_cast(uint32_t,
                                __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a),
                                                          __builtin_bit_cast(ushort2_t, b)));
  }
  // of a lane's elements and its neighbour's
  template <int WORDS> static __device__ __forceinline__ uint32_t of(const uint32_t (&w)[WORDS]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) m = largest(m, w[i] & (PAIRS ? 0x7fff7fffu : 0x7fffffffu));
    if constexpr (PAIRS) m = max(m >> 16, m & 0xffffu);
    return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR1, 0xF, 0xF, false));
  }
  static __device__ __forceinline__ float value(uint32_t pattern) {
    if constexpr (PAIRS) return Mfma<DT>::widen(pattern);
    else return __uint_as_float(pattern);
  }
};

__device__ __forceinline__ uint32_t of_neighbour(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, DPP_QUAD_XOR1, 0xF, 0xF, false);
}

constexpr int CACHE4_NT = 256;

// Waves of a launch: token windows by groups, K and V each.
inline int64_t cache4_waves(bool step, int64_t T, int HG) {
  return step ? T * ((HG + 31) / 32) * 2 : (T + 15) / 16 * ((HG + 1) / 2) * 2;
}

// The part of a run of tokens that a wave of 16-token windows moves whole: the window's tokens
// t0 .. t0 + 15 hold at most one first token of a part whose 16 tokens follow one another.
struct Window {
  int64_t slot;   // of token t0 - 16 + lane, or -1
  uint64_t full;  // lanes whose token begins such a part

  __device__ __forceinline__ Window(const Cache4Args &a, int t0) {
    const int lane = __lane_id(), t = t0 - 16 + lane;
    const bool in = t >= 0 && t < a.T;
    const int64_t s = a.slots[min(max(t, 0), a.T - 1)];
    const uint64_t room = (uint64_t)a.num_blocks << (4 + a.shift);
    slot = in && (uint64_t)s < room ? s : -1;
    const int64_t before = __shfl_up(slot, 1);
    const uint64_t on = __builtin_amdgcn_ballot_w64(lane > 0 && slot > 0 && slot == before + 1);
    const bool begins = slot >= 0 && slot % 16 == 0 && lane < 48 &&
                        ((on >> 1 >> lane) & 0x7fff) == 0x7fff;
    full = __builtin_amdgcn_ballot_w64(begins);
  }
  // Whether the token in lane `l` (16 .. 31) is moved with its part.
  __device__ __forceinline__ bool in_part(int l, int64_t s) const {
    return s >= 0 && (full >> (l - (int)(s % 16)) & 1);
  }
};

// Calls `body(token, hg, slot, in, whole)` for a lane's groups: head and group hg = h * G + g of
// `token` (its own only where `in`), whose slot is `slot` (-1: none).  STEP: 32 groups of one token a
// wave; else two groups of 16 tokens.  whole: the wave's 16 tokens are a part (a wave-uniform
// compile-time flag).
template <bool STEP, typename F>
__device__ __forceinline__ void for_units(const Cache4Args &a, int64_t w, F body) {
  const int lane = __lane_id(), HG = a.H * a.G;
  if constexpr (STEP) {
    const int per = (HG + 31) / 32;
    const int token = (int)(w / per), hg = (int)(w % per) * 32 + lane / 2;
    const int64_t s = a.slots[token];
    const uint64_t room = (uint64_t)a.num_blocks << (4 + a.shift);
    body(token, hg, (uint64_t)s < room ? s : -1, hg < HG, std::false_type{});
  } else {
    const int per = (HG + 1) / 2;
    const int t0 = (int)(w / per) * 16, hg = (int)(w % per) * 2 + (lane >> 1 & 1);
    const Window win(a, t0);
    const uint64_t starts = win.full & 0xffff0000u;
    const int l = 16 + lane / 4;
    if (starts) {  // wave-uniform
      const int first = __builtin_ctzll(starts);
      const int token = t0 - 16 + first + lane / 4;
      body(token, hg, __shfl(win.slot, first + lane / 4), hg < HG, std::true_type{});
    }
    const int64_t s = __shfl(win.slot, l);
    const bool mine = t0 + lane / 4 < a.T && !win.in_part(l, s);
    if (__builtin_amdgcn_ballot_w64(mine) != 0)
      body(t0 + lane / 4, hg, s, hg < HG && mine, std::false_type{});
  }
}

// Where a group lies in the cache.
struct Place {
  uint8_t *tile, *scale;  // its 256 bytes of K or V, and the scale byte of its token
  int t;                  // token within the part
  __device__ __forceinline__ Place(const Cache4Args &a, int v, int hg, int64_t slot) {
    const E2m1Layout lay(a.H, a.G, 1 << a.shift);
    const int h = hg / a.G, g = hg % a.G;
    const int64_t block = slot >> (4 + a.shift);
    const int part = (int)(slot >> 4) & ((1 << a.shift) - 1);
    t = (int)(slot & 15);
    uint8_t *b = a.cache + block * lay.block_bytes;
    tile = b + (v ? lay.values(h, part) : lay.keys(h, part)) + g * 256;
    scale = b + lay.scales(h, part) + (t / 4) * 8 * a.G + (v ? 4 * a.G : 0) + g * 4 + t % 4;
  }
};

template <int DT, bool ALIGNED, bool STEP>
__global__ __launch_bounds__(CACHE4_NT) void append_4bit_kernel(Cache4Args a, int64_t waves) {
  using T = typename Elem<DT>::T;
  constexpr int WORDS = 16 * sizeof(T) / 4;
  __shared__ __align__(16) uint8_t s_turn[CACHE4_NT / 64][512];
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t w = (int64_t)blockIdx.x * (CACHE4_NT / 64) + wave;
  if (w >= waves) return;
  const int v = (int)(w & 1), odd = lane & 1;
  for_units<STEP>(a, w >> 1, [&](int token, int hg, int64_t slot, bool in, auto whole) {
    in = in && slot >= 0;
    const int h = hg / a.G, d = (hg % a.G) * 32 + 16 * odd;
    uint32_t x[WORDS];
    if (in && d < a.D) {
      load16<DT, ALIGNED>((const T *)a.x[v] + token * a.st[v] + h * a.sh[v] + d, x);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) x[i] = 0;
    }
    const uint32_t m = Magnitude<DT>::of(x);
    const bool finite = m < Magnitude<DT>::INF;
    const uint32_t byte = finite ? e2m1_scale_byte(Magnitude<DT>::value(m)) : E2M1_NAN;
    const float scale = e2m1_scale(finite ? byte : 127);
    uint32_t c[2] = {e2m1_pack8<DT>(x, scale), e2m1_pack8<DT>(x + WORDS / 2, scale)};
    if (!finite) c[0] = c[1] = 0;
    const Place at(a, v, hg, in ? slot : 0);
    if (in && !odd) *at.scale = (uint8_t)byte;
    if (!v) {
      if (in) *reinterpret_cast<uint2 *>(at.tile + at.t * 16 + 8 * odd) = make_uint2(c[0], c[1]);
      return;
    }
    // the even lane takes the bytes of dims 0 .. 7 (+ 16), the odd one's those of 8 .. 15
    const uint32_t got = of_neighbour(odd ? c[0] : c[1]);
    const uint32_t lo = odd ? got : c[0], hi = odd ? c[1] : got;
    const uint32_t even = (lo & 0x0f0f0f0fu) | (hi << 4 & 0xf0f0f0f0u);
    const uint32_t odds = (lo >> 4 & 0x0f0f0f0fu) | (hi & 0xf0f0f0f0u);
    if constexpr (decltype(whole)::value) {
      uint8_t *turn = s_turn[wave] + (lane >> 1 & 1) * 256 + 128 * odd + lane / 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        turn[32 * i] = (uint8_t)(even >> (8 * i));
        turn[32 * i + 16] = (uint8_t)(odds >> (8 * i));
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      // lane l < 32: 16 tokens of dims l % 16 (+ 16) of the l / 16-th group
      const int other = (int)(hg & ~1) + (lane >> 4 & 1);
      const Place to(a, 1, other, slot);  // (the part's block is the same for every token)
      if (lane < 32 && other < a.H * a.G)
        *reinterpret_cast<uint4 *>(to.tile + (lane & 15) * 16) =
            *reinterpret_cast<const uint4 *>(s_turn[wave] + lane * 16);
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
    } else if (in) {
      uint8_t *p = at.tile + 128 * odd + at.t;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[32 * i] = (uint8_t)(even >> (8 * i));
        p[32 * i + 16] = (uint8_t)(odds >> (8 * i));
      }
    }
  });
}

template <int DT, bool ALIGNED, bool STEP>
__global__ __launch_bounds__(CACHE4_NT) void gather_4bit_kernel(Cache4Args a, int64_t waves) {
  using T = typename Elem<DT>::T;
  constexpr int WORDS = 16 * sizeof(T) / 4;
  __shared__ __align__(16) uint8_t s_turn[CACHE4_NT / 64][512];
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t w = (int64_t)blockIdx.x * (CACHE4_NT / 64) + wave;
  if (w >= waves) return;
  const int v = (int)(w & 1), odd = lane & 1;
  for_units<STEP>(a, w >> 1, [&](int token, int hg, int64_t slot, bool in, auto whole) {
    const bool held = in && slot >= 0;
    const int h = hg / a.G, d = (hg % a.G) * 32 + 16 * odd;
    const Place at(a, v, held ? hg : 0, held ? slot : 0);
    uint32_t c[2] = {0, 0}, byte = 127;
    if (held) byte = *at.scale;
    if (!v) {
      if (held) {
        const uint2 u = *reinterpret_cast<const uint2 *>(at.tile + at.t * 16 + 8 * odd);
        c[0] = u.x, c[1] = u.y;
      }
    } else {
      uint32_t even = 0, odds = 0;  // bytes of dims 8 odd + 0, 2, 4, 6 and 1, 3, 5, 7 (+ 16)
      if constexpr (decltype(whole)::value) {
        const int other = (hg & ~1) + (lane >> 4 & 1);
        if (lane < 32 && other < a.H * a.G) {
          const Place from(a, 1, other, slot);
          *reinterpret_cast<uint4 *>(s_turn[wave] + lane * 16) =
              *reinterpret_cast<const uint4 *>(from.tile + (lane & 15) * 16);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        const uint8_t *turn = s_turn[wave] + (lane >> 1 & 1) * 256 + 128 * odd + lane / 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          even |= (uint32_t)turn[32 * i] << (8 * i);
          odds |= (uint32_t)turn[32 * i + 16] << (8 * i);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
      } else if (held) {
        const uint8_t *p = at.tile + 128 * odd + at.t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          even |= (uint32_t)p[32 * i] << (8 * i);
          odds |= (uint32_t)p[32 * i + 16] << (8 * i);
        }
      }
      const uint32_t lo = (even & 0x0f0f0f0fu) | (odds << 4 & 0xf0f0f0f0u);
      const uint32_t hi = (even >> 4 & 0x0f0f0f0fu) | (odds & 0xf0f0f0f0u);
      const uint32_t got = of_neighbour(odd ? lo : hi);
      c[0] = odd ? got : lo;
      c[1] = odd ? hi : got;
    }
    if (!in || d >= a.D) return;
    const float scale = e2m1_scale(byte);
    uint32_t x[WORDS];
    e2m1_unpack8<DT>(c[0], scale, x);
    e2m1_unpack8<DT>(c[1], scale, x + WORDS / 2);
    store16<DT, ALIGNED>((T *)a.x[v] + token * a.st[v] + h * a.sh[v] + d, x);
  });
}

// A decode step's tokens lie in parts of their own: a wave a token and 32 groups.  A prompt's fill
// parts.  The host does not see which they are: calls of up to 512 tokens (the most rows of a
// step that the projections take) are taken for steps, since a step's call comes for every token
// generated and a prompt's once a request.  16 heads of 64, us, written / read, as a step against as
// a prompt: 256 rows 3.66 / 3.12 against 4.05 / 3.24, 512 4.52 / 3.31 against 4.86 / 3.51; a prompt
// of 512 loses what three or four steps gain, 4.21 / 3.30 against 2.99 / 3.21; of 590 it would be
// 4.84 / 3.77 against 3.11 / 3.40, and eight of 590 18.3 / 11.6 against 7.0 / 8.2.
inline bool is_step(int64_t T) { return T <= 512; }

template <bool APPEND>
int move_4bit(const char *who, const void *key, const void *value, int64_t k_st, int64_t k_sh,
              int64_t v_st, int64_t v_sh, void *cache, const int64_t *slots, int64_t T, int H, int D,
              int BS, int64_t num_blocks, int dtype, hipStream_t stream) {
  clear_error();
  const int st = check_4bit_cache(who, dtype, H, D, BS, num_blocks);
  if (st != VFL_OK) return st;
  const int G = e2m1_groups(D);
  const bool step = is_step(T);
  if (T < 0 || T > 2147483647LL - 64 ||
      !grid_fits((cache4_waves(step, T, H * G) + 3) / 4, CACHE4_NT)) {
    set_error("%s: %lld tokens x %d heads", who, (long long)T, H);
    return VFL_E_INVALID;
  }
  if (T == 0 || (APPEND && num_blocks == 0)) return VFL_OK;
  if (!key || !value || !slots || (num_blocks && !cache)) {
    set_error("%s: null pointer argument", who);
    return VFL_E_INVALID;
  }
  const int eb = elem_bytes(dtype);
  if ((uintptr_t)cache % 16 || (uintptr_t)slots % 8 || (uintptr_t)key % eb ||
      (uintptr_t)value % eb) {
    set_error("%s: misaligned pointer (cache 16 bytes, others their element)", who);
    return VFL_E_INVALID;
  }
  Cache4Args a;
  a.x[0] = key, a.x[1] = value;
  a.st[0] = k_st, a.st[1] = v_st, a.sh[0] = k_sh, a.sh[1] = v_sh;
  a.cache = (uint8_t *)cache, a.slots = slots;
  a.T = (int)T, a.H = H, a.D = D, a.G = G, a.shift = block_shift(BS);
  a.num_blocks = num_blocks;
  const int64_t waves = cache4_waves(step, T, H * G);
  const dim3 grid((unsigned)((waves + 3) / 4));
  const int64_t vec = 16 / eb;
  const bool aligned = (uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0 && k_st % vec == 0 &&
                       k_sh % vec == 0 && v_st % vec == 0 && v_sh % vec == 0;
  auto go = [&](auto dt, auto al, auto sp) {
    constexpr int DT = decltype(dt)::value;
    constexpr bool AL = decltype(al)::value, SP = decltype(sp)::value;
    if constexpr (APPEND) append_4bit_kernel<DT, AL, SP><<<grid, CACHE4_NT, 0, stream>>>(a, waves);
    else gather_4bit_kernel<DT, AL, SP><<<grid, CACHE4_NT, 0, stream>>>(a, waves);
  };
  auto by_step = [&](auto dt, auto al) {
    if (step) go(dt, al, std::true_type{});
    else go(dt, al, std::false_type{});
  };
  auto by_alignment = [&](auto dt) {
    if (aligned) by_step(dt, std::true_type{});
    else by_step(dt, std::false_type{});
  };
  if (dtype == VFL_FLOAT32) by_alignment(std::integral_constant<int, VFL_FLOAT32>{});
  else if (dtype == VFL_BFLOAT16) by_alignment(std::integral_constant<int, VFL_BFLOAT16>{});
  else by_alignment(std::integral_constant<int, VFL_FLOAT16>{});
  return launch_status(who);
}

}  // namespace

}  // namespace vfl

using namespace vfl;

extern "C" int vfl_reshape_and_cache_4bit(const void *key, const void *value,
                                          int64_t key_stride_token, int64_t key_stride_head,
                                          int64_t value_stride_token, int64_t value_stride_head,
                                          void *cache, const int64_t *slot_mapping,
                                          int64_t num_tokens, int num_heads, int head_dim,
                                          int block_size, int64_t num_blocks, int dtype,
                                          void *stream) {
  return move_4bit<true>("reshape_and_cache_4bit", key, value, key_stride_token, key_stride_head,
                         value_stride_token, value_stride_head, cache, slot_mapping, num_tokens,
                         num_heads, head_dim, block_size, num_blocks, dtype, (hipStream_t)stream);
}

extern "C" int vfl_gather_cache_4bit(const void *cache, const int64_t *slot_mapping, void *key,
                                     void *value, int64_t key_stride_token,
                                     int64_t key_stride_head, int64_t value_stride_token,
                                     int64_t value_stride_head, int64_t num_tokens, int num_heads,
                                     int head_dim, int block_size, int64_t num_blocks, int dtype,
                                     void *stream) {
  return move_4bit<false>("gather_cache_4bit", key, value, key_stride_token, key_stride_head,
                          value_stride_token, value_stride_head, const_cast<void *>(cache),
                          slot_mapping, num_tokens, num_heads, head_dim, block_size, num_blocks,
                          dtype, (hipStream_t)stream);
}
