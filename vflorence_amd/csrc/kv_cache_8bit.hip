// Appending keys and values to a paged cache held in e4m3, one scale per (block, head) for
// K and one for V (gfx950).
//
// A run is the tokens of a call, one after another, whose slots lie in one block (of a slot that
// comes twice, the later token).  Skipped tokens, whose slots lie outside the pool, are as if they
// were not in the call: a run goes on behind them.  Per run and head
//   a = max |x| over the run's finite values,  need = the smallest power of two with
//   a / need <= 448,  new = max(old, need)  (old = 0 where the run holds the block's offset
//   0: the block starts over, what it held is dropped)
//   held bytes <- rne(held * old / new),  the run's tokens <- rne(x / new)
// Powers of two make x / new exact, so each value is rounded once, and a block whose scale
// grows later loses nothing but what falls under e4m3's smallest step: no value's error
// grows with the number of appends, which any other scale would cost.  Infinities and NaN
// become NaN and leave the scale alone.
//
// What bounds it: prompts HBM (64 prompts of 256 to 1024 tokens x 16 heads, bf16: 53.3 us, 4.7
// TB/s read and written, of a copy's 5.1); steps their chain of slots, rows and stores (256 rows
// x 16 heads 4.7 us, 4 x 12 3.0 us).  A wave takes a block's tokens of a head, so that a tile is
// written whole; the heads of a block run on one XCD, whose L2 then writes the block's line of
// scales whole.  Magnitudes are compared as 16-bit patterns, two at a time, and the conversion
// takes the scale's exponent off: the same prompts ran in 57.0 us with values widened, compared
// and multiplied one by one (the vector units busy for 34 us of them, now for 20; cycles at 2.4
// GHz).
#include <stdio.h>

#include "e4m3.h"

namespace vfl {

int check_8bit_cache(const char *who, int dtype, int num_heads, int head_dim, int block_size,
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

// N consecutive elements as words of memory (16-byte loads, 8-byte ones for four 16-bit elements,
// where the rows are aligned for them).
template <int DT, bool ALIGNED, int N>
__device__ __forceinline__ void load_raw(const typename Elem<DT>::T *p, uint32_t *w) {
  constexpr int WORDS = N * (int)sizeof(typename Elem<DT>::T) / 4;
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (DT == VFL_FLOAT32) w[i] = __float_as_uint(p[i]);
      else w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    }
  } else if constexpr (WORDS % 4 == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 u = reinterpret_cast<const uint4 *>(p)[i / 4];
      w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
    }
  } else {
    static_assert(WORDS == 2, "a 16-bit quad");
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    w[0] = u.x, w[1] = u.y;
  }
}

// Magnitudes are compared as patterns without their sign, which order like the values, an
// infinity and then NaN above them all; 16-bit ones two at a time.
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
template <int DT> struct Pattern {
  static constexpr bool PAIRS = DT != VFL_FLOAT32;
  static constexpr uint32_t MAGNITUDE = PAIRS ? 0x7fff7fffu : 0x7fffffffu;
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
  template <int WORDS>
  static __device__ __forceinline__ void add(uint32_t &m, const uint32_t (&w)[WORDS]) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) m = largest(m, w[i] & MAGNITUDE);
  }
  // the same, what is not finite left out
  template <int WORDS>
  static __device__ __forceinline__ void add_finite(uint32_t &m, const uint32_t (&w)[WORDS]) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      uint32_t x = w[i] & MAGNITUDE;
      if constexpr (PAIRS) {
        if ((x & 0xffffu) >= INF) x &= 0xffff0000u;
        if ((x >> 16) >= INF) x &= 0xffffu;
      } else if (x >= INF) {
        x = 0;
      }
      m = largest(m, x);
    }
  }
  // over the wave, of both halves of a pair
  static __device__ __forceinline__ uint32_t over_wave(uint32_t m) {
    if constexpr (PAIRS) m = max(m >> 16, m & 0xffffu);
    int x = row_max16((int)m);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((int)a[0], (int)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (uint32_t)max((int)b[0], (int)b[1]);
  }
  static __device__ __forceinline__ float value(uint32_t pattern) {
    if constexpr (PAIRS) return Mfma<DT>::widen(pattern);
    else return __uint_as_float(pattern);
  }
};

// Four elements (as words of memory) over `scale`, a power of two whose exponent the conversion
// takes off, rounded to nearest even; an infinity or a NaN becomes NaN.
typedef short short2_t __attribute__((ext_vector_type(2)));
template <int DT> __device__ __forceinline__ uint32_t e4m3_pack(const uint32_t *w, float scale) {
  short2_t r = {0, 0};
  if constexpr (DT == VFL_FLOAT32) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __uint_as_float(w[0]), __uint_as_float(w[1]),
                                                 scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __uint_as_float(w[2]), __uint_as_float(w[3]),
                                                 scale, true);
  } else if constexpr (DT == VFL_BFLOAT16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w[0]), scale,
                                                  false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w[1]), scale,
                                                  true);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2_t, w[0]), scale,
                                                 false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2_t, w[1]), scale,
                                                 true);
  }
  return __builtin_bit_cast(uint32_t, r);
}

// Rows of four bytes to columns: word i of the result holds byte i of every word.
__device__ __forceinline__ void transpose_bytes(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // w0.0 w1.0 w0.1 w1.1
  const uint32_t b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);  // w0.2 w1.2 w0.3 w1.3
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// A workgroup takes the runs that begin among `window` tokens (up to 32), for one head; its NS
// waves take 64 dims each and share the maxima through LDS.  PARTS: 16-token parts of a block.
// K: lane = (token l / 4 of a part, dims 16 (l % 4) ..), a row's 16 values per 16-byte
// store.  V: lane = (tokens 4 (l / 16) .. + 3, dims 4 (l % 16) .. + 3), whose 16 bytes lie
// together in the token-interleaved pool.
template <int DT, bool ALIGNED, int NS, int PARTS>
__global__ __launch_bounds__(64 * NS) void append_8bit_kernel(
    const typename Elem<DT>::T *__restrict__ key, const typename Elem<DT>::T *__restrict__ value,
    int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, uint8_t *__restrict__ kc,
    uint8_t *__restrict__ vc, float *__restrict__ scales, const int64_t *__restrict__ slots,
    int T, int H, int D, int num_blocks, int window) {
  constexpr int BS = 16 * PARTS;
  using P = Pattern<DT>;
  constexpr int KW = 16 * (int)sizeof(typename Elem<DT>::T) / 4, VW = KW / 4;
  __shared__ uint32_t s_max[2][NS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t pos;
  int h;
  xcd_position(blockIdx.x, (unsigned)H, pos, h);  // a block's scales: written through one L2
  if (pos * window >= T) return;
  const int t0 = (int)pos * window;
  const int kd = 64 * wave + 16 * (lane & 3), vd = 64 * wave + 4 * (lane & 15);
  const bool k_in = kd < D, v_in = vd < D;

  // Lane l: block and offset of token t0 - back + l (block -1: skipped, or no token).  One load
  // covers the window, what lies before it and the rest of its last run.
  constexpr int SHIFT = PARTS == 1 ? 4 : 5;
  const uint64_t pool = (uint64_t)num_blocks << SHIFT;  // slots
  auto block_of = [&](int64_t slot) { return (uint64_t)slot < pool ? (int)(slot >> SHIFT) : -1; };
  const int back = window < 32 ? 32 - window : 1;
  const int tl = t0 - back + lane;
  const int64_t slot = slots[min(max(tl, 0), T - 1)];
  const uint64_t own = ((1ull << window) - 1) << back;  // the window's lanes
  const uint64_t none = __builtin_amdgcn_ballot_w64((unsigned)tl >= (unsigned)T);
  const int bl = (unsigned)tl < (unsigned)T ? block_of(slot) : -1;
  const int off = (int)(slot & (BS - 1));
  const uint64_t held = __builtin_amdgcn_ballot_w64(bl >= 0);
  // Where many skipped tokens follow one another: the first or last of the tokens from lo up to
  // hi (SCAN of them at most) that is not, or -1; eight loads in flight.  (16 heads: 1000 tokens
  // before 7192 skipped ones 9.5 us, 25 with one load; every other one of 256 rows skipped 4.8.)
  constexpr int SCAN = 512;
  auto find_held = [&](int lo, int hi, auto backwards) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(slots + lo), 0, __builtin_amdgcn_readfirstlane((hi - lo) * 8), 0x00020000);
    uint64_t x[SCAN / 64];
#pragma unroll
    for (int c = 0; c < SCAN / 64; ++c)
      x[c] = __builtin_bit_cast(
          uint64_t, __builtin_amdgcn_raw_buffer_load_b64(r, lane * 8 + c * 512, 0, 0));
    int found = -1;
#pragma unroll
    for (int i = 0; i < SCAN / 64; ++i) {  // the one to find comes last
      const int c = backwards.value ? i : SCAN / 64 - 1 - i;
      const uint64_t m = __builtin_amdgcn_ballot_w64(64 * c + lane < hi - lo && x[c] < pool);
      if (m) found = 64 * c + (backwards.value ? 63 - __builtin_clzll(m) : __builtin_ctzll(m));
    }
    return found < 0 ? -1 : lo + found;
  };
  int before = __shfl_up(bl, 1);  // block of the last token that is not skipped
  if (__builtin_expect((~(held | none) & (own | own >> 1)) != 0, 0)) {  // some are
    const uint64_t lower = held & ((1ull << lane) - 1);
    before = __shfl(bl, lower ? 63 - __builtin_clzll(lower) : 0);
    if ((held & own) && !(held & ((1ull << back) - 1))) {  // before the wave's first one
      int token = -1;
      for (int hi = t0 - back; token < 0 && hi > 0; hi -= SCAN)
        token = find_held(max(hi - SCAN, 0), hi, std::true_type{});
      const int first = token < 0 ? -1 : block_of(slots[token]);
      if (!lower) before = first;
    }
  }
  uint64_t leaders = __builtin_amdgcn_ballot_w64(bl >= 0 && bl != before) & own;

  for (; leaders; leaders &= leaders - 1) {
    const int at = __builtin_ctzll(leaders), t = t0 - back + at;
    const int blk = __builtin_amdgcn_readlane(bl, at);
    // n tokens side by side, and whether the run may go on behind skipped tokens or the wave's
    const uint64_t same = __builtin_amdgcn_ballot_w64(bl == blk);
    int n = __builtin_ctzll(~(same >> at));
    const bool on = at + n == 64 || !(((held | none) >> (at + n)) & 1);
    // lane o: the run's token that takes the block's offset o (its last one), from t on; last, the
    // run's last token (which is always taken)
    const int off0 = __builtin_amdgcn_readlane(off, at);
    int src = -1, last = n - 1;
    if (__builtin_expect(!on && __builtin_amdgcn_ballot_w64(lane > at && lane < at + n &&
                                                            off != off0 + lane - at) == 0,
                         1)) {
      src = lane >= off0 && lane < off0 + n ? lane - off0 : -1;  // in order
    } else {
      // which of the tokens i, i + 1, .. (offsets o of lanes `from` on) lie in the block, and
      // which end the run
      uint64_t mine = same >> at, ends = ((held | none) & ~same) >> at;
      int o = off, from = at, i = 0;
      n = 0;
      while (true) {
        if (ends) mine &= (ends & -ends) - 1;
        n += __builtin_popcountll(mine);
        for (; mine; mine &= mine - 1) {
          const int j = __builtin_ctzll(mine);
          if (__builtin_amdgcn_readlane(o, from + j) == lane) src = i + j;
          last = i + j;
        }
        if (ends) break;
        int next = -1;
        for (int lo = t + i + 64 - from; next < 0 && lo < T; lo += SCAN)
          next = find_held(lo, min(lo + SCAN, T), std::false_type{});
        if (next < 0) break;
        i = next - t;
        from = 0;
        const int64_t x = slots[min(next + lane, T - 1)];
        const int b = next + lane < T ? block_of(x) : -2;
        o = (int)(x & (BS - 1));
        mine = __builtin_amdgcn_ballot_w64(b == blk);
        ends = __builtin_amdgcn_ballot_w64(b != blk && b != -1);
      }
    }
    const bool fresh = __builtin_amdgcn_readlane(src, 0) >= 0;
    float *sc = scales + 2 * ((int64_t)blk * H + h);
    const float old_k = fresh ? 0.f : sc[0], old_v = fresh ? 0.f : sc[1];

    uint32_t kx[PARTS][KW], vx[PARTS][4][VW];
    int ks[PARTS], vs[PARTS][4];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      ks[p] = __shfl(src, 16 * p + (lane >> 2));
      if (!k_in) ks[p] = -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        vs[p][j] = __shfl(src, 16 * p + 4 * (lane >> 4) + j);
        if (!v_in) vs[p][j] = -1;
      }
    }
    auto k_row = [&](int p, int i) {
      load_raw<DT, ALIGNED, 16>(key + (t + i) * k_st + h * k_sh + (k_in ? kd : 0), kx[p]);
    };
    auto v_row = [&](int p, int j, int i) {
      load_raw<DT, ALIGNED, 4>(value + (t + i) * v_st + h * v_sh + (v_in ? vd : 0), vx[p][j]);
    };
    uint32_t km = 0, vm = 0;
    if (n > 1) {
      // every lane reads some row that is taken (what repeats changes no maximum): a load under
      // a condition would wait for the one before
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        k_row(p, ks[p] < 0 ? last : ks[p]);
#pragma unroll
        for (int j = 0; j < 4; ++j) v_row(p, j, vs[p][j] < 0 ? last : vs[p][j]);
      }
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        P::add(km, kx[p]);
#pragma unroll
        for (int j = 0; j < 4; ++j) P::add(vm, vx[p][j]);
      }
    } else {
      // one token: the few lanes that hold it (all lanes: 256 rows x 16 heads 7.2 us, not 5.2)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        if (ks[p] >= 0) {
          k_row(p, 0);
          P::add(km, kx[p]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (vs[p][j] >= 0) {
            v_row(p, j, 0);
            P::add(vm, vx[p][j]);
          }
      }
    }
    km = P::over_wave(km);
    vm = P::over_wave(vm);
    if (max(km, vm) >= P::INF) {  // wave-uniform, rare: the finite values alone
      km = vm = 0;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        if (n > 1 || ks[p] >= 0) P::add_finite(km, kx[p]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n > 1 || vs[p][j] >= 0) P::add_finite(vm, vx[p][j]);
      }
      km = P::over_wave(km);
      vm = P::over_wave(vm);
    }
    if constexpr (NS > 1) {
      __syncthreads();  // the previous run's maxima have been read
      if (lane == 0) s_max[0][wave] = km, s_max[1][wave] = vm;
      __syncthreads();  // and every wave has read the old scales
#pragma unroll
      for (int w = 0; w < NS; ++w) km = max(km, s_max[0][w]), vm = max(vm, s_max[1][w]);
    }
    const float new_k = fmaxf(old_k, e4m3_scale(P::value(km)));
    const float new_v = fmaxf(old_v, e4m3_scale(P::value(vm)));
    const bool all_k = fresh || new_k != old_k, all_v = fresh || new_v != old_v;
    const float ratio_k = old_k / new_k, ratio_v = old_v / new_v;

    const int64_t tile = ((int64_t)blk * H + h) * (BS * D);
    uint8_t *kt = kc + tile, *vt = vc + tile;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      uint4 *row = reinterpret_cast<uint4 *>(kt + (16 * p + (lane >> 2)) * D + kd);
      if (k_in && (ks[p] >= 0 || all_k)) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (ks[p] >= 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = e4m3_pack<DT>(kx[p] + i * VW, new_k);
        } else if (!fresh) {
          const uint4 u = *row;
          w[0] = e4m3_rescale(u.x, ratio_k), w[1] = e4m3_rescale(u.y, ratio_k);
          w[2] = e4m3_rescale(u.z, ratio_k), w[3] = e4m3_rescale(u.w, ratio_k);
        }
        *row = make_uint4(w[0], w[1], w[2], w[3]);
      }
      const bool any = vs[p][0] >= 0 || vs[p][1] >= 0 || vs[p][2] >= 0 || vs[p][3] >= 0;
      if (v_in && (any || all_v)) {
        uint4 *group = reinterpret_cast<uint4 *>(vt + ((4 * p + (lane >> 4)) * D + vd) * 4);
        uint32_t w[4] = {0, 0, 0, 0};
        if (!fresh) {
          const uint4 u = *group;
          w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
          if (all_v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = e4m3_rescale(w[i], ratio_v);
          }
        }
        uint32_t u[4], taken = 0;  // the bytes of the tokens that the run brings
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u[j] = e4m3_pack<DT>(vx[p][j], new_v);
          if (vs[p][j] >= 0) taken |= 0xffu << (8 * j);
        }
        transpose_bytes(u);  // dim i's values of the four tokens
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (w[i] & ~taken) | (u[i] & taken);
        *group = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (threadIdx.x == 0) {
      if (all_k) sc[0] = new_k;
      if (all_v) sc[1] = new_v;
    }
  }
}

template <int DT, bool ALIGNED, int PARTS, typename... A>
static void launch_append_steps(int steps, dim3 grid, hipStream_t stream, A... a) {
#define VFL_APPEND(NS) \
  append_8bit_kernel<DT, ALIGNED, NS, PARTS><<<grid, dim3(64 * NS), 0, stream>>>(a...)
  switch (steps) {
    case 1: VFL_APPEND(1); break;
    case 2: VFL_APPEND(2); break;
    case 3: VFL_APPEND(3); break;
    case 4: VFL_APPEND(4); break;
    default: VFL_APPEND(8); break;  // head size 512
  }
#undef VFL_APPEND
}

// Tokens whose runs a workgroup takes.  A decode step's tokens are runs of their own and want
// a workgroup each; a prompt's fill blocks.  The host does not see which they are: calls of up
// to 512 tokens (the most rows of a step that the projections take) get one, longer ones a
// block's.  Windows of 1 and of 16, us, bf16: steps of 256 and 512 rows x 16 heads 4.7 / 19.8 and
// 6.7 / 21.0, of 2048 rows 18.9 / 31.5; a prompt of 590 tokens x 12 heads 6.1 / 3.1, 64 prompts
// of 256 to 1024 tokens x 16 heads 159 / 52.9.
inline int append_window(int64_t T, int BS) { return T <= 512 ? 1 : BS; }

template <int DT>
static int launch_append(bool aligned, const void *key, const void *value, int64_t k_st,
                         int64_t k_sh, int64_t v_st, int64_t v_sh, void *kc, void *vc,
                         float *scales, const int64_t *slots, int64_t T, int H, int D, int BS,
                         int64_t num_blocks, hipStream_t stream) {
  using E = typename Elem<DT>::T;
  const int window = append_window(T, BS), steps = (D + 63) / 64;
  const int64_t groups = xcd_grid((T + window - 1) / window, H);
  if (!grid_fits(groups, 64 * (steps > 4 ? 8 : steps))) {
    set_error("reshape_and_cache_8bit: %lld tokens x %d heads exceed a launch", (long long)T, H);
    return VFL_E_INVALID;
  }
  const dim3 grid((unsigned)groups);
  auto go = [&](auto al, auto parts) {
    launch_append_steps<DT, decltype(al)::value, decltype(parts)::value>(
        steps, grid, stream, (const E *)key, (const E *)value, k_st, k_sh, v_st, v_sh,
        (uint8_t *)kc, (uint8_t *)vc, scales, slots, (int)T, H, D, (int)num_blocks,
        window);
  };
  using std::integral_constant;
  if (aligned) {
    if (BS == 16) go(integral_constant<bool, true>{}, integral_constant<int, 1>{});
    else go(integral_constant<bool, true>{}, integral_constant<int, 2>{});
  } else {
    if (BS == 16) go(integral_constant<bool, false>{}, integral_constant<int, 1>{});
    else go(integral_constant<bool, false>{}, integral_constant<int, 2>{});
  }
  return launch_status("reshape_and_cache_8bit");
}

}  // namespace vfl

using namespace vfl;

extern "C" int vfl_reshape_and_cache_8bit(const void *key, const void *value,
                                          int64_t key_stride_token, int64_t key_stride_head,
                                          int64_t value_stride_token, int64_t value_stride_head,
                                          void *k_cache, void *v_cache, float *kv_scales,
                                          const int64_t *slot_mapping, int64_t num_tokens,
                                          int num_heads, int head_dim, int block_size,
                                          int64_t num_blocks, int dtype, void *stream) {
  clear_error();
  const int st = check_8bit_cache("reshape_and_cache_8bit", dtype, num_heads, head_dim,
                                  block_size, num_blocks);
  if (st != VFL_OK) return st;
  if (num_tokens < 0 || (num_tokens + 1024) * num_heads > 2147483647LL) {
    set_error("reshape_and_cache_8bit: %lld tokens x %d heads", (long long)num_tokens, num_heads);
    return VFL_E_INVALID;
  }
  if (num_tokens == 0 || num_blocks == 0) return VFL_OK;
  if (!key || !value || !k_cache || !v_cache || !kv_scales || !slot_mapping) {
    set_error("reshape_and_cache_8bit: null pointer argument");
    return VFL_E_INVALID;
  }
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)kv_scales % 4 ||
      (uintptr_t)slot_mapping % 8 || (uintptr_t)key % elem_bytes(dtype) ||
      (uintptr_t)value % elem_bytes(dtype)) {
    set_error("reshape_and_cache_8bit: misaligned pointer (caches 16 bytes, others their "
              "element)");
    return VFL_E_INVALID;
  }
  const int64_t vec = 16 / elem_bytes(dtype);
  const bool aligned = (uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0 &&
                       key_stride_token % vec == 0 && key_stride_head % vec == 0 &&
                       value_stride_token % vec == 0 && value_stride_head % vec == 0;
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto dt) {
    return launch_append<decltype(dt)::value>(
        aligned, key, value, key_stride_token, key_stride_head, value_stride_token,
        value_stride_head, k_cache, v_cache, kv_scales, slot_mapping, num_tokens, num_heads,
        head_dim, block_size, num_blocks, s);
  };
  if (dtype == VFL_FLOAT32) return go(std::integral_constant<int, VFL_FLOAT32>{});
  if (dtype == VFL_BFLOAT16) return go(std::integral_constant<int, VFL_BFLOAT16>{});
  return go(std::integral_constant<int, VFL_FLOAT16>{});
}
