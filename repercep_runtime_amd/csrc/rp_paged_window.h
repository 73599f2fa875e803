// Attention of each sequence's last tokens over a paged cache, as its kernels
// share it: the arguments, and which keys a run of tokens sees.
//
// The rows of a kv head are its query heads' tokens, token by token: row r is
// token r / group, head r % group, so one tile of rows reads a key once for all
// heads that share it.  Token i of sequence b stands at p = len - qlen + i and
// sees key j where
//   j <= p,  and  p - j < window  or  j < sinks.
#pragma once

#include "rp_paged_mma.h"

namespace rp {

struct WindowArgs {
  const uint16_t* q;
  int64_t qsb, qsh, qss;
  const int32_t* lens;
  const int32_t* qlens;          // or null: S each
  float c;                       // |sm_scale| * log2(e)
  uint32_t flip;                 // the sign of sm_scale, for a pair of q's values
  float lift;                    // see base_lift
  int32_t window, sinks;         // window: 0x7fffffff where there is none
  uint16_t* out;
  int64_t osb, osh, oss;
  float* lse;                    // (B, H, S), or null
  int32_t H, group, S;
  int32_t tiles, splits;         // row tiles of a kv head, parts of a tile's keys
  int32_t room;                  // few_kernel: the whole batch's parts of a kv head and row tile
  int64_t groups;                // B * kv heads
  float* part;                   // (B, H, S, splits, D): the parts' weighted means
  float2* ml;                    // (B, H, S, splits): base (in powers of two), sum of weights
};

// How a call is launched.
struct WindowLaunch {
  int columns;                   // of 16 rows, few_kernel; 0: prompt_kernel
  int waves;                     // of prompt_kernel
  bool stream;                   // few_kernel: V past the caches
};

// The kernels for one type of q and of the cache, each in a source file of its
// own (they compile side by side).
template <int QT, int CT>
void launch_window(const WindowArgs& a, const PagedView& c, int64_t D, const WindowLaunch& l,
                   hipStream_t st);

namespace {

constexpr float kSlack = 8.0f;                  // powers of two, see rp_paged_prompt.h

// How far bases lie above the scores, in powers of two: of fp16 weights as far as
// their range asks (F16), of bf16 ones not at all, unless sums overflowed (AGAIN).
template <bool F16, bool AGAIN>
__device__ __forceinline__ float base_lift(const WindowArgs& a) {
  return F16 || AGAIN ? a.lift : 0.0f;
}

// A sequence's place: its length, its new tokens, the first one's position.
struct Place {
  int32_t n, m, first;
  __device__ __forceinline__ Place(const WindowArgs& a, int b) {
    n = max(0, a.lens[b]);
    m = a.qlens ? max(0, min(a.S, a.qlens[b])) : a.S;
    first = n - m;
  }
};

__device__ __forceinline__ bool sees(const WindowArgs& a, int32_t p, int32_t j) {
  return j <= p && (p - j < a.window || j < a.sinks);
}

// The keys that tokens at positions p0 .. p1 see between them, in tiles of T:
// those of the sinks, then those of the window (one run where they meet).
template <int T>
struct KeyTiles {
  int32_t lo, hi, sinks;         // keys [lo, hi) and [0, sinks)
  int32_t sink_tiles, first, count;

  __device__ __forceinline__ KeyTiles(const WindowArgs& a, const PagedView& c, int32_t p0,
                                      int32_t p1) {
    hi = (int32_t)max((int64_t)0, min((int64_t)p1 + 1, c.capacity()));
    lo = min(hi, max(0, max(0, p0) - a.window + 1));
    sinks = min(a.sinks, lo);
    first = lo / T;
    sink_tiles = (sinks + T - 1) / T;
    if (sink_tiles >= first) {
      if (sinks > 0) first = 0;
      sink_tiles = 0;
    }
    count = max(0, sink_tiles + (hi + T - 1) / T - first);
  }
  __device__ __forceinline__ int32_t key(int32_t tile) const {
    return (tile < sink_tiles ? tile : first + tile - sink_tiles) * T;
  }
  // Whether any of the tokens sees key j.
  __device__ __forceinline__ bool any(int32_t j) const { return j < hi && (j >= lo || j < sinks); }
};

// The keys that rows r0 .. r0 + n - 1 of a sequence see between them.
template <int T>
__device__ __forceinline__ KeyTiles<T> tile_keys(const WindowArgs& a, const PagedView& c,
                                                 const Place& pl, int r0, int n) {
  const int last = min(r0 + n, pl.m * a.group) - 1;
  return KeyTiles<T>(a, c, pl.first + r0 / a.group, last >= r0 ? pl.first + last / a.group : -1);
}

// 16-bit floats with infinities and NaNs as 0, a pair.
template <bool F16>
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
  if ((w & E) == E) w &= 0xffff0000u;
  if ((w >> 16 & E) == E) w &= 0x0000ffffu;
  return w;
}

template <bool F16>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (F16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
}

template <int QT>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (QT == kInF16) return pack_f16x2(a, b);
  else return f32_to_bf16_bits(a) | f32_to_bf16_bits(b) << 16;
}

}  // namespace
}  // namespace rp
