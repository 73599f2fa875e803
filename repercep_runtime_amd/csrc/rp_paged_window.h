// Attention of each sequence's last tokens over a paged cache, as its kernels
// share it: the arguments, which keys a run of tokens sees, and the join of
// parts.  Everything here has internal linkage.
//
// The rows of a kv head are its query heads' tokens, token by token: row r is
// token r / group, head r % group, so one tile of rows reads a key once for all
// heads that share it.  Token i of sequence b stands at p = len - qlen + i and
// sees key j where
//   j <= p,  and  p - j < window  or  j < sinks.
#pragma once

#include "rp_paged_mma.h"

namespace rp {
namespace {

struct WindowArgs {
  const uint16_t* q;
  int64_t qsb, qsh, qss;
  const int32_t* lens;
  const int32_t* qlens;          // or null: S each
  float c;                       // |sm_scale| * log2(e)
  uint32_t flip;                 // the sign of sm_scale, for a pair of q's values
  float lift;                    // how far bases lie above the scores, in powers of two
  int32_t window, sinks;         // window: 0x7fffffff where there is none
  uint16_t* out;
  int64_t osb, osh, oss;
  float* lse;                    // (B, H, S), or null
  int32_t H, group, S;
  int32_t tiles, splits;         // row tiles of a kv head, parts of a tile's keys
  int64_t groups;                // B * kv heads
  float* part;                   // (B, H, S, splits, D): the parts' weighted means
  float2* ml;                    // (B, H, S, splits): base (in powers of two), sum of weights
};

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

// 16-bit floats with infinities and NaNs as 0, a pair.
template <bool F16>
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
  if ((w & E) == E) w &= 0xffff0000u;
  if ((w >> 16 & E) == E) w &= 0x0000ffffu;
  return w;
}

template <int QT>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (QT == kInF16) return pack_f16x2(a, b);
  else return f32_to_bf16_bits(a) | f32_to_bf16_bits(b) << 16;
}

// Joins the parts of 256 / (64 W) rows, W waves a row: each part's mean counts
// by its sum about the largest base.  Half a wave or more takes a part's columns.
template <int QT, int D, int W>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a, int64_t rows) {
  constexpr int COLS = D / 4, GR = W * kWave / COLS;     // lanes a part, parts at a time
  __shared__ f32x4 sums[256];
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + threadIdx.x / (W * kWave);
  const int tid = threadIdx.x % (W * kWave), lane = threadIdx.x & (kWave - 1);
  const int col = tid % COLS, gr = tid / COLS;
  const bool in = row < rows;
  const int64_t bh = in ? row / a.S : 0;
  const int i = in ? (int)(row % a.S) : 0;
  const float2* ml = a.ml + (in ? row : 0) * a.splits;
  float base = neg_inf(), sum = 0.0f;
  for (int s = lane; s < a.splits; s += kWave)
    if (ml[s].y != 0.0f) base = fmaxf(base, ml[s].x);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) base = fmaxf(base, __shfl_xor(base, o, kWave));
  const float b0 = base == neg_inf() ? 0.0f : base;
  for (int s = lane; s < a.splits; s += kWave)
    if (ml[s].y != 0.0f) sum += ml[s].y * __builtin_amdgcn_exp2f(ml[s].x - b0);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.part + (in ? row : 0) * a.splits * D) + col;
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = gr; s < a.splits; s += GR) {
    const float2 p = ml[s];
    const f32x4 y = part[(int64_t)s * COLS];
    const float f = p.y * __builtin_amdgcn_exp2f(p.x - b0) * inv;
    // a part without keys wrote nothing
    if (p.y != 0.0f) x += y * f;
  }
  sums[threadIdx.x] = x;
  __syncthreads();
  if (gr != 0 || !in) return;
#pragma unroll
  for (int g = 1; g < GR; ++g) x += sums[threadIdx.x + g * COLS];
  const int64_t b = bh / a.H, h = bh % a.H;
  uint16_t* out = a.out + b * a.osb + h * a.osh + (int64_t)i * a.oss + 4 * col;
  if (sum == 0.0f) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  *reinterpret_cast<u32x2*>(out) = u32x2{pack_out<QT>(x[0], x[1]), pack_out<QT>(x[2], x[3])};
  if (col == 0 && a.lse)
    a.lse[row] = sum == 0.0f ? neg_inf() : (b0 + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace
}  // namespace rp
