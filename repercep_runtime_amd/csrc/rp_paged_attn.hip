// Attention of one new token per sequence over a paged key-value cache.
//
// A call reads every attended row of K and V once per kv head and does
// 4 * (H / Hkv) * D operations with a row's pair, so its floor is the cache's
// bytes; the kernel is built to keep loads in flight.
//
// * Products run on the matrix cores (16x16x32) although a decoder has few
//   query heads per kv head: the 16 columns are the query heads of one kv
//   head, unused ones idle, and 32 keys take D / 32 * 2 + D / 16 * 2
//   instructions, far below what their bytes take to arrive.  In S^T = K Q^T
//   a lane ends up with the scores of one head (its column) and the eight keys
//   4 g + 0..3 and 16 + 4 g + 0..3 of a step's 32 (g = lane / 16).  O^T = V^T P^T
//   sums over those same keys if lane group g brings V's rows in that order, so
//   P goes from the first product to the second inside its lane: nothing
//   passes through LDS in the loop.
// * V's operand needs eight keys of one column in a register quad.  A lane
//   loads D / 16 columns of each of its eight rows and transposes them with
//   byte permutes (v_perm_b32), one per pair of values.
// * P enters the second product as the sum of three bf16 numbers, which is the
//   fp32 weight exactly, however small it is beside the largest; fp16 would end
//   at 2^-24.  An fp16 V is the exact sum of two bf16 numbers, its first eight
//   bits and the other three.  So a value takes three instructions, an fp16 one
//   six (with two fp16 parts of a weight, 32 long fp16 sequences took 251 us and
//   640 keys 10.1, now 259 and 12.3); the products are idle otherwise.
// * The running maximum is lazy: a lane's scores are weighed against its
//   column's base, and only when one exceeds it by 2^8 (kSlack) does the wave
//   agree on a new base and rescale.  Every lane of a column holds the same
//   base, and the final sums are exact about any base.  Sums about a base of
//   values near fp32's largest may overflow where their mean does not, and a
//   zero part of a weight makes NaN of an infinite value: a wave whose sums are
//   not finite takes its keys again, about a base so high that the weights' sum
//   stays below 1 and with no part zero.  Waves, chunks and parts are joined as
//   means, which fit.
// * K rows of step i + 1 are requested as soon as step i's first product has
//   read its registers, V rows after the second one, so a wave always has a
//   step's K or V on its way.
//
// Bound by HBM where the cache is large: 64 sequences of 2048 to 16384 keys, 32
// heads on 8 of 128, bf16, 2.4 GB in 445 us (5.4 TB/s), one of 131071 e4m3fn keys
// in 46 us and 5 of the join; by the latencies of a wave's steps where it is
// small: 640 keys of 32 heads in 11.7 us.
//
// The keys of a (sequence, kv head) are split into chunks of equal size over
// workgroups, a chunk over a workgroup's waves; waves join through LDS,
// chunks through fp32 partial sums and join_kernel.  A sequence longer than
// expected takes several rounds of its workgroups.

#include "rp_paged_mma.h"

namespace rp {
namespace {

constexpr int kDWaves = 4;
constexpr int kDThreads = kDWaves * kWave;
constexpr int kMaxChunk = kDWaves * 1024;       // a wave holds 64 tiles' pages in one register
constexpr int kJThreads = 256;
constexpr int kMaxSplits = 1024;
constexpr float kSlack = 8.0f;                  // powers of two

struct DecodeArgs {
  const uint16_t* q;
  int64_t qsb, qsh;
  const int32_t* lens;
  float c;                       // sm_scale * log2(e)
  float lift;                    // how far the high base lies above the scores, in powers of two
  uint16_t* out;
  int64_t osb, osh;
  float* lse;
  float* weights;
  int64_t wsb, wsh;
  int32_t H, group, tiles;       // query heads, per kv head, 16-head tiles per kv head
  int32_t splits, chunk;
  float* part;                   // (B, H, splits, D): the part's weighted means
  float2* ml;                    // (B, H, splits): base (in powers of two), sum of weights
  float* scores;                 // (B, H, score_ld): scores in powers of two, for the key weights
  int64_t score_ld;
};

// Weights a, b as three packed bf16 numbers each, eight bits at a time: exact.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t* to) {
  to[0] = pack_cut(a, b);
  a -= bf16_cut(a);
  b -= bf16_cut(b);
  to[1] = pack_cut(a, b);
  to[2] = pack_cut(a - bf16_cut(a), b - bf16_cut(b));
}

// Two fp16 values as packed bf16 numbers `hi` (toward zero) and the rest `lo`, both exact.
__device__ __forceinline__ void split_f16(uint32_t w, uint32_t* hi, uint32_t* lo) {
  const float a = f16_to_f32(w & 0xffffu), b = f16_to_f32(w >> 16);
  *hi = pack_cut(a, b);
  // the rest is 2^8 at most; what an infinity or a NaN leaves counts for nothing beside `hi`
  *lo = pack_cut(fminf(a - bf16_cut(a), 512.0f), fminf(b - bf16_cut(b), 512.0f));
}

// One wave's state over its keys.  PG16: pages hold 16 rows or more, so each
// half of a step lies in one page.
template <int QT, int CT, int D, bool PG16, bool STREAM>
struct Wave : StepRows<QT == kInF16, CT, D, STREAM> {
  typedef StepRows<QT == kInF16, CT, D, STREAM> Rows;
  using Rows::FP8, Rows::EB, Rows::NT, Rows::DPL, Rows::VW;
  using Rows::c, Rows::lane, Rows::m, Rows::g, Rows::head, Rows::kr, Rows::vr, Rows::kscale,
      Rows::vscale, Rows::v_col, Rows::k_frag;
  static constexpr bool QF16 = QT == kInF16;          // the first product's type; the second's is bf16
  static constexpr bool VF16 = CT == RP_CACHE_F16;

  const DecodeArgs& a;
  const int32_t* table;
  int32_t pages;                 // lane i: page of 16-key tile i of this wave's range (PG16)
  int k0;
  u32x4 q[NT];
  f32x4 acc[DPL];
  float base, sum, lift;
  uint32_t least;                // the least a positive weight's second and third part may be
  float* score_row;

  __device__ __forceinline__ Wave(const DecodeArgs& a_, const PagedView& c_) : Rows(c_), a(a_) {}

  __device__ __forceinline__ void load_q(const uint16_t* src, bool live) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int d = FP8 && D >= 64 ? 64 * (t / 2) + 16 * g + 8 * (t % 2) : 32 * t + 8 * g;
      q[t] = live ? *reinterpret_cast<const u32x4*>(src + d) : u32x4{0u, 0u, 0u, 0u};
    }
  }

  __device__ __forceinline__ void reset(float lift_) {
    base = neg_inf();
    sum = 0.0f;
    lift = lift_;
    // For an infinity in V each part of a positive weight has to be positive, or
    // 0 * inf makes NaN of it (e4m3fn has none): 2^-126 where it is 0.
    least = lift_ == 0.0f ? 0u : 0x00800080u;
#pragma unroll
    for (int j = 0; j < DPL; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Whether any sum of a live column is infinite or NaN.
  __device__ __forceinline__ bool overflown(bool live) const {
    f32x4 z = acc[0] * 0.0f;
#pragma unroll
    for (int j = 1; j < DPL; ++j) z += acc[j] * 0.0f;
    const float y = (z[0] + z[1]) + (z[2] + z[3]);
    return __any(live && y != y);
  }

  __device__ __forceinline__ void begin(int from) {
    k0 = from;
    if constexpr (PG16) pages = paged_page(c, table, (int64_t)from + 16 * lane);
  }

  __device__ __forceinline__ int32_t tile_page(int k, int half) const {
    return __builtin_amdgcn_readlane(pages, ((k - k0) >> 4) + half);
  }

  __device__ __forceinline__ void load_k(int k) {
    if constexpr (PG16) {
      // a page that is none is read as page 0 and masked
#pragma unroll
      for (int half = 0; half < 2; ++half) this->load_k16(half, max(tile_page(k, half), 0), k + 16 * half);
    } else {
      this->load_k_any([&](int j) { return max(paged_page(c, table, j), 0); }, k);
    }
  }

  __device__ __forceinline__ void load_v(int k) {
    if constexpr (PG16) {
#pragma unroll
      for (int half = 0; half < 2; ++half) this->load_v16(half, max(tile_page(k, half), 0), k + 16 * half);
    } else {
      this->load_v_any([&](int j) { return max(paged_page(c, table, j), 0); }, k);
    }
  }

  // Which of the lane's eight keys exist.
  __device__ __forceinline__ uint32_t present(int k, int end) const {
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = PG16 ? tile_page(k, e / 4) >= 0 : paged_page(c, table, this->key(k, e)) >= 0;
      if (in && this->key(k, e) < end) mask |= 1u << e;
    }
    return mask;
  }

  // A pair of columns of eight rows, times the weights, into two sums.
  __device__ __forceinline__ static void add_columns(const uint32_t* w, const u32x4* w3,
                                                     f32x4* to) {
    u32x4 f0, f1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f0[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
      f1[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
    }
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      to[0] = mma<false>(f0, w3[e], to[0]);
      to[1] = mma<false>(f1, w3[e], to[1]);
    }
  }

  // Keys [k, k + 32) of which those below `end` exist; `more`: another step follows.
  template <bool MORE>
  __device__ __forceinline__ void step(int k, int end) {
    f32x4 s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) s[half] = mma<QF16>(k_frag(half, t), q[t], s[half]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s[e / 4][e % 4] * a.c;
      if constexpr (FP8) x[e] *= kscale[e / 4][e % 4];
    }
    bool whole;
    if constexpr (PG16)
      whole = k + kStep <= end && tile_page(k, 0) >= 0 && tile_page(k, 1) >= 0;
    else
      whole = false;
    uint32_t mask = 0xffu;
    if (!whole) {
      mask = present(k, end);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = mask >> e & 1 ? x[e] : neg_inf();
    }
    if constexpr (MORE) load_k(k + kStep);
    if (score_row) {
      *reinterpret_cast<f32x4*>(score_row + k + 4 * g) = f32x4{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<f32x4*>(score_row + k + 16 + 4 * g) = f32x4{x[4], x[5], x[6], x[7]};
    }
    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                      fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (__any(top > base + (kSlack - lift))) {
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float next = fmaxf(base, top + lift);
      const float r = next == neg_inf() ? 1.0f : __builtin_amdgcn_exp2f(base - next);
      sum *= r;
#pragma unroll
      for (int j = 0; j < DPL; ++j) acc[j] *= r;
      base = next;
    }
    // a column that has seen no score yet weighs about 0: exp2(-inf) is 0
    const float b = base == neg_inf() ? 0.0f : base;
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(x[e] - b);
    sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    if constexpr (FP8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] *= vscale[e / 4][e % 4];
    }
    if (!whole) {
      // what is no row may hold anything: neither it nor its scale takes part
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = mask >> e & 1;
        p[e] = in ? p[e] : 0.0f;
#pragma unroll
        for (int i = 0; i < VW; ++i) vr[e][i] = in ? vr[e][i] : 0u;
      }
    }
    u32x4 w3[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t t[3];
      split_pair(p[2 * i], p[2 * i + 1], t);
      if constexpr (!FP8) {
        const uint32_t f = pk_min_u16(t[0], least);
        t[1] = pk_max_u16(t[1], f);
        t[2] = pk_max_u16(t[2], f);
      }
#pragma unroll
      for (int e = 0; e < 3; ++e) w3[e][i] = t[e];
    }
#pragma unroll
    for (int j = 0; j < DPL; j += 2) {
      // the pair of columns j, j + 1 of each row as bf16 values
      uint32_t w[8], rest[VF16 ? 8 : 1];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (VF16) split_f16(vr[e][j / 2], &w[e], &rest[e]);
        else if constexpr (!FP8) w[e] = vr[e][j / 2];
        else w[e] = j % 4 ? codes_to_16<false, true>(vr[e][j / 4]) : codes_to_16<false, false>(vr[e][j / 4]);
      }
      add_columns(w, w3, &acc[j]);
      if constexpr (VF16) add_columns(rest, w3, &acc[j]);
    }
    if constexpr (MORE) load_v(k + kStep);
  }
};

template <int QT, int CT, int D, bool PG16, bool STREAM>
__global__ __launch_bounds__(kDThreads) void attend_kernel(DecodeArgs a, PagedView c) {
  typedef Wave<QT, CT, D, PG16, STREAM> W;
  __shared__ f32x4 sacc[kDWaves / 2][W::DPL][kWave];
  __shared__ float sbase[kDWaves][16], ssum[kDWaves][16];
  const int split = blockIdx.x, b = blockIdx.z;
  const int kv = blockIdx.y / a.tiles, tile = blockIdx.y % a.tiles;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n = (int)paged_len(c, a.lens[b]);
  // a part beyond the sequence's end has nothing to say, and join_kernel does
  // not ask it; the first part always answers
  if (split > 0 && (int64_t)split * a.chunk >= n) return;
  W w(a, c);
  w.place(threadIdx.x & (kWave - 1), kv);
  w.table = c.table + b * c.table_stride;
  const int first = tile * 16;                         // of the group's query heads
  const bool live = first + w.m < a.group;
  const int h = kv * a.group + first + w.m;
  w.load_q(a.q + b * a.qsb + (int64_t)h * a.qsh, live);
  w.score_row = a.scores && live ? a.scores + ((int64_t)b * a.H + h) * a.score_ld : nullptr;

  for (float lift = 0.0f;; lift = a.lift) {
    w.reset(lift);
    for (int64_t c0 = (int64_t)split * a.chunk; c0 < n; c0 += (int64_t)a.splits * a.chunk) {
      const int rem = (int)min((int64_t)a.chunk, n - c0);
      const int per = ((rem + kDWaves - 1) / kDWaves + kStep - 1) / kStep * kStep;
      const int from = (int)c0 + wave * per, end = min(from + per, (int)c0 + rem);
      if (from >= end) continue;
      w.begin(from);
      w.load_k(from);
      w.load_v(from);
      int k = from;
      for (; k + kStep < end; k += kStep) w.template step<true>(k, end);
      w.template step<false>(k, end);
    }
    if (lift != 0.0f || !w.overflown(live)) break;
  }

  // the waves' parts about one base
  w.sum += __shfl_xor(w.sum, 16, kWave);
  w.sum += __shfl_xor(w.sum, 32, kWave);
  if (w.g == 0) {
    sbase[wave][w.m] = w.base;
    ssum[wave][w.m] = w.sum;
  }
  __syncthreads();
  float base = sbase[0][w.m];
#pragma unroll
  for (int i = 1; i < kDWaves; ++i) base = fmaxf(base, sbase[i][w.m]);
  const float b0 = base == neg_inf() ? 0.0f : base;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kDWaves; ++i) sum += ssum[i][w.m] * __builtin_amdgcn_exp2f(sbase[i][w.m] - b0);
  const float r = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(w.base - b0) / sum;
#pragma unroll
  for (int j = 0; j < W::DPL; ++j) w.acc[j] *= r;
#pragma unroll
  for (int half = kDWaves / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int j = 0; j < W::DPL; ++j) sacc[wave - half][j][w.lane] = w.acc[j];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int j = 0; j < W::DPL; ++j) w.acc[j] += sacc[wave][j][w.lane];
    }
    __syncthreads();
  }
  if (wave != 0 || !live) return;
  const int64_t bh = (int64_t)b * a.H + h;
  if (a.splits > 1) {
    float* part = a.part + (bh * a.splits + split) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < W::DPL; ++j) part[W::column(4 * w.g + i, j)] = w.acc[j][i];
    if (w.g == 0) a.ml[bh * a.splits + split] = float2{base, sum};
    return;
  }
  uint16_t* out = a.out + b * a.osb + h * a.osh;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < W::DPL; ++j) {
      const float x = sum == 0.0f ? 0.0f : w.acc[j][i];
      out[W::column(4 * w.g + i, j)] = QT == kInF16
          ? __builtin_bit_cast(uint16_t, (_Float16)x) : (uint16_t)f32_to_bf16_bits(x);
    }
  if (w.g == 0) {
    if (a.lse) a.lse[bh] = sum == 0.0f ? neg_inf() : (base + __builtin_amdgcn_logf(sum)) * kLn2;
    if (a.ml) a.ml[bh] = float2{base, sum};
  }
}

// Joins the parts of a (sequence, query head), or adds the key weights.
//
// Blocks with blockIdx.x < heads_x join: the parts' bases and sums are read a
// part a thread and turned into factors, then D / 4 threads take a part's
// columns and the block 1024 / D parts at a time.  The others add the key
// weights of up to 1024 keys of a kv head from the stored scores.
struct JoinShared {
  float factor[kMaxSplits];
  float red[2][kJThreads / kWave];
};

// The parts' joint base and sum, and in sh.factor each part's sum about that
// base.  Called by the whole block.
__device__ __forceinline__ float2 join_parts(const float2* ml, int parts, JoinShared& sh) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  constexpr int PER = kMaxSplits / kJThreads;
  float2 p[PER];
  float base = neg_inf();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = threadIdx.x + i * kJThreads;
    p[i] = at < parts ? ml[at] : float2{neg_inf(), 0.0f};
    base = fmaxf(base, p[i].x);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) base = fmaxf(base, __shfl_xor(base, o, kWave));
  if (lane == 0) sh.red[0][wave] = base;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJThreads / kWave; ++w) base = fmaxf(base, sh.red[0][w]);
  const float b0 = base == neg_inf() ? 0.0f : base;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = threadIdx.x + i * kJThreads;
    const float f = p[i].y * __builtin_amdgcn_exp2f(p[i].x - b0);
    if (at < parts) sh.factor[at] = f;
    sum += f;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  if (lane == 0) sh.red[1][wave] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kJThreads / kWave; ++w) sum += sh.red[1][w];
  return float2{b0, sum};
}

// The same by one wave: base and sum.
__device__ __forceinline__ float2 wave_parts(const float2* ml, int parts, int lane) {
  float base = neg_inf(), sum = 0.0f;
  for (int i = lane; i < parts; i += kWave) base = fmaxf(base, ml[i].x);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) base = fmaxf(base, __shfl_xor(base, o, kWave));
  const float b0 = base == neg_inf() ? 0.0f : base;
  for (int i = lane; i < parts; i += kWave) sum += ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - b0);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  return float2{b0, sum};
}

template <int QT, int D>
__global__ __launch_bounds__(kJThreads) void join_kernel(DecodeArgs a, PagedView c, int heads_x) {
  __shared__ JoinShared sh;
  const int b = blockIdx.y;
  const int n = (int)paged_len(c, a.lens[b]);
  const int parts = (int)max((int64_t)1, min((int64_t)a.splits, ((int64_t)n + a.chunk - 1) / a.chunk));
  if ((int)blockIdx.x < heads_x) {
    constexpr int COLS = D / 4, GR = kJThreads / COLS;
    __shared__ f32x4 group_sum[GR][COLS];
    const int h = blockIdx.x;
    const int64_t bh = (int64_t)b * a.H + h;
    const float2 t = join_parts(a.ml + bh * a.splits, parts, sh);
    const int d = threadIdx.x % COLS, gr = threadIdx.x / COLS;
    const f32x4* part = reinterpret_cast<const f32x4*>(a.part + bh * a.splits * D) + d;
    const float inv = t.y == 0.0f ? 0.0f : 1.0f / t.y;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = gr; i < parts; i += GR) x += part[(int64_t)i * COLS] * (sh.factor[i] * inv);
    group_sum[gr][d] = x;
    __syncthreads();
    if (gr != 0) return;
#pragma unroll
    for (int i = 1; i < GR; ++i) x += group_sum[i][d];
    uint16_t* out = a.out + b * a.osb + h * a.osh + 4 * d;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = t.y == 0.0f ? 0.0f : x[e];
      out[e] = QT == kInF16 ? __builtin_bit_cast(uint16_t, (_Float16)y) : (uint16_t)f32_to_bf16_bits(y);
    }
    if (threadIdx.x == 0 && a.lse)
      a.lse[bh] = t.y == 0.0f ? neg_inf() : (t.x + __builtin_amdgcn_logf(t.y)) * kLn2;
    return;
  }
  const int blocks = (gridDim.x - heads_x) / c.heads;
  const int kv = (blockIdx.x - heads_x) / blocks, block = (blockIdx.x - heads_x) % blocks;
  const int64_t j = ((int64_t)block * kJThreads + threadIdx.x) * 4;
  if ((int64_t)block * kJThreads * 4 >= n) return;
  // sixteen heads at a time: a wave finds the base and sum of every fourth
  // one, then every thread weighs its four keys under each
  float2* stat = reinterpret_cast<float2*>(sh.factor);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t bh0 = (int64_t)b * a.H + kv * a.group;
  float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < a.group; i0 += 16) {
    const int heads = min(16, a.group - i0);
    __syncthreads();
    for (int i = wave; i < heads; i += kJThreads / kWave) {
      const float2 t = wave_parts(a.ml + (bh0 + i0 + i) * a.splits, parts, lane);
      if (lane == 0) stat[i] = float2{t.x, t.y == 0.0f ? 0.0f : 1.0f / t.y};
    }
    __syncthreads();
    if (j < n) {
      const float* s = a.scores + (bh0 + i0) * a.score_ld + j;
#pragma unroll 4
      for (int i = 0; i < heads; ++i) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(s + (int64_t)i * a.score_ld);
        const float2 t = stat[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] += __builtin_amdgcn_exp2f(x[e] - t.x) * t.y;
      }
    }
  }
  float* to = a.weights + b * a.wsb + kv * a.wsh + j;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e < n) to[e] += w[e];
}

// How a call's keys are split: chunks of `chunk` keys, `splits` of them at
// most (the last ones empty for shorter sequences).
struct Plan {
  int32_t splits, chunk;
};

// * Key weights need join_kernel anyway, so their calls split down to 1024
//   workgroups, four a CU, which evens out ragged lengths (8 sequences of 1 to
//   4100 keys: a seventh less time than on 512).
// * Else a second launch is worth its 4 us where a workgroup's keys take
//   longer than that: not up to 384 KB of them (640 keys of 128: 12.5 us a call
//   unsplit, 16.9 in five parts; captured, where launches cost less, 11.3 and
//   9.8), nor with two workgroups a CU, what its
//   registers hold, already (16 sequences x 32 heads: 17 us unsplit, 23 in two
//   parts).  Fewer are split to no more than those 512: 131071 keys in 8 heads
//   take 55 us on 512 workgroups, 58 on 1024, 64 on 2048.
// * More than 512 are split where the last round of them would leave most CUs
//   without work (a third of the workgroups, two of three CUs, still take most
//   of the card's rate), and so are 257 to 384, of which some CUs get two and
//   the others one: 264 heads of 4096 keys 120 -> 95 us in three parts, 320
//   129 -> 111 us; 416 heads 140 us unsplit, 151 in two parts; 520 heads
//   203 -> 183 us in eight.  Parts of less than 256 KB lose more than they
//   gain: 520 heads of 900 keys 46 us unsplit, 56 in eight parts.
inline Plan decode_plan(int64_t groups, int64_t keys, int64_t key_bytes, bool weights) {
  constexpr int64_t kUnit = kDWaves * kStep, kRound = 512;
  int64_t splits = 1;
  if (weights) {
    splits = (2 * kRound + groups - 1) / groups;
  } else if (keys * key_bytes > 384 << 10) {
    splits = kRound / groups;
    if (splits == 0 || (groups > kRound / 2 && groups <= kRound * 3 / 4)) {
      splits = 8;                                  // a short last round at least
      for (int64_t s = groups < kRound ? 2 : 1; s <= 4; ++s) {
        const int64_t last = groups * s % kRound;
        if (last == 0 || last >= kRound / 3) {
          splits = s;
          break;
        }
      }
      splits = max((int64_t)1, min(splits, keys * key_bytes / (256 << 10)));
    }
  }
  const int64_t most = (keys + kUnit - 1) / kUnit;
  if (splits > most) splits = most;
  if (splits > kMaxSplits) splits = kMaxSplits;
  int64_t chunk = ((keys + splits - 1) / splits + kUnit - 1) / kUnit * kUnit;
  if (chunk > kMaxChunk) chunk = kMaxChunk;        // a workgroup takes several chunks
  splits = min(splits, (keys + chunk - 1) / chunk);
  return Plan{(int32_t)splits, (int32_t)chunk};
}

// Calls that read more than the 256 MB last-level cache, of which nothing would
// be left by the next call, read past it (a page that sequences share counts
// once for each, which is too much for long prompts with many candidates): V's
// rows, whose lines one
// instruction takes whole, with the non-temporal hint.  One state of 8 heads
// of 128, per call: 403 MB 71 us against 84, 806 MB 130 against 144, e4m3fn
// 554 MB 87 against 102; 202 MB 40.5 us against 38.7 without the hint.  K's
// rows, taken a half line at a time, are slower with it at every size.
constexpr int64_t kStreamBytes = 256 << 20;

struct Layout {
  Plan plan;
  bool stream;
  int64_t score_ld;
  size_t ml, part, scores, total;      // byte offsets
};

inline Layout decode_layout(int64_t B, int64_t H, const rp_paged_cache* c, int64_t max_seq_len,
                            bool weights) {
  const int64_t cap = c->max_pages * c->page_size, group = H / c->heads;
  const int64_t keys = max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
  Layout l;
  const int64_t key_bytes =
      2 * (c->head_dim * cache_elem_bytes(c->dtype) + (c->dtype == RP_CACHE_E4M3 ? 4 : 0));
  l.plan = decode_plan(B * c->heads * ((group + 15) / 16), keys, key_bytes, weights);
  l.stream = B * c->heads * keys * key_bytes > kStreamBytes;
  auto up = [](int64_t x) { return (size_t)((x + 255) / 256 * 256); };
  const bool split = l.plan.splits > 1;
  // whole steps are written, the last one past the capacity
  l.score_ld = (cap + kStep - 1) / kStep * kStep;
  l.ml = 0;
  l.part = l.ml + (split || weights ? up(B * H * l.plan.splits * 8) : 0);
  l.scores = l.part + (split ? up(B * H * l.plan.splits * c->head_dim * 4) : 0);
  l.total = l.scores + (weights ? up(B * H * l.score_ld * 4) : 0);
  return l;
}

template <int QT, int CT, int D>
void launch_decode_d(const DecodeArgs& a, const PagedView& c, int64_t B, bool stream,
                     hipStream_t st) {
  const dim3 grid((unsigned)a.splits, (unsigned)(c.heads * a.tiles), (unsigned)B);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kDThreads), 0, st, a, c);
  };
  if (c.shift < 4) go(attend_kernel<QT, CT, D, false, false>);
  else if (stream) go(attend_kernel<QT, CT, D, true, true>);
  else go(attend_kernel<QT, CT, D, true, false>);
  const int heads_x = a.splits > 1 ? a.H : 0;
  const int64_t blocks = a.weights ? (c.capacity() + 4 * kJThreads - 1) / (4 * kJThreads) : 0;
  if (heads_x + blocks > 0)
    hipLaunchKernelGGL((join_kernel<QT, D>), dim3((unsigned)(heads_x + blocks * c.heads), (unsigned)B),
                       dim3(kJThreads), 0, st, a, c, heads_x);
}

template <int QT, int CT>
void launch_decode(const DecodeArgs& a, const PagedView& c, int64_t B, int64_t D, bool stream,
                   hipStream_t st) {
  if (D == 32) launch_decode_d<QT, CT, 32>(a, c, B, stream, st);
  else if (D == 64) launch_decode_d<QT, CT, 64>(a, c, B, stream, st);
  else if (D == 128) launch_decode_d<QT, CT, 128>(a, c, B, stream, st);
  else launch_decode_d<QT, CT, 256>(a, c, B, stream, st);
}

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" size_t rp_paged_attn_workspace_bytes(int64_t B, int64_t H, const rp_paged_cache* cache,
                                                int64_t max_seq_len, int with_key_weights) {
  // sizes that the call refuses need none
  if (!cache || B <= 0 || B > 65535 || H <= 0 || H > 65535 || cache->heads <= 0 ||
      cache->heads > H || cache->page_size <= 0 || cache->max_pages <= 0 ||
      cache->max_pages > (1 << 30) / cache->page_size || cache->head_dim <= 0 ||
      cache->head_dim > 256 || max_seq_len < 0)
    return 0;
  return decode_layout(B, H, cache, max_seq_len, with_key_weights != 0).total;
}

extern "C" int rp_paged_attn_decode(const void* q, int q_dtype, int64_t B, int64_t H, int64_t qsb,
                                    int64_t qsh, const rp_paged_cache* cache,
                                    const int32_t* seq_lens, float sm_scale, void* out,
                                    int64_t osb, int64_t osh, float* lse, float* key_weights,
                                    int64_t wsb, int64_t wsh, int64_t max_seq_len,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !out || !seq_lens) {
    rp_set_error("paged_attn_decode: null pointer");
    return RP_ERR_INVALID_ARGUMENT;
  }
  PagedView c;
  const int rc = paged_view("paged_attn_decode", cache, &c);
  if (rc != RP_OK) return rc;
  if (q_dtype != RP_DTYPE_BF16 && q_dtype != RP_DTYPE_F16) {
    rp_set_error("paged_attn_decode: unknown q dtype %d", q_dtype);
    return RP_ERR_INVALID_ARGUMENT;
  }
  const bool fp8 = cache->dtype == RP_CACHE_E4M3;
  if (!fp8 && (cache->dtype == RP_CACHE_F16) != (q_dtype == RP_DTYPE_F16)) {
    rp_set_error("paged_attn_decode: a 16-bit cache has q's dtype");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B <= 0 || H <= 0 || H % cache->heads != 0 || max_seq_len < 0) {
    rp_set_error("paged_attn_decode: needs B > 0, H a multiple of the cache's %lld heads and "
                 "max_seq_len >= 0 (B=%lld H=%lld)", (long long)cache->heads, (long long)B,
                 (long long)H);
    return RP_ERR_INVALID_ARGUMENT;
  }
  const float c2 = sm_scale * kLog2e;              // scores in powers of two
  if (!(c2 - c2 == 0.0f)) {
    rp_set_error("paged_attn_decode: sm_scale and sm_scale * log2(e) must be finite");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B > 65535 || H > 65535 || cache->stride_row > (1 << 25)) {
    rp_set_error("paged_attn_decode: too many sequences or heads, or rows too far apart");
    return RP_ERR_UNSUPPORTED;
  }
  if (fp8 && c.shift >= 4 && ((reinterpret_cast<uintptr_t>(c.ks) | reinterpret_cast<uintptr_t>(c.vs)) & 15) != 0) {
    rp_set_error("paged_attn_decode: scales must be 16-byte aligned");
    return RP_ERR_UNSUPPORTED;
  }
  if (((qsb | qsh) & 7) != 0 || ((osb | osh) & 3) != 0 ||
      (reinterpret_cast<uintptr_t>(q) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 7) != 0) {
    rp_set_error("paged_attn_decode: q rows must be 16-byte and out rows 8-byte aligned");
    return RP_ERR_UNSUPPORTED;
  }
  if (!rows_apart(cache->head_dim, {{B, osb}, {H, osh}})) {
    rp_set_error("paged_attn_decode: out rows overlap");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const int64_t tiles = (H / cache->heads + 15) / 16;
  const int64_t blocks = key_weights ? c.capacity() / (4 * kJThreads) + 1 : 0;
  if (cache->heads * tiles > 65535 || (H + blocks * cache->heads) * kJThreads > kMaxGridThreads) {
    rp_set_error("paged_attn_decode: too many heads or positions");
    return RP_ERR_UNSUPPORTED;
  }
  const Layout l = decode_layout(B, H, cache, max_seq_len, key_weights != nullptr);
  if (l.total > 0 && (!workspace || workspace_bytes < l.total ||
                      (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)) {
    rp_set_error("paged_attn_decode: workspace of %zu bytes, 256-byte aligned, needed", l.total);
    return RP_ERR_WORKSPACE;
  }
  if (key_weights && !rows_apart(c.capacity(), {{B, wsb}, {cache->heads, wsh}})) {
    rp_set_error("paged_attn_decode: key_weights rows of %lld positions overlap",
                 (long long)c.capacity());
    return RP_ERR_INVALID_ARGUMENT;
  }
  char* ws = static_cast<char*>(workspace);
  DecodeArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.qsb = qsb;
  a.qsh = qsh;
  a.lens = seq_lens;
  // weights of 2^(kSlack - lift) at most, of no more keys than the table has places
  a.lift = kSlack + (float)(64 - __builtin_clzll((unsigned long long)c.capacity()));
  a.c = c2;
  a.out = static_cast<uint16_t*>(out);
  a.osb = osb;
  a.osh = osh;
  a.lse = lse;
  a.weights = key_weights;
  a.wsb = wsb;
  a.wsh = wsh;
  a.H = (int32_t)H;
  a.group = (int32_t)(H / cache->heads);
  a.tiles = (int32_t)tiles;
  a.splits = l.plan.splits;
  a.chunk = l.plan.chunk;
  a.ml = l.part > l.ml ? reinterpret_cast<float2*>(ws + l.ml) : nullptr;
  a.part = l.scores > l.part ? reinterpret_cast<float*>(ws + l.part) : nullptr;
  a.scores = key_weights ? reinterpret_cast<float*>(ws + l.scores) : nullptr;
  a.score_ld = l.score_ld;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t D = cache->head_dim;
  if (q_dtype == RP_DTYPE_F16) {
    if (fp8) launch_decode<kInF16, RP_CACHE_E4M3>(a, c, B, D, l.stream, st);
    else launch_decode<kInF16, RP_CACHE_F16>(a, c, B, D, l.stream, st);
  } else {
    if (fp8) launch_decode<kInBf16, RP_CACHE_E4M3>(a, c, B, D, l.stream, st);
    else launch_decode<kInBf16, RP_CACHE_BF16>(a, c, B, D, l.stream, st);
  }
  return paged_launched("paged_attn_decode");
}
