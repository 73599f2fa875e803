// Attention of few new tokens per sequence (one, some drafted ones) over a
// paged key-value cache: up to 64 rows of a kv head, bound by the keys' bytes.
//
// A wave takes steps of 32 keys, K and V straight into registers (StepRows),
// for NQ columns of 16 rows at once, so a key is read once for all rows.  The
// products and the order of their operands are rp_paged_attn.hip's: S^T = K Q^T
// leaves a lane with eight scores of its column's row, O^T = V^T P^T takes them
// from the same lane.  The steps that the rows see between them, those of the
// sinks first, are shared out evenly over the parts and a part's four waves; a
// sequence's parts are as many as its steps deserve, so that the batch's longest
// one does not hold up the others.
//
// Weights enter the product with V as the sum of two 16-bit numbers, 16 bits
// of them or more, which the matrix cores do while the next rows arrive.  Bases
// and what infinities in V ask for: rp_paged_prompt.h.
//
// One token of 32 sequences in a window of 1024, 32 heads on 8 of 128, bf16, takes
// 27 us (4.9 TB/s), 8 tokens after 131063 fp16 keys of 8 heads 124 (4.3 TB/s, two row
// tiles).  1 to 6 tokens of 16 sequences of 640 to 8000 e4m3fn keys take 42 (3.5
// TB/s): a wave lives 65k cycles, about 30 of those us; 39% of them it waits for
// rows, 42% it issues, three quarters of that vector work.
// Two columns of 16 rows fit 256 registers, two waves a SIMD; four took 512 and
// lost on e4m3fn caches (64 rows of 8000 keys, 16 sequences, 114 us; two tiles of
// two 100), and won on 16-bit ones (130 against 137).
#pragma once

#include "rp_paged_window.h"

namespace rp {
namespace {

constexpr int kFewWaves = 4, kFewThreads = kFewWaves * kWave;

template <int QT, int CT, int D, bool PG16, bool STREAM, int NQ>
struct Few : StepRows<QT == kInF16, CT, D, STREAM> {
  typedef StepRows<QT == kInF16, CT, D, STREAM> Rows;
  using Rows::FP8, Rows::NT, Rows::DPL, Rows::VW;
  using Rows::c, Rows::lane, Rows::m, Rows::g, Rows::vr, Rows::kscale, Rows::vscale, Rows::k_frag;
  static constexpr bool QF16 = QT == kInF16;            // the first product's type
  static constexpr bool VF16 = CT == RP_CACHE_F16;      // the second's

  const WindowArgs& a;
  const KeyTiles<kStep>& keys;
  const int32_t* table;
  int32_t pages, ahead;          // lane i: page of half step i from u0 and from u0 + 32 (PG16)
  int u0, to;                    // to: behind the wave's last step
  int32_t page[2];               // of the step in the registers (PG16)
  int32_t pmin, pmax, pos[NQ];
  u32x4 q[NQ][NT];
  f32x4 acc[NQ][DPL];
  float base[NQ], sum[NQ];

  __device__ __forceinline__ Few(const WindowArgs& a_, const PagedView& c_,
                                 const KeyTiles<kStep>& k_) : Rows(c_), a(a_), keys(k_) {}

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      base[n] = neg_inf();
      sum[n] = 0.0f;
#pragma unroll
      for (int j = 0; j < DPL; ++j) acc[n][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  __device__ __forceinline__ int32_t row_page(int j) const {
    return keys.any(j) ? paged_page(c, table, j) : -1;
  }
  __device__ __forceinline__ int32_t pages_from(int u) const {
    const int at = u + (lane >> 1);
    return at < to ? paged_page(c, table, keys.key(at) + 16 * (lane & 1)) : -1;
  }
  __device__ __forceinline__ void begin(int from, int to_) {
    to = to_;
    u0 = from;
    if constexpr (PG16) {
      pages = pages_from(from);
      ahead = pages_from(from + 32);
    }
  }

  // Brings the K rows, or the V rows, of step u.  What is no row is read as one
  // of page 0 and masked.
  __device__ __forceinline__ void load_k(int u) {
    const int k = keys.key(u);
    if constexpr (PG16) {
      if (u - u0 == 32) {
        u0 = u;
        pages = ahead;
        ahead = pages_from(u + 32);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        page[half] = __builtin_amdgcn_readlane(pages, 2 * (u - u0) + half);
        this->load_k16(half, max(page[half], 0), k + 16 * half);
      }
    } else {
      this->load_k_any([&](int j) { return max(row_page(j), 0); }, k);
    }
  }
  __device__ __forceinline__ void load_v(int u) {
    const int k = keys.key(u);
    if constexpr (PG16) {
#pragma unroll
      for (int half = 0; half < 2; ++half) this->load_v16(half, max(page[half], 0), k + 16 * half);
    } else {
      this->load_v_any([&](int j) { return max(row_page(j), 0); }, k);
    }
  }

  __device__ __forceinline__ static u32x4 pick(const uint32_t* w, uint32_t sel) {
    u32x4 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], sel);
    return f;
  }

  // Step u; `more`: step u + 1 follows, whose rows are requested on the way.
  template <bool CAREFUL>
  __device__ __forceinline__ void step(int u, bool more) {
    const int k = keys.key(u);
    const float lift = base_lift<VF16, CAREFUL>(a);
    f32x4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const u32x4 f = k_frag(half, t);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][half] = mma<QF16>(f, q[n][t], s[n][half]);
      }
    f32x4 ks[2] = {{a.c, a.c, a.c, a.c}, {a.c, a.c, a.c, a.c}};
    if constexpr (FP8) {
      ks[0] *= kscale[0];
      ks[1] *= kscale[1];
    }
    // which of the lane's eight keys hold rows that any token sees
    bool whole = false;
    uint32_t here = 0xffu;
    if constexpr (PG16)
      whole = page[0] >= 0 && page[1] >= 0 && k + kStep - 1 <= pmin &&
              (k > pmax - a.window || k + kStep <= a.sinks);
    if (!whole) {
      here = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = this->key(k, e);
        const bool in = PG16 ? page[e / 4] >= 0 && keys.any(j) : row_page(j) >= 0;
        here |= in ? 1u << e : 0u;
      }
    }
    if (more) load_k(u + 1);

    u32x4 w[2][NQ];                                      // the weights' two parts
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float x[8];
      uint32_t seen = 0xffu;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[n][e / 4][e % 4] * ks[e / 4][e % 4];
      if (!whole) {
        seen = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool in = (here >> e & 1) && sees(a, pos[n], this->key(k, e));
          seen |= in ? 1u << e : 0u;
          x[e] = in ? x[e] : neg_inf();
        }
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                        fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      if (__any(top > base[n] + (kSlack - lift))) {
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float next = fmaxf(base[n], top + lift);
        const float r = next == neg_inf() ? 1.0f : __builtin_amdgcn_exp2f(base[n] - next);
        sum[n] *= r;
#pragma unroll
        for (int j = 0; j < DPL; ++j) acc[n][j] *= r;
        base[n] = next;
      }
      const float b = base[n] == neg_inf() ? 0.0f : base[n];   // no score yet: exp2(-inf) is 0
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(x[e] - b);
      sum[n] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      if constexpr (FP8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] *= vscale[e / 4][e % 4];
          if (!whole) p[e] = seen >> e & 1 ? p[e] : 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y = p[2 * i], z = p[2 * i + 1];
        if constexpr (VF16) {
          const uint32_t hi = round_pair<true>(y, z);
          w[0][n][i] = hi;
          w[1][n][i] = round_pair<true>(y - f16_to_f32(hi & 0xffffu), z - f16_to_f32(hi >> 16));
        } else {
          w[0][n][i] = pack_cut(y, z);
          w[1][n][i] = round_pair<false>(y - bf16_cut(y), z - bf16_cut(z));
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < VW; ++i) vr[e][i] = here >> e & 1 ? vr[e][i] : 0u;
    }
#pragma unroll
    for (int j = 0; j < DPL; j += 2) {
      // the pair of columns j, j + 1 of each row
      uint32_t y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (!FP8) y[e] = vr[e][j / 2];
        else y[e] = j % 4 ? codes_to_16<false, true>(vr[e][j / 4]) : codes_to_16<false, false>(vr[e][j / 4]);
      }
      const u32x4 f[2] = {pick(y, 0x05040100u), pick(y, 0x07060302u)};
      if constexpr (!CAREFUL) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            acc[n][j] = mma<VF16>(f[0], w[e][n], acc[n][j]);
            acc[n][j + 1] = mma<VF16>(f[1], w[e][n], acc[n][j + 1]);
          }
      } else {
        // one token at a time, V as that token sees it
        for (int32_t at = max(0, pmin); at <= pmax; ++at) {
          uint32_t mask[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mask[i] = (sees(a, at, this->key(k, 2 * i)) ? 0xffffu : 0u) |
                      (sees(a, at, this->key(k, 2 * i + 1)) ? 0xffff0000u : 0u);
#pragma unroll
          for (int col = 0; col < 2; ++col) {
            u32x4 v = f[col], fin;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] &= mask[i];
              fin[i] = finite_pair<VF16>(v[i]);          // a second part of 0 beside an infinity
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              f32x4 z = mma<VF16>(v, w[0][n], acc[n][j + col]);
              z = mma<VF16>(fin, w[1][n], z);
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[n][j + col][i] = pos[n] == at ? z[i] : acc[n][j + col][i];
            }
          }
        }
      }
    }
    if (more) load_v(u + 1);
  }

  template <bool CAREFUL>
  __device__ __forceinline__ void run(int from, int end) {
    reset();
    if (from >= end) return;
    begin(from, end);
    load_k(from);
    load_v(from);
    for (int u = from; u < end; ++u) step<CAREFUL>(u, u + 1 < end);
  }

  // Whether any sum of a live row is infinite or NaN.
  __device__ __forceinline__ bool spoiled(const bool* live) const {
    bool bad = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      f32x4 z = acc[n][0] * 0.0f;
#pragma unroll
      for (int j = 1; j < DPL; ++j) z += acc[n][j] * 0.0f;
      const float y = (z[0] + z[1]) + (z[2] + z[3]);
      bad |= live[n] && y != y;
    }
    return __any(bad);
  }
};

// Which part of which sequence a workgroup takes: of a kv head's `room` parts each
// sequence has one, and of those left a share by its steps.
struct Share {
  int b, split, own;             // sequence (-1: none), its part, of how many
};

__device__ __forceinline__ Share part_of(const WindowArgs& a, const PagedView& c, int at, int r0,
                                         int n) {
  const int lane = threadIdx.x & (kWave - 1), B = (int)(a.groups / c.heads);
  if (B == 1) return at < a.splits ? Share{0, at, a.splits} : Share{-1, 0, 1};
  auto steps = [&](int b) { return b < B ? tile_keys<kStep>(a, c, Place(a, b), r0, n).count : 0; };
  auto sum = [&](double x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, kWave);
    return x;
  };
  int mine = steps(lane);
  double all = mine;                                     // whole numbers: exact
  for (int b = kWave + lane; b < B + lane; b += kWave) all += steps(b);
  all = fmax(sum(all), 1.0);
  int before = 0;
  for (int b0 = 0; b0 < B; b0 += kWave) {
    if (b0 > 0) mine = steps(b0 + lane);
    const int own = b0 + lane < B ? min(a.splits, 1 + (int)((double)(a.room - B) * mine / all)) : 0;
    int upto = own;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
      const int y = __shfl_up(upto, o, kWave);
      if (lane >= o) upto += y;
    }
    const uint64_t past = __ballot(before + upto > at);
    if (past) {
      const int l = __builtin_ctzll(past), own_l = __shfl(own, l, kWave);
      return Share{b0 + l, at - before - (__shfl(upto, l, kWave) - own_l), own_l};
    }
    before += __shfl(upto, kWave - 1, kWave);
  }
  return Share{-1, 0, 1};
}

template <int QT, int CT, int D, bool PG16, bool STREAM, int NQ>
__global__ __launch_bounds__(kFewThreads, D <= 128 ? 2 : 1) void few_kernel(WindowArgs a, PagedView c) {
  typedef Few<QT, CT, D, PG16, STREAM, NQ> W;
  __shared__ f32x4 sacc[kFewWaves / 2][NQ][W::DPL][kWave];
  __shared__ float sbase[kFewWaves][NQ][16], ssum[kFewWaves][NQ][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // The row tiles of a part's keys on one XCD, one after the other: what one
  // brings the next ones find in its L2.
  const int64_t parts = (a.splits > 1 ? (int64_t)a.room : a.groups / c.heads) * c.heads;
  const int64_t lanes8 = parts % 8 == 0 ? 8 : 1;
  const int64_t eight = blockIdx.x / (lanes8 * a.tiles), in = blockIdx.x % (lanes8 * a.tiles);
  const int64_t at = eight * lanes8 + in % lanes8;
  const int tile = (int)(in / lanes8), kv = (int)(at % c.heads), r0 = tile * 16 * NQ;
  int b = (int)(at / c.heads), split = 0, own = 1;
  if (a.splits > 1) {
    const Share s = part_of(a, c, b, r0, 16 * NQ);
    b = s.b;
    split = s.split;
    own = s.own;
    if (b < 0) return;
  }

  const Place pl(a, b);
  const int rows = pl.m * a.group, all = a.S * a.group;
  const int last = min(r0 + 16 * NQ, rows) - 1;
  const int32_t pmin = last >= r0 ? pl.first + r0 / a.group : 0x7fffffff;   // see prompt_kernel
  const int32_t pmax = last >= r0 ? max(-1, pl.first + last / a.group) : -1;
  const KeyTiles<kStep> keys = tile_keys<kStep>(a, c, pl, r0, 16 * NQ);
  W w(a, c, keys);
  w.place(threadIdx.x & (kWave - 1), kv);
  w.table = c.table + b * c.table_stride;
  w.pmin = pmin;
  w.pmax = pmax;
  bool live[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = r0 + 16 * n + w.m, token = row / a.group;
    live[n] = row < rows;
    w.pos[n] = live[n] ? pl.first + token : -1;
    const uint16_t* src = a.q + b * a.qsb + (int64_t)(kv * a.group + row % a.group) * a.qsh +
                          (int64_t)token * a.qss;
#pragma unroll
    for (int t = 0; t < W::NT; ++t) {
      const int d = W::FP8 && D >= 64 ? 64 * (t / 2) + 16 * w.g + 8 * (t % 2) : 32 * t + 8 * w.g;
      w.q[n][t] = live[n] ? *reinterpret_cast<const u32x4*>(src + d) : u32x4{0u, 0u, 0u, 0u};
      w.q[n][t] ^= a.flip;
    }
  }
  if (split == 0) {                                      // the parts that the sequence has not
    const int none = a.splits - own;
    for (int i = threadIdx.x; i < 16 * NQ * none; i += kFewThreads) {
      const int row = r0 + i / none;
      if (row >= all) break;
      const int64_t orow = ((int64_t)b * a.H + kv * a.group + row % a.group) * a.S + row / a.group;
      a.ml[orow * a.splits + own + i % none] = float2{neg_inf(), 0.0f};
    }
  }
  // the part's steps, and the wave's of them
  const int t0 = (int)((int64_t)keys.count * split / own);
  const int t1 = (int)((int64_t)keys.count * (split + 1) / own);
  const int from = t0 + (t1 - t0) * wave / kFewWaves, end = t0 + (t1 - t0) * (wave + 1) / kFewWaves;
  w.template run<false>(from, end);
  if (w.spoiled(live)) w.template run<true>(from, end);

  // the waves' parts about one base
  float base[NQ], sum[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    w.sum[n] += __shfl_xor(w.sum[n], 16, kWave);
    w.sum[n] += __shfl_xor(w.sum[n], 32, kWave);
    if (w.g == 0) {
      sbase[wave][n][w.m] = w.base[n];
      ssum[wave][n][w.m] = w.sum[n];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    base[n] = sbase[0][n][w.m];
#pragma unroll
    for (int i = 1; i < kFewWaves; ++i) base[n] = fmaxf(base[n], sbase[i][n][w.m]);
    const float b0 = base[n] == neg_inf() ? 0.0f : base[n];
    sum[n] = 0.0f;
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i)
      sum[n] += ssum[i][n][w.m] * __builtin_amdgcn_exp2f(sbase[i][n][w.m] - b0);
    if (!live[n]) sum[n] = 0.0f;                         // a row past the new tokens
    const float r = sum[n] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(w.base[n] - b0) / sum[n];
#pragma unroll
    for (int j = 0; j < W::DPL; ++j) w.acc[n][j] *= r;
  }
#pragma unroll
  for (int half = kFewWaves / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int j = 0; j < W::DPL; ++j) sacc[wave - half][n][j][w.lane] = w.acc[n][j];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int j = 0; j < W::DPL; ++j) w.acc[n][j] += sacc[wave][n][j][w.lane];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = r0 + 16 * n + w.m;
    if (row >= all) continue;
    const int token = row / a.group, head = kv * a.group + row % a.group;
    const int64_t orow = ((int64_t)b * a.H + head) * a.S + token;
    float* part = a.part + (orow * a.splits + split) * D;
    uint16_t* out = a.out + b * a.osb + (int64_t)head * a.osh + (int64_t)token * a.oss;
    // a lane's columns of each of its four rows of O^T lie next to each other
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < W::DPL; j += 2) {
        const float y = sum[n] == 0.0f ? 0.0f : w.acc[n][j][i];
        const float z = sum[n] == 0.0f ? 0.0f : w.acc[n][j + 1][i];
        const int col = W::Rows::column(4 * w.g + i, j);
        if (a.splits > 1) *reinterpret_cast<float2*>(part + col) = float2{y, z};
        else *reinterpret_cast<uint32_t*>(out + col) = pack_out<QT>(y, z);
      }
    if (w.g != 0) continue;
    if (a.splits > 1) a.ml[orow * a.splits + split] = float2{base[n], sum[n]};
    else if (a.lse)
      a.lse[orow] = sum[n] == 0.0f ? neg_inf() : (base[n] + __builtin_amdgcn_logf(sum[n])) * kLn2;
  }
}

template <int QT, int CT, int D, int NQ>
void launch_few_n(const WindowArgs& a, const PagedView& c, bool stream, hipStream_t st) {
  const dim3 grid((unsigned)((a.splits > 1 ? (int64_t)a.room * c.heads : a.groups) * a.tiles));
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kFewThreads), 0, st, a, c); };
  if (c.shift < 4) go(few_kernel<QT, CT, D, false, false, NQ>);
  else if (stream) go(few_kernel<QT, CT, D, true, true, NQ>);
  else go(few_kernel<QT, CT, D, true, false, NQ>);
}

template <int QT, int CT, int D>
void launch_few_d(const WindowArgs& a, const PagedView& c, int columns, bool stream,
                  hipStream_t st) {
  if constexpr (D < 256) {
    if (columns == 2) return launch_few_n<QT, CT, D, 2>(a, c, stream, st);
  }
  launch_few_n<QT, CT, D, 1>(a, c, stream, st);
}

template <int QT, int CT>
void launch_few(const WindowArgs& a, const PagedView& c, int64_t D, int columns, bool stream,
                hipStream_t st) {
  if (D == 32) launch_few_d<QT, CT, 32>(a, c, columns, stream, st);
  else if (D == 64) launch_few_d<QT, CT, 64>(a, c, columns, stream, st);
  else if (D == 128) launch_few_d<QT, CT, 128>(a, c, columns, stream, st);
  else launch_few_d<QT, CT, 256>(a, c, columns, stream, st);
}

}  // namespace
}  // namespace rp
