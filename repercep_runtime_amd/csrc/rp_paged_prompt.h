// Attention of many new tokens per sequence (a prompt, a chunk of one) over a
// paged key-value cache, causal, within a window, with sinks.
//
// Both products run on the matrix cores (32x32x16).  A wave owns 32 rows; a
// workgroup's waves share tiles of 64 keys (32 at 256 dims), K and V staged through registers into
// LDS as 16-bit rows, two tiles deep: any page size, e4m3fn codes converted
// once for all waves, what no row sees as zeros.
//
// * S^T = K Q^T: a lane ends up with 32 scores of one row, so the softmax's
//   maximum and sum stay in the lane but for its partner in the wave's other
//   half.  The keys it holds are those that O^T = V^T P^T asks of it, if V's
//   operand is read in that order (ds_read_b64_tr_b16: four keys of a column):
//   P never leaves the lane.
// * The running maximum is lazy: rows are weighed about their base, which is
//   only moved, and the sums rescaled, when a score exceeds it by 2^kSlack.
//   A bf16 P is weighed about the largest score, and again, token by token as
//   below, if a sum of values near the type's largest overflows: then about a base
//   so high that a row's weights add up to less than 1 (always there, products with
//   values below 2^-100 lost bits).  An fp16 P is weighed about a base below the
//   largest score, so that weights down to 2^-21 of the largest keep their 11 bits,
//   and smaller ones 2^-31 of it.
// * P enters the second product rounded once to 16 bits, as precise as the
//   output.  For an e4m3fn cache, whose row scales can be of any size, it is
//   bf16; an fp16 output then takes it as the sum of two bf16 numbers.
// * A row of V that only some of a wave's rows see may hold infinities or NaNs,
//   which 0 P does not silence.  Sums that come out infinite or NaN are taken
//   again token by token, V masked for each.
// * A tile takes a wave 32 matrix instructions (1024 cycles) and about 200 vector
//   ones; one after the other they took 3000 cycles.  So a tile's weights and
//   product with V run beside the next tile's scores (fused), in an order that is
//   written out, since the compiler's own put the LDS reads right before their
//   uses; and the two waves of a SIMD take turns at that and at staging.  What
//   each brought, a prompt of 16384 tokens, 32 heads on 8 of 128, bf16:
//   one phase after the other 2.59 ms, side by side 2.41, in written order 2.22,
//   in turns and weights spread evenly 2.17, the rows of the tile after the
//   next stored and asked for before the next tile's scores are weighed 2.12.
//
// That prompt takes 2.11 to 2.18 ms, 1.01 to 1.04 PFLOP/s, where a library product of
// 16384^2 reaches 1.38 (2.56 ms on a card where that reaches 1.21); fp16 2.25, bf16
// over e4m3fn rows 2.45.  Matrix cores 48% busy, the VALU 51%, no LDS conflicts;
// waves spend 27% of their cycles at barriers and counters, 28% without an issue
// slot.  256 dims, four waves a workgroup and so one a SIMD, take 6.5 ms (0.68
// PFLOP/s).

#pragma once

#include <type_traits>

#include "rp_paged_window.h"

#define RP_INLINE __attribute__((always_inline))

namespace rp {
namespace {

constexpr int kAhead = 4;                       // matrix instructions that LDS reads are ahead

template <bool F16>
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Bits 0 .. n of a word: none below 0, all from 31.
__device__ __forceinline__ uint32_t bits_up_to(int32_t n) {
  return n < 0 ? 0u : 0xffffffffu >> (31 - min(n, 31));
}

// LDS by address, which the compiler takes as it is: one register and a constant
// offset a read.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  uint32_t at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
  asm("" : "+v"(at));
  return at;
}
__device__ __forceinline__ u32x4 lds_read16(uint32_t at) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)at;
}
// Four keys of a column: the 16 lanes of a row of lanes bring four rows of 16
// columns, four lanes a row, and each takes a column.
__device__ __forceinline__ u32x2 column4(uint32_t at) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(uintptr_t)at));
}

template <int QT, int CT, int D, int NW>
struct Prompt {
  static constexpr bool FP8 = CT == RP_CACHE_E4M3;
  static constexpr bool QF16 = QT == kInF16;            // the first product's type
  static constexpr bool VF16 = CT == RP_CACHE_F16;      // the second's
  static constexpr int PARTS = FP8 && QF16 ? 2 : 1;     // of a weight
  static constexpr int EB = FP8 ? 1 : 2, NT = NW * kWave;
  static constexpr int QSTEPS = D / 16, DB = D / 32;
  // Keys a tile, up to one page entry a lane, in blocks of 32.  At 256 dims a wave's
  // sums and Q leave no registers, and LDS no room, for 64: Q spilled, and 16384
  // tokens took 9.5 ms, with 32 6.5.
  static constexpr int TILE = D == 256 ? 32 : 64, KB = TILE / 32;
  static constexpr uint64_t ALL = ~0ull >> (64 - TILE);
  // Rows of LDS, without bank conflicts: eight rows of K at one column are read
  // at a time, four rows of V's 64 bytes.
  static constexpr int LDK = D + 8, LDV = D == 32 ? 32 : D + 32;
  static constexpr int CPR = D * EB / 16;               // 16-byte chunks a row
  static constexpr int NCH = (TILE * CPR + NT - 1) / NT;
  static constexpr int WROWS = kWave / CPR;             // rows of a wave's chunks
  static constexpr int ROWS = NW * 32;

  // Q in LDS: 256 registers a lane, two waves a SIMD, hold it barely or not, read
  // back from scratch they wait for the staged loads, which the same counter counts.
  // 16384 tokens with Q in LDS and in registers: bf16 2.15 and 2.12 ms, fp16 2.27 and
  // 2.32, bf16 over e4m3fn rows 2.49 and 2.90, fp16 over those 3.19 and 3.21.
  static constexpr bool QLDS = D == 256 || (D == 128 && NW == 8);

  struct alignas(16) Shared {
    uint16_t k[2][TILE][LDK];
    uint16_t v[2][TILE][LDV];
    float ks[2][TILE], vs[2][TILE];                   // e4m3fn only
    uint16_t q[QLDS ? ROWS : 1][LDK];
    int redo;
  };
};

template <int QT, int CT, int D, int NW>
__global__ __launch_bounds__(NW* kWave) void prompt_kernel(WindowArgs a, PagedView c) {
  typedef Prompt<QT, CT, D, NW> P;
  __shared__ typename P::Shared sh;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int m = lane & 31, h = lane >> 5;

  // The workgroups of eight (sequence, kv head) pairs at a time, one pair an
  // XCD, so that a pair's keys stay in one L2; the tiles with most keys first.
  int64_t at = blockIdx.x;
  const int split = (int)(at % a.splits);
  at /= a.splits;
  const int64_t lanes8 = min((int64_t)8, a.groups);
  const int64_t eight = at / (lanes8 * a.tiles);
  const int64_t width = min(lanes8, a.groups - eight * lanes8);
  at -= eight * lanes8 * a.tiles;
  const int64_t pair = eight * lanes8 + at % width;
  const int tile = a.tiles - 1 - (int)(at / width);
  const int b = (int)(pair / c.heads), kv = (int)(pair % c.heads);

  const Place pl(a, b);
  const int rows = pl.m * a.group, all = a.S * a.group;
  const int r0 = tile * P::ROWS;                         // the workgroup's first row
  const int row = r0 + 32 * wave + m;
  const int token = row / a.group, head = kv * a.group + row % a.group;
  const bool live = row < rows;
  const int64_t orow = ((int64_t)b * a.H + head) * a.S + token;
  const int32_t pos = live ? pl.first + token : -1;
  // the wave's rows' first and last positions (no row: the largest number and -1,
  // between which no pass over positions has a step)
  const int w0 = r0 + 32 * wave, w1 = min(w0 + 32, rows) - 1;
  const int32_t pmin = w1 >= w0 ? pl.first + w0 / a.group : 0x7fffffff;
  const int32_t pmax = w1 >= w0 ? max(-1, pl.first + w1 / a.group) : -1;
  const KeyTiles<P::TILE> keys = tile_keys<P::TILE>(a, c, pl, r0, P::ROWS);
  const int t0 = (int)((int64_t)keys.count * split / a.splits);
  const int t1 = (int)((int64_t)keys.count * (split + 1) / a.splits);
  const int32_t* table = c.table + b * c.table_stride;

  u32x4 q[P::QLDS ? 1 : P::QSTEPS];
  {
    const uint16_t* src = a.q + b * a.qsb + (int64_t)head * a.qsh + (int64_t)token * a.qss + 8 * h;
#pragma unroll
    for (int t = 0; t < P::QSTEPS; ++t) {
      u32x4 x = live ? *reinterpret_cast<const u32x4*>(src + 16 * t) : u32x4{0u, 0u, 0u, 0u};
      x ^= a.flip;
      if constexpr (P::QLDS) *reinterpret_cast<u32x4*>(&sh.q[32 * wave + m][16 * t + 8 * h]) = x;
      else q[t] = x;
    }
  }
  const uint32_t qlds = lds_address(&sh.q[P::QLDS ? 32 * wave + m : 0][8 * h]);
  auto q_frag = [&](int t) RP_INLINE -> u32x4 {
    if constexpr (P::QLDS) return lds_read16(qlds + 32 * t);
    else return q[t];
  };
  // the lane's part of a K operand: the key m of 32, dims 16 t + 8 h .. + 7
  const uint32_t klds = lds_address(&sh.k[0][m][8 * h]);
  auto k_frag = [&](int buf, int n) RP_INLINE -> u32x4 {     // of keys 32 (n % KB) .., t = n / KB
    return lds_read16(klds + 2 * ((buf * P::TILE + 32 * (n % P::KB)) * P::LDK + 16 * (n / P::KB)));
  };

  f32x16 acc[P::DB];
  float base, sum, lift;

  // ---- staging: lane l's page entry says where key l of a tile lies; a thread
  // brings chunks of 16 bytes, a row's by threads next to each other
  u32x4 kreg[P::NCH], vreg[P::NCH];
  float ksreg = 0.0f, vsreg = 0.0f;
  // (the entry as it stands in the table: checking it here would wait for it)
  auto entry = [&](int t) RP_INLINE -> int32_t {
    return table[min((keys.key(t) + lane) >> c.shift, c.max_pages - 1)];
  };
  // the page, or -1 where there is none
  auto page_of = [&](int t, int32_t e) RP_INLINE -> int32_t {
    return t < t1 && lane < P::TILE && keys.key(t) + lane < keys.hi && e >= 0 && e < c.num_pages ? e : -1;
  };
  // which keys of tile t any of the workgroup's rows sees
  auto present = [&](int t, int32_t pages) RP_INLINE -> uint64_t {
    return __ballot(pages >= 0 && keys.any(keys.key(t) + lane));
  };
  // Where key l of a tile lies, in bytes from the head's first row.  What is no
  // row is read as one of page 0; what no row sees is put into LDS as zeros.
  auto offset_of = [&](int t, int32_t page) RP_INLINE -> int64_t {
    return max(0, page) * (c.sp * P::EB) + ((keys.key(t) + lane) & c.page_mask()) * (c.sr * P::EB);
  };
  const char* const khead = c.k + kv * c.sh * P::EB;
  const char* const vhead = c.v + kv * c.sh * P::EB;
  // a wave's rows of a chunk lie in one page, unless pages are smaller
  const bool one_page = c.page_mask() >= P::WROWS - 1;
  const uint32_t lane_off = (uint32_t)((lane / P::CPR) * c.sr * P::EB + lane % P::CPR * 16);
  auto load = [&](auto one, u32x4* to, const char* from, int64_t off) RP_INLINE {
    const int lo = (int)off, hi = (int)(off >> 32);
#pragma unroll
    for (int i = 0; i < P::NCH; ++i) {
      const int rw = min(wave * P::WROWS + i * (P::NT / P::CPR), P::TILE - P::WROWS);
      if constexpr (decltype(one)::value) {
        const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, rw) << 32 |
                            (uint32_t)__builtin_amdgcn_readlane(lo, rw);
        to[i] = *reinterpret_cast<const u32x4*>(from + at + lane_off);
      } else {
        const int r = rw + lane / P::CPR;
        const uint64_t at = (uint64_t)(uint32_t)__shfl(hi, r, kWave) << 32 | (uint32_t)__shfl(lo, r, kWave);
        to[i] = *reinterpret_cast<const u32x4*>(from + at + lane % P::CPR * 16);
      }
    }
  };
  auto load_rows = [&](int64_t koff, int64_t voff) RP_INLINE {
    if (one_page) {
      load(std::true_type{}, vreg, vhead, voff);
      load(std::true_type{}, kreg, khead, koff);
    } else {
      load(std::false_type{}, vreg, vhead, voff);
      load(std::false_type{}, kreg, khead, koff);
    }
  };
  auto load_scale = [&](int t, int32_t page, const float* from) RP_INLINE -> float {
    return from[paged_scale(c, max(0, page), kv, keys.key(t) + lane)];
  };
  auto store = [&](uint16_t* to, int ld, u32x4* from, uint64_t here, auto f16) RP_INLINE {
#pragma unroll
    for (int i = 0; i < P::NCH; ++i) {
      const int ch = tid + i * P::NT;
      if (P::TILE * P::CPR % P::NT != 0 && ch >= P::TILE * P::CPR) break;
      const int r = ch / P::CPR;
      u32x4 x = from[i];
      if (here != P::ALL) x &= here >> r & 1 ? 0xffffffffu : 0u;
      if constexpr (!P::FP8) {
        *reinterpret_cast<u32x4*>(to + r * ld + ch % P::CPR * 8) = x;
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          u32x4 y;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            y[2 * e] = codes_to_16<decltype(f16)::value, false>(x[2 * half + e]);
            y[2 * e + 1] = codes_to_16<decltype(f16)::value, true>(x[2 * half + e]);
          }
          *reinterpret_cast<u32x4*>(to + r * ld + ch % P::CPR * 16 + 8 * half) = y;
        }
      }
    }
  };
  auto store_k = [&](int buf, uint64_t here) RP_INLINE {
    store(&sh.k[buf][0][0], P::LDK, kreg, here, std::bool_constant<P::QF16>{});
    if constexpr (P::FP8) {
      if (wave == 0 && lane < P::TILE) sh.ks[buf][lane] = here >> lane & 1 ? ksreg * a.c : 0.0f;
    }
  };
  auto store_v = [&](int buf, uint64_t here) RP_INLINE {
    store(&sh.v[buf][0][0], P::LDV, vreg, here, std::false_type{});
    if constexpr (P::FP8) {
      if (wave == 1 && lane < P::TILE) sh.vs[buf][lane] = here >> lane & 1 ? vsreg : 0.0f;
    }
  };

  // ---- a tile's scores, in powers of two but for the factor c1
  const float c1 = P::FP8 ? 1.0f : a.c;
  auto product = [&](int buf, f32x16* to) RP_INLINE {
#pragma unroll
    for (int i = 0; i < 16; ++i) to[0][i] = to[P::KB - 1][i] = 0.0f;
#pragma unroll
    for (int n = 0; n < P::KB * P::QSTEPS; ++n)
      to[n % P::KB] = mma32<P::QF16>(k_frag(buf, n), q_frag(n / P::KB), to[n % P::KB]);
  };
  uint32_t seen[P::KB];                                      // bit 8 i + e: key 8 i + 4 h + e
  bool whole;
  float top;
  auto larger = [&](const f32x16* s, int i) RP_INLINE {   // top, of scores i of each block too
    if (i == 0) top = s[0][0];
    else top = __builtin_elementwise_maximum(top, s[0][i]);
    if constexpr (P::KB == 2) top = __builtin_elementwise_maximum(top, s[1][i]);
  };
  // Masks the scores s of the tile at kb and finds their largest (`found`: it
  // is, unless some are masked).
  auto weigh = [&](f32x16* s, int buf, int32_t kb, uint64_t here, bool found) RP_INLINE {
    if constexpr (P::FP8) {
#pragma unroll
      for (int k = 0; k < P::KB; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 f = *reinterpret_cast<const f32x4*>(&sh.ks[buf][32 * k + 8 * i + 4 * h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[k][4 * i + e] *= f[e];
        }
    }
    whole = here == P::ALL && kb + P::TILE - 1 <= pmin &&
            (kb > pmax - a.window || kb + P::TILE <= a.sinks);
    if (!whole) {
#pragma unroll
      for (int k = 0; k < P::KB; ++k) {
        const int32_t j = kb + 32 * k + 4 * h, d = max(-1, pos - j);
        seen[k] = (uint32_t)(here >> 32 * k) >> 4 * h & bits_up_to(d) &
                  (~bits_up_to(d - a.window) | bits_up_to(a.sinks - 1 - j));
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[k][i] = seen[k] & 1u << (8 * (i / 4) + i % 4) ? s[k][i] : neg_inf();
      }
    }
    if (!whole || !found) {
      // of a row with a NaN a NaN, which moves no base: the row is NaN
#pragma unroll
      for (int i = 0; i < 16; ++i) larger(s, i);
    }
    top *= c1;
    if (__any(top > base + (kSlack - lift))) {
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float next = fmaxf(base, top + lift);
      const float r = next == neg_inf() ? 1.0f : __builtin_amdgcn_exp2f(base - next);
      sum *= r;
#pragma unroll
      for (int d = 0; d < P::DB; ++d) acc[d] *= r;
      base = next;
    }
  };

  // ---- P from s, and its product with V
  uint32_t p[P::PARTS][P::KB][8];
  // Weights 2 j, 2 j + 1 of block k (of 16), about the base b0, f their scales.
  auto weight_pair = [&](const f32x16* s, int k, int j, float b0, float f0, float f1) RP_INLINE {
    float u = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][2 * j], c1, -b0));
    float v = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][2 * j + 1], c1, -b0));
    sum += u + v;
    if constexpr (P::FP8) {
      u *= f0;
      v *= f1;
      if (!whole) {                                      // what is not seen weighs 0 whatever its scale
        const uint32_t bit = 8 * (j / 2) + 2 * (j % 2);
        u = seen[k] >> bit & 1 ? u : 0.0f;
        v = seen[k] >> bit & 2 ? v : 0.0f;
      }
    }
    if constexpr (P::PARTS == 1) {
      p[0][k][j] = round_pair<P::VF16>(u, v);
    } else {
      p[0][k][j] = pack_cut(u, v);
      p[P::PARTS - 1][k][j] = round_pair<false>(u - bf16_cut(u), v - bf16_cut(v));
    }
  };
  auto scales = [&](int buf, int g) RP_INLINE -> f32x4 {      // of weights 4 g .. 4 g + 3 of 32
    return *reinterpret_cast<const f32x4*>(&sh.vs[buf][32 * (g / 4) + 8 * (g % 4) + 4 * h]);
  };
  auto weight_base = [&]() RP_INLINE -> float {
    return base == neg_inf() ? 0.0f : base;              // no score yet: exp2(-inf) is 0
  };
  auto weights = [&](const f32x16* s, int buf) RP_INLINE {
    const float b0 = weight_base();
#pragma unroll
    for (int g = 0; g < 4 * P::KB; ++g) {
      f32x4 f = {1.0f, 1.0f, 1.0f, 1.0f};
      if constexpr (P::FP8) f = scales(buf, g);
      weight_pair(s, g / 4, 2 * (g % 4), b0, f[0], f[1]);
      weight_pair(s, g / 4, 2 * (g % 4) + 1, b0, f[2], f[3]);
    }
  };
  // V's operand n of a tile: columns 32 d .. + 31 (d = n % DB) of keys 16 (n / DB)
  // + 4 h + {0..3, 8..11}
  const int l16 = lane & 15;
  const uint32_t vlds =
      lds_address(&sh.v[0][4 * h + (l16 >> 2)][(lane >> 4 & 1) * 16 + (l16 & 3) * 4]);
  auto v_frag = [&](int buf, int n) RP_INLINE -> u32x4 {
    const uint32_t at =
        vlds + 2 * ((buf * P::TILE + 16 * (n / P::DB)) * P::LDV + 32 * (n % P::DB));
    const u32x2 lo = column4(at), hi = column4(at + 2 * 8 * P::LDV);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto p_frag = [&](int e, int n) RP_INLINE -> u32x4 {
    const int k = n / P::DB / 2, u = n / P::DB % 2;
    return u32x4{p[e][k][4 * u], p[e][k][4 * u + 1], p[e][k][4 * u + 2], p[e][k][4 * u + 3]};
  };
  auto values = [&](int buf) RP_INLINE {
#pragma unroll
    for (int n = 0; n < 2 * P::KB * P::DB; ++n) {
      const u32x4 f = v_frag(buf, n);
#pragma unroll
      for (int e = 0; e < P::PARTS; ++e)
        acc[n % P::DB] = mma32<P::VF16>(f, p_frag(e, n), acc[n % P::DB]);
    }
  };
  // The same one token of the wave at a time, V as that token sees it.
  auto values_apart = [&](int buf, int32_t kb) RP_INLINE {
    for (int32_t at = max(0, pmin); at <= pmax; ++at) {
      const bool mine = pos == at;
#pragma unroll
      for (int n = 0; n < 2 * P::KB * P::DB; ++n) {
        u32x4 f = v_frag(buf, n);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int32_t j = kb + 16 * (n / P::DB) + 4 * h + (e < 2 ? 2 * e : 4 + 2 * e);
          f[e] &= (sees(a, at, j) ? 0xffffu : 0u) | (sees(a, at, j + 1) ? 0xffff0000u : 0u);
        }
        f32x16 y = mma32<P::VF16>(f, p_frag(0, n), acc[n % P::DB]);
        if constexpr (P::PARTS == 2) {
          // a second part of 0 would make NaN of an infinity
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = finite_pair<P::VF16>(f[e]);
          y = mma32<P::VF16>(f, p_frag(1, n), y);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n % P::DB][i] = mine ? y[i] : acc[n % P::DB][i];
      }
    }
  };

  // Tile t's weights and product with V, from its scores s, beside tile t + 1's
  // scores: matrix instructions one by one, each with the LDS reads of the one
  // kAhead later and a share of the vector work, in the order written.
  auto fused = [&](const f32x16* s, f32x16* next, int buf) RP_INLINE {
    constexpr int NK = P::KB * P::QSTEPS, NV = 2 * P::KB * P::DB;
    constexpr int QA = P::KB == 2 ? 2 : 4;               // Q's operands in registers
    u32x4 kf[kAhead], vf[kAhead], qf[QA];
    f32x4 sf[2];
    const float b0 = weight_base();
    __builtin_amdgcn_s_setprio(1);                       // before the half that stages
    if constexpr (P::FP8) sf[0] = scales(buf, 0);
#pragma unroll
    for (int t = 0; t < QA - 1; ++t) qf[t] = q_frag(t);
#pragma unroll
    for (int n = 0; n < kAhead; ++n) kf[n] = k_frag(buf ^ 1, n);
#pragma unroll
    for (int i = 0; i < 16; ++i) next[0][i] = next[P::KB - 1][i] = 0.0f;
    // The pairs of weights evenly over the steps before the product that asks for
    // the last of them, each in time for its own.
    auto some_weights = [&](int step) RP_INLINE {
      constexpr int T = NK + 3 * NV / 4;
#pragma unroll
      for (int j = 0; j < 8 * P::KB; ++j) {
        if (2 * j * T / (16 * P::KB + 1) != step) continue;
        const int g = j / 2;
        if constexpr (P::FP8) {
          if (j % 2 == 0 && g + 1 < 4 * P::KB) sf[(g + 1) % 2] = scales(buf, g + 1);
        }
        const f32x4 f = P::FP8 ? sf[g % 2] : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
        weight_pair(s, j / 8, j % 8, b0, f[2 * (j % 2)], f[2 * (j % 2) + 1]);
      }
      if (step % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    };
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const int t = n / P::KB, later = t + QA - 1;
      if (n % P::KB == 0 && later < P::QSTEPS) qf[later % QA] = q_frag(later);
      next[n % P::KB] = mma32<P::QF16>(kf[n % kAhead], qf[t % QA], next[n % P::KB]);
      if (n + kAhead < NK) kf[n % kAhead] = k_frag(buf ^ 1, n + kAhead);
      else vf[(n + kAhead - NK) % kAhead] = v_frag(buf, n + kAhead - NK);
      some_weights(n);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
#pragma unroll
      for (int e = 0; e < P::PARTS; ++e)
        acc[n % P::DB] = mma32<P::VF16>(vf[n % kAhead], p_frag(e, n), acc[n % P::DB]);
      if (n + kAhead < NV) vf[n % kAhead] = v_frag(buf, n + kAhead);
      if constexpr (!P::FP8) {
#pragma unroll
        for (int i = 16 * n / NV; i < 16 * (n + 1) / NV; ++i) larger(next, i);
      }
      some_weights(NK + n);
    }
    __builtin_amdgcn_s_setprio(0);
    // found here, not where they are used
    asm volatile("" : "+v"(sum));
    if constexpr (!P::FP8) asm volatile("" : "+v"(top));
  };

  auto reset = [&](float to) RP_INLINE {
    lift = to;
    base = neg_inf();
    sum = 0.0f;
#pragma unroll
    for (int d = 0; d < P::DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  };
  // All tiles.  Of eight waves two share a SIMD, one of each half of the
  // workgroup, and the halves take turns: while one runs its products (fused),
  // the other masks and stages, between two barriers a tile.  K is staged a tile
  // ahead of V; the second half, half a tile behind, stages one further ahead, so
  // that a tile is whole before the first half asks for it:
  //   first half   fused(t) | mask t + 1, store K t + 2 and V t + 1 | fused(t + 1)
  //   second half  store K t + 2 and V t + 1 | fused(t) | mask t + 1, store t + 3 and t + 2
  auto run = [&]() RP_INLINE {
    reset(base_lift<P::VF16, false>(a));
    if (t0 >= t1) return;
    const bool second = NW == 8 && wave >= 4;
    uint64_t q0, q1 = 0, q2 = 0;                         // the tiles' keys that are there, t + 1 on
    int32_t page, ahead;                                 // of tile tk; tile tk + 1's entry
    int64_t off;                                         // of tile tk
    int tk = t0;                                         // the tile whose K is in the registers
    // K of tile tk + 1, V of tile tk; which of K's keys are there
    auto next_rows = [&]() RP_INLINE -> uint64_t {
      if constexpr (P::FP8) {
        if (wave == 1) vsreg = load_scale(tk, page, c.vs);
      }
      page = page_of(++tk, ahead);
      ahead = entry(tk + 1);
      const int64_t before = off;
      off = offset_of(tk, page);
      load_rows(off, before);
      if constexpr (P::FP8) {
        if (wave == 0) ksreg = load_scale(tk, page, c.ks);
      }
      return present(tk, page);
    };
    auto put_rows = [&](uint64_t here, uint64_t before) RP_INLINE {
      store_k((tk - t0) & 1, here);
      store_v((tk - t0 + 1) & 1, before);
    };
    f32x16 even[P::KB], odd[P::KB];                              // the tiles' scores in turn
    {
      page = page_of(t0, entry(t0));
      off = offset_of(t0, page);
      ahead = entry(t0 + 1);
      const uint64_t here = present(t0, page);
      load_rows(off, off);
      if constexpr (P::FP8) {
        if (wave == 0) ksreg = load_scale(t0, page, c.ks);
      }
      store_k(0, here);
      q0 = next_rows();
      put_rows(q0, here);
      __syncthreads();
      product(0, even);
      weigh(even, 0, keys.key(t0), here, false);
      q1 = next_rows();
      __syncthreads();                                   // K's first tile is overwritten next
      if (second) {
        put_rows(q1, q0);
        q2 = next_rows();
        __syncthreads();
      }
    }
    auto step = [&](int t, int buf, const f32x16* s, f32x16* next) RP_INLINE {
      fused(s, next, buf);
      if constexpr (NW == 8) __syncthreads();
      put_rows(second ? q2 : q1, second ? q1 : q0);
      const uint64_t here = next_rows();
      weigh(next, buf ^ 1, keys.key(t + 1), q0, !P::FP8);
      q0 = q1;
      q1 = second ? q2 : here;
      q2 = here;
      __syncthreads();
    };
    int t = t0;
    for (; t + 2 < t1; t += 2) {
      step(t, 0, even, odd);
      step(t + 1, 1, odd, even);
    }
    if (t + 1 < t1) {
      step(t, 0, even, odd);
      weights(odd, 1);
      values(1);
    } else {
      weights(even, 0);
      values(0);
    }
    if (NW == 8 && !second) __syncthreads();
  };
  // The same a tile after the other, each token's part of V by itself.
  auto run_apart = [&]() RP_INLINE {
    reset(base_lift<P::VF16, true>(a));
    for (int t = t0; t < t1; ++t) {
      const int32_t page = page_of(t, entry(t));
      const int64_t off = offset_of(t, page);
      const uint64_t here = present(t, page);
      load_rows(off, off);
      if constexpr (P::FP8) {
        if (wave == 0) ksreg = load_scale(t, page, c.ks);
        if (wave == 1) vsreg = load_scale(t, page, c.vs);
      }
      __syncthreads();
      store_k(0, here);
      store_v(0, here);
      __syncthreads();
      f32x16 s[P::KB];
      product(0, s);
      weigh(s, 0, keys.key(t), here, false);
      weights(s, 0);
      values_apart(0, keys.key(t));
    }
  };
  if (tid == 0) sh.redo = 0;
  run();
  {
    f32x16 z = acc[0] * 0.0f;
#pragma unroll
    for (int d = 1; d < P::DB; ++d) z += acc[d] * 0.0f;
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) y += z[i];
    __syncthreads();
    if (live && y != y) sh.redo = 1;
    __syncthreads();
    if (sh.redo) run_apart();
  }

  if (row >= all) return;
  sum += __shfl_xor(sum, 32, kWave);
  if (!live) sum = 0.0f;                                 // a row past the new tokens
  const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (a.splits > 1) {
    if (h == 0) a.ml[orow * a.splits + split] = float2{base, sum};
    if (sum == 0.0f) return;
    float* part = a.part + (orow * a.splits + split) * D + 4 * h;
#pragma unroll
    for (int d = 0; d < P::DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(part + 32 * d + 8 * i) =
            f32x4{acc[d][4 * i] * r, acc[d][4 * i + 1] * r, acc[d][4 * i + 2] * r, acc[d][4 * i + 3] * r};
    return;
  }
  uint16_t* out = a.out + b * a.osb + (int64_t)head * a.osh + (int64_t)token * a.oss + 4 * h;
#pragma unroll
  for (int d = 0; d < P::DB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 y = {acc[d][4 * i] * r, acc[d][4 * i + 1] * r, acc[d][4 * i + 2] * r, acc[d][4 * i + 3] * r};
      if (sum == 0.0f) y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      *reinterpret_cast<u32x2*>(out + 32 * d + 8 * i) =
          u32x2{pack_out<QT>(y[0], y[1]), pack_out<QT>(y[2], y[3])};
    }
  if (a.lse && h == 0)
    a.lse[orow] = sum == 0.0f ? neg_inf() : (base + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <int QT, int CT, int D>
void launch_prompt_d(const WindowArgs& a, const PagedView& c, int waves, hipStream_t st) {
  const dim3 grid((unsigned)(a.groups * a.tiles * a.splits));
  if constexpr (D < 256) {
    if (waves == 8) {
      hipLaunchKernelGGL((prompt_kernel<QT, CT, D, 8>), grid, dim3(8 * kWave), 0, st, a, c);
      return;
    }
  }
  hipLaunchKernelGGL((prompt_kernel<QT, CT, D, 4>), grid, dim3(4 * kWave), 0, st, a, c);
}

template <int QT, int CT>
void launch_prompt(const WindowArgs& a, const PagedView& c, int64_t D, int waves, hipStream_t st) {
  if (D == 32) launch_prompt_d<QT, CT, 32>(a, c, waves, st);
  else if (D == 64) launch_prompt_d<QT, CT, 64>(a, c, waves, st);
  else if (D == 128) launch_prompt_d<QT, CT, 128>(a, c, waves, st);
  else launch_prompt_d<QT, CT, 256>(a, c, waves, st);
}

}  // namespace
}  // namespace rp
