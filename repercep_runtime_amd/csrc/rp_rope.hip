// RMSNorm of each head of Q and K, and their rotation by position, in one
// pass: 16-bit rows in, 16-bit rows out.
//
//   y = x / sqrt(mean x^2 + eps) * weight
//   pair j of y (j < rot / 2; j and j + rot / 2, or 2 j and 2 j + 1) turned by
//   the angle position[axis of j] * freq[j], the rest as it is
//
// The floor is one read and one write of the rows.  D / 16 lanes hold a row,
// 16 values each: the halves of eight pairs, so a rotation stays inside its
// lane and only the sum of squares crosses lanes (a DPP butterfly).  A wave
// takes 1024 / D tokens, one a lane group, and goes through their heads: a
// lane's eight angles are computed once a token, whatever the number of heads,
// and the wave's rows of one head lie next to each other in the output.
//
// Bound by HBM: queries and keys of 75600 tokens, 40 heads of 128 each, in 626 us,
// 5.0 TB/s (a copy of 4 GiB reaches 4.7); 16 tokens of a decoder's step in 5.2 us,
// a launch and its dependent loads.
//
// Angles are products in 64 bits, in turns, whose fraction is exact to 2^-24
// at any 32-bit position; their sines and cosines, the norm and the rotation
// are in fp32, and the result is rounded once.

#include "rp_common.h"

namespace rp {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMaxAxes = RP_ROPE_MAX_AXES;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct RopeRows {
  const uint16_t* x;
  uint16_t* y;
  const uint16_t* weight;        // (D), or null: ones
  int64_t sb, sh, ss, ob, oh, os;
};

struct RopeArgs {
  RopeRows rows[2];              // Q and K
  const int32_t* pos;
  int64_t psa, psb, pss;
  const void* freq;              // float or double (rot / 2)
  int32_t freq64;
  int32_t ends[kMaxAxes];        // pairs below ends[a] (and not below ends[a - 1]) turn by axis a
  int32_t axes, rot;
  int64_t tokens, S;
  int32_t H, heads;              // query heads; with the kv heads
  int32_t per, chunks;           // heads a wave, waves a token group
  float eps;
};

template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (DT == kInF16) return pack_f16x2(lo, hi);
  else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
  }
}

template <int DT>
__device__ __forceinline__ void unpack16(const u32x4& w, float* to) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    to[e] = in_to_f32<DT>(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
}

// The sum over the L = D / 16 lanes of a row, in each of them.
template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o >= 1; o /= 2) v += __shfl_xor(v, o, kWave);
  return v;
}

template <int DT, int D, bool HALF, bool NORM>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
  constexpr int L = D / 16, T = kWave / L;          // lanes a row, tokens a wave
  const int lane = threadIdx.x & (kWave - 1), li = lane % L;
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t group = wave / a.chunks;
  const int h0 = (int)(wave % a.chunks) * a.per, h1 = min(a.heads, h0 + a.per);
  const int64_t token = group * T + lane / L;
  if (token >= a.tokens) return;                    // whole lane groups leave
  const int64_t b = token / a.S, s = token % a.S;

  // the lane's two runs of eight values, and whether they are halves of pairs
  const bool turned = 16 * li < a.rot;
  const int d0 = HALF && turned ? 8 * li : 16 * li;
  const int d1 = HALF && turned ? a.rot / 2 + 8 * li : 16 * li + 8;
  float cs[8], sn[8];
  if (turned) {
    const int32_t* pos = a.pos + b * a.psb + s * a.pss;
    int32_t p[kMaxAxes];
#pragma unroll
    for (int i = 0; i < kMaxAxes; ++i) p[i] = i < a.axes ? pos[i * a.psa] : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = 8 * li + e;
      const double f = a.freq64 ? static_cast<const double*>(a.freq)[j]
                                : (double)static_cast<const float*>(a.freq)[j];
      int32_t at = p[0];
#pragma unroll
      for (int i = 1; i < kMaxAxes; ++i) at = j >= a.ends[i - 1] ? p[i] : at;
      constexpr double kTurns = 0.15915494309189533577;     // 1 / (2 pi)
      const double t = (double)at * (f * kTurns);
      sincospif(2.0f * (float)(t - __builtin_rint(t)), &sn[e], &cs[e]);
    }
  }

  u32x4 next[2];
  auto load = [&](int h) {
    const RopeRows& r = a.rows[h < a.H ? 0 : 1];
    const uint16_t* x = r.x + b * r.sb + (int64_t)(h < a.H ? h : h - a.H) * r.sh + s * r.ss;
    next[0] = *reinterpret_cast<const u32x4*>(x + d0);
    next[1] = *reinterpret_cast<const u32x4*>(x + d1);
  };
  float w[16];
  int of = -1;                                      // whose weight w holds
  load(h0);
  for (int h = h0; h < h1; ++h) {
    const int which = h < a.H ? 0 : 1;
    const RopeRows& r = a.rows[which];
    float x[16];
    unpack16<DT>(next[0], x);
    unpack16<DT>(next[1], x + 8);
    if (h + 1 < h1) load(h + 1);
    if constexpr (NORM) {
      if (which != of) {
        of = which;
        if (r.weight) {
          unpack16<DT>(*reinterpret_cast<const u32x4*>(r.weight + d0), w);
          unpack16<DT>(*reinterpret_cast<const u32x4*>(r.weight + d1), w + 8);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = 1.0f;
        }
      }
      float scale = 1.0f, eps = a.eps, mean;
      for (;;) {                                    // at most twice
        float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 16; ++e) q[e % 4] = __builtin_fmaf(x[e], x[e], q[e % 4]);
        mean = row_sum<L>((q[0] + q[1]) + (q[2] + q[3])) * (1.0f / D) + eps;
        if (scale != 1.0f) break;
        // squares that leave fp32's range are taken again of scaled values
        if (mean == __builtin_inff()) scale = 0x1p-80f;
        else if (mean < 0x1p-80f) scale = 0x1p90f;
        else break;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= scale;
        eps *= scale;
        eps *= scale;
      }
      const float rs = __builtin_amdgcn_rsqf(mean);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = x[e] * rs * w[e];
    }
    u32x4 y[2];
    if (turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = HALF ? e : 2 * e, j = HALF ? e + 8 : 2 * e + 1;
        const float u = x[i], v = x[j];
        x[i] = u * cs[e] - v * sn[e];
        x[j] = v * cs[e] + u * sn[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[0][e] = pack16<DT>(x[2 * e], x[2 * e + 1]);
      y[1][e] = pack16<DT>(x[8 + 2 * e], x[9 + 2 * e]);
    }
    uint16_t* out = r.y + b * r.ob + (int64_t)(which ? h - a.H : h) * r.oh + s * r.os;
    *reinterpret_cast<u32x4*>(out + d0) = y[0];
    *reinterpret_cast<u32x4*>(out + d1) = y[1];
  }
}

template <int DT, int D>
void launch_rope(const RopeArgs& a, bool half, bool norm, unsigned blocks, hipStream_t st) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, st, a);
  };
  if (half) norm ? go(rope_kernel<DT, D, true, true>) : go(rope_kernel<DT, D, true, false>);
  else norm ? go(rope_kernel<DT, D, false, true>) : go(rope_kernel<DT, D, false, false>);
}

template <int DT>
void launch_rope(const RopeArgs& a, int64_t D, bool half, bool norm, unsigned blocks,
                 hipStream_t st) {
  if (D == 32) launch_rope<DT, 32>(a, half, norm, blocks, st);
  else if (D == 64) launch_rope<DT, 64>(a, half, norm, blocks, st);
  else if (D == 128) launch_rope<DT, 128>(a, half, norm, blocks, st);
  else launch_rope<DT, 256>(a, half, norm, blocks, st);
}

// Heads a wave: eight at most, fewer where that leaves less than 2048 waves, two a
// SIMD.  75600 tokens of 80 heads take 626 us at eight (5.0 TB/s), 655 at four,
// 636 at twelve, 663 at forty; 8188 tokens of 40 heads of 64 17.5 us at eight,
// 24.9 at one.
constexpr int64_t kWavesWanted = 2048, kHeadsMost = 8;

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" int rp_qk_norm_rope(const void* q, const void* k, int dtype, int64_t B, int64_t S,
                               int64_t H, int64_t Hkv, int64_t D, int64_t qsb, int64_t qsh,
                               int64_t qss, int64_t ksb, int64_t ksh, int64_t kss,
                               const void* q_weight, const void* k_weight, int norm, float eps,
                               const int32_t* positions, int64_t psa, int64_t psb, int64_t pss,
                               const void* freq, int freq_is_double, int64_t rot,
                               const int64_t* sections, int axes, int rope_mode, void* q_out,
                               int64_t qob, int64_t qoh, int64_t qos, void* k_out, int64_t kob,
                               int64_t koh, int64_t kos, void* stream) {
  if (!q || !q_out || !positions || !freq || !sections || (Hkv > 0 && (!k || !k_out))) {
    rp_set_error("qk_norm_rope: null pointer");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (dtype != RP_DTYPE_BF16 && dtype != RP_DTYPE_F16) {
    rp_set_error("qk_norm_rope: unknown dtype %d", dtype);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B <= 0 || S <= 0 || H <= 0 || Hkv < 0) {
    rp_set_error("qk_norm_rope: non-positive size (B=%lld S=%lld H=%lld Hkv=%lld)", (long long)B,
                 (long long)S, (long long)H, (long long)Hkv);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (D != 32 && D != 64 && D != 128 && D != 256) {
    rp_set_error("qk_norm_rope: head dim %lld not in {32, 64, 128, 256}", (long long)D);
    return RP_ERR_UNSUPPORTED;
  }
  if (rope_mode != RP_ROPE_HALF && rope_mode != RP_ROPE_INTERLEAVED) {
    rp_set_error("qk_norm_rope: unknown rope mode %d", rope_mode);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (rot <= 0 || rot > D || rot % 16 != 0) {
    rp_set_error("qk_norm_rope: %lld rotated dims are not a multiple of 16 up to %lld",
                 (long long)rot, (long long)D);
    return RP_ERR_UNSUPPORTED;
  }
  if (axes < 1 || axes > kMaxAxes) {
    rp_set_error("qk_norm_rope: %d axes not in [1, %d]", axes, kMaxAxes);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (norm && !(eps >= 0.0f && eps - eps == 0.0f)) {
    rp_set_error("qk_norm_rope: eps must be finite and not negative");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (!norm && (q_weight || k_weight)) {
    rp_set_error("qk_norm_rope: weights without a norm");
    return RP_ERR_INVALID_ARGUMENT;
  }
  RopeArgs a{};
  int64_t pairs = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    if (i < axes) {
      if (sections[i] < 0) {
        rp_set_error("qk_norm_rope: negative section");
        return RP_ERR_INVALID_ARGUMENT;
      }
      pairs += sections[i] > rot ? rot : sections[i];
    }
    a.ends[i] = i < axes - 1 ? (int32_t)pairs : 0x7fffffff;
  }
  if (pairs != rot / 2) {
    rp_set_error("qk_norm_rope: sections add up to %lld pairs, not %lld", (long long)pairs,
                 (long long)(rot / 2));
    return RP_ERR_INVALID_ARGUMENT;
  }
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                          reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out) |
                          reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight);
  if ((bases & 15) != 0 || ((qsb | qsh | qss | ksb | ksh | kss | qob | qoh | qos | kob | koh | kos) & 7) != 0) {
    rp_set_error("qk_norm_rope: rows and weights must be 16-byte aligned");
    return RP_ERR_UNSUPPORTED;
  }
  if ((reinterpret_cast<uintptr_t>(freq) & (freq_is_double ? 7 : 3)) != 0) {
    rp_set_error("qk_norm_rope: freq must be aligned to its type");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B > 0x7fffffff || S > 0x7fffffff / B || H > 65535 || Hkv > 65535) {
    rp_set_error("qk_norm_rope: too many tokens or heads");
    return RP_ERR_UNSUPPORTED;
  }
  if (!rows_apart(D, {{B, qob}, {H, qoh}, {S, qos}}) ||
      (Hkv > 0 && !rows_apart(D, {{B, kob}, {Hkv, koh}, {S, kos}}))) {
    rp_set_error("qk_norm_rope: output rows overlap");
    return RP_ERR_INVALID_ARGUMENT;
  }
  // Waves run in any order: what one writes no other may read or write.  A row is
  // read by the lanes that write it, so an output can take its own input's place.
  const RowSet in[] = {{q, 2 * D, {{B, 2 * qsb}, {H, 2 * qsh}, {S, 2 * qss}}},
                       {k, 2 * D, {{B, 2 * ksb}, {Hkv, 2 * ksh}, {S, 2 * kss}}},
                       whole(q_weight, 2 * D),
                       whole(k_weight, 2 * D),
                       {positions, 4, {{axes, 4 * psa}, {B, 4 * psb}, {S, 4 * pss}}},
                       whole(freq, (freq_is_double ? 4 : 2) * rot)};
  const RowSet to[] = {{q_out, 2 * D, {{B, 2 * qob}, {H, 2 * qoh}, {S, 2 * qos}}},
                       {k_out, 2 * D, {{B, 2 * kob}, {Hkv, 2 * koh}, {S, 2 * kos}}}};
  if (outputs_meet(to, in, 2)) {
    rp_set_error("qk_norm_rope: an output shares memory with another array, or with its input at "
                 "other strides");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const int64_t tokens_a_wave = kWave / (D / 16);
  a.rows[0] = RopeRows{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(q_out),
                       static_cast<const uint16_t*>(q_weight), qsb, qsh, qss, qob, qoh, qos};
  a.rows[1] = RopeRows{static_cast<const uint16_t*>(k), static_cast<uint16_t*>(k_out),
                       static_cast<const uint16_t*>(k_weight), ksb, ksh, kss, kob, koh, kos};
  a.pos = positions;
  a.psa = psa;
  a.psb = psb;
  a.pss = pss;
  a.freq = freq;
  a.freq64 = freq_is_double != 0;
  a.axes = axes;
  a.rot = (int32_t)rot;
  a.tokens = B * S;
  a.S = S;
  a.H = (int32_t)H;
  a.heads = (int32_t)(H + Hkv);
  a.eps = eps;
  const int64_t groups = (a.tokens + tokens_a_wave - 1) / tokens_a_wave;
  int64_t chunks = (kWavesWanted + groups - 1) / groups;
  if (chunks < (a.heads + kHeadsMost - 1) / kHeadsMost) chunks = (a.heads + kHeadsMost - 1) / kHeadsMost;
  if (chunks > a.heads) chunks = a.heads;
  a.per = (int32_t)((a.heads + chunks - 1) / chunks);
  a.chunks = (a.heads + a.per - 1) / a.per;
  const int64_t blocks = (groups * a.chunks + kWaves - 1) / kWaves;
  if (blocks * kThreads > kMaxGridThreads) {
    rp_set_error("qk_norm_rope: too many tokens or heads");
    return RP_ERR_UNSUPPORTED;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool half = rope_mode == RP_ROPE_HALF;
  if (dtype == RP_DTYPE_F16) launch_rope<kInF16>(a, D, half, norm != 0, (unsigned)blocks, st);
  else launch_rope<kInBf16>(a, D, half, norm != 0, (unsigned)blocks, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    rp_set_error("qk_norm_rope: launch failed: %s", hipGetErrorString(e));
    return RP_ERR_LAUNCH;
  }
  return RP_OK;
}
