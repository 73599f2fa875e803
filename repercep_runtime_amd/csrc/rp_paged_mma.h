// What the attention kernels over a paged cache share beside the cache itself:
// operand types, 16-bit matrix products, e4m3fn codes as 16-bit floats, a step's
// rows in a wave's registers.
// Everything here has internal linkage.
#pragma once

#include "rp_paged_dev.h"

namespace rp {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.693147180559945309f;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

template <bool F16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two e4m3fn codes of a dword (its low or high half) as a pair of 16-bit
// floats, exact: e4m3fn is a subset of both.
template <bool F16, bool HI>
__device__ __forceinline__ uint32_t codes_to_16(uint32_t w) {
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
}

__device__ __forceinline__ float bf16_cut(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_cut(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

constexpr int kStep = 32;                       // keys per step of a wave

// The K and V rows of a step in a wave's registers, for products with columns
// of 16 query rows.  Lane g * 16 + m brings K's rows m and 16 + m, a part of
// each, and of V's rows 4 g + 0..3 and 16 + 4 g + 0..3 the columns column(m, j).
template <bool QF16, int CT, int D, bool STREAM>
struct StepRows {
  static constexpr bool FP8 = CT == RP_CACHE_E4M3;
  static constexpr int EB = FP8 ? 1 : 2;
  static constexpr int NT = D / 32;                   // first products per 16 keys
  static constexpr int DPL = D / 16;                  // V columns per lane
  static constexpr int KL = FP8 ? (D + 63) / 64 : NT; // 16-byte K loads per 16 keys (8 at D = 32, fp8)
  static constexpr int VB = DPL * EB;                 // V bytes per lane and row
  static constexpr int VW = VB < 4 ? 1 : VB / 4;

  const PagedView& c;
  int lane, m, g;
  int64_t head;                  // kv head
  uint32_t koff, voff[4];        // byte offsets of a lane's rows within a tile of 16
  u32x4 kr[2][KL];
  uint32_t vr[8][VW];
  f32x4 kscale[2], vscale[2];

  __device__ __forceinline__ explicit StepRows(const PagedView& c_) : c(c_) {}

  __device__ __forceinline__ void place(int lane_, int64_t head_) {
    lane = lane_;
    m = lane & 15;
    g = lane >> 4;
    head = head_;
    koff = (uint32_t)(m * c.sr * EB);
#pragma unroll
    for (int r = 0; r < 4; ++r) voff[r] = (uint32_t)((4 * g + r) * c.sr * EB) + v_col();
  }

  // The lane's eight keys of the step at k, as its scores and V rows count them.
  __device__ __forceinline__ int key(int k, int e) const {
    return k + 4 * g + (e < 4 ? e : 12 + e);
  }

  __device__ __forceinline__ void k_row(const char* p, int half) {
    if constexpr (FP8 && D == 32) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p + 8 * g);
      kr[half][0] = u32x4{x[0], x[1], 0u, 0u};
    } else {
#pragma unroll
      for (int t = 0; t < KL; ++t)
        kr[half][t] = *reinterpret_cast<const u32x4*>(p + 64 * t + 16 * g);
    }
  }

  template <typename T>
  __device__ __forceinline__ static T v_load(const char* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
    else return *reinterpret_cast<const T*>(p);
  }

  __device__ __forceinline__ void v_row(const char* p, int e) {
    if constexpr (VB == 2) {
      vr[e][0] = v_load<uint16_t>(p);
    } else if constexpr (VB == 4) {
      vr[e][0] = v_load<uint32_t>(p);
    } else if constexpr (VB == 8) {
      const u32x2 x = v_load<u32x2>(p);
      vr[e][0] = x[0];
      vr[e][1] = x[1];
    } else {
#pragma unroll
      for (int i = 0; i < VB / 16; ++i) {
        const u32x4 x = v_load<u32x4>(p + 256 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) vr[e][4 * i + j] = x[j];
      }
    }
  }

  // Bytes of a lane's first column, and the column of its value j.
  __device__ __forceinline__ int v_col() const { return m * (VB > 16 ? 16 : VB); }
  __device__ __forceinline__ static int column(int mm, int j) {
    if constexpr (VB > 16) return (j < 8 ? 0 : 128) + 8 * mm + j % 8;
    else return mm * DPL + j;
  }

  // The tile `half` of the step, all in one page: the 16 keys at k.
  __device__ __forceinline__ void load_k16(int half, int32_t page, int k) {
    const char* tile = c.k + paged_row(c, page, head, k) * EB;
    k_row(tile + koff, half);
    if constexpr (FP8)
      kscale[half] = *reinterpret_cast<const f32x4*>(c.ks + paged_scale(c, page, head, k) + 4 * g);
  }
  __device__ __forceinline__ void load_v16(int half, int32_t page, int k) {
    const char* tile = c.v + paged_row(c, page, head, k) * EB;
#pragma unroll
    for (int r = 0; r < 4; ++r) v_row(tile + voff[r], 4 * half + r);
    if constexpr (FP8)
      vscale[half] = *reinterpret_cast<const f32x4*>(c.vs + paged_scale(c, page, head, k) + 4 * g);
  }

  // The step at k with each row's page from page(position).
  template <typename F>
  __device__ __forceinline__ void load_k_any(F page, int k) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int j = k + 16 * half + m;
      k_row(c.k + paged_row(c, page(j), head, j) * EB, half);
    }
    if constexpr (FP8) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        kscale[e / 4][e % 4] = c.ks[paged_scale(c, page(key(k, e)), head, key(k, e))];
    }
  }
  template <typename F>
  __device__ __forceinline__ void load_v_any(F page, int k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int32_t p = page(key(k, e));
      v_row(c.v + paged_row(c, p, head, key(k, e)) * EB + v_col(), e);
      if constexpr (FP8) vscale[e / 4][e % 4] = c.vs[paged_scale(c, p, head, key(k, e))];
    }
  }

  // Operand words of K's fragment t of a half step.
  __device__ __forceinline__ u32x4 k_frag(int half, int t) const {
    if constexpr (!FP8) {
      return kr[half][t];
    } else {
      const u32x4& x = kr[half][t / 2];
      const uint32_t w0 = t % 2 ? x[2] : x[0], w1 = t % 2 ? x[3] : x[1];
      return u32x4{codes_to_16<QF16, false>(w0), codes_to_16<QF16, true>(w0),
                   codes_to_16<QF16, false>(w1), codes_to_16<QF16, true>(w1)};
    }
  }
};

}  // namespace
}  // namespace rp
