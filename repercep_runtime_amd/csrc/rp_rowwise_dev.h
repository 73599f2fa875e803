// Device bodies of the row-wise e4m3fn quantizer, shared by the row-wise
// entry points (rp_rowwise.hip) and the paged cache's writer (rp_paged.hip),
// so a row has the same codes and scale through both.  Everything here has
// internal linkage.
#pragma once

#include "rp_common.h"

namespace rp {
namespace {

typedef unsigned int u32x4r __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2r __attribute__((ext_vector_type(2)));

// qmul and dequant of a row from the bit pattern of its |x| maximum.
template <int DT>
__device__ __forceinline__ void rowwise_scales(uint32_t amax_bits, float* qmul, float* dequant) {
  if constexpr (DT == kInF16) {
    const float lo = 17.0f * 0x1p-24f;  // fp16(1e-6)
    float a = f16_to_f32(amax_bits);
    if (!(a != a) && a < lo) a = lo;
    const float r = f16_round(1.0f / a);
    *qmul = f16_round(r * kScaleDivisor);
    *dequant = f16_round(a * (1.0f / kScaleDivisor));
  } else {
    const float lo = __uint_as_float(0x3586u << 16);  // bf16(1e-6)
    float a = bf16_to_f32(amax_bits);
    if (!(a != a) && a < lo) a = lo;
    const float r = bf16_round(1.0f / a);
    *qmul = bf16_round(r * kScaleDivisor);
    *dequant = bf16_round(a / kScaleDivisor);
  }
}

__device__ __forceinline__ uint32_t pk_umax16r(uint32_t a, uint32_t b) {
  const uint32_t lo = umax32(a & 0xffffu, b & 0xffffu);
  const uint32_t hi = umax32(a >> 16, b >> 16);
  return lo | (hi << 16);
}

// Eight inputs (one 16-byte vector) -> eight codes.
template <int DT>
__device__ __forceinline__ uint2 quant8(const u32x4r& v, float qm) {
  uint2 o;
  const float a0 = clamp_e4m3(in_to_f32<DT>(v[0] & 0xffffu) * qm);
  const float a1 = clamp_e4m3(in_to_f32<DT>(v[0] >> 16) * qm);
  const float a2 = clamp_e4m3(in_to_f32<DT>(v[1] & 0xffffu) * qm);
  const float a3 = clamp_e4m3(in_to_f32<DT>(v[1] >> 16) * qm);
  const float a4 = clamp_e4m3(in_to_f32<DT>(v[2] & 0xffffu) * qm);
  const float a5 = clamp_e4m3(in_to_f32<DT>(v[2] >> 16) * qm);
  const float a6 = clamp_e4m3(in_to_f32<DT>(v[3] & 0xffffu) * qm);
  const float a7 = clamp_e4m3(in_to_f32<DT>(v[3] >> 16) * qm);
  o.x = pack4_e4m3(a0, a1, a2, a3);
  o.y = pack4_e4m3(a4, a5, a6, a7);
  return o;
}

__device__ __forceinline__ uint32_t absmax8(const u32x4r& v) {
  uint32_t m = pk_umax16r(v[0] & 0x7fff7fffu, v[1] & 0x7fff7fffu);
  m = pk_umax16r(m, pk_umax16r(v[2] & 0x7fff7fffu, v[3] & 0x7fff7fffu));
  return umax32(m & 0xffffu, m >> 16);
}

}  // namespace
}  // namespace rp
