// Attention of one new token per sequence over a paged key-value cache.
//
// One workgroup per (sequence, query head): its waves take the keys in turn,
// a wave's lanes share a key's head dim, and each wave keeps a running
// maximum, sum and output, joined at the end.

#include "rp_paged_dev.h"

namespace rp {
namespace {

constexpr int kDThreads = 256;

struct DecodeArgs {
  const uint16_t* q;
  int64_t qsb, qsh;
  const int32_t* lens;
  float scale;
  uint16_t* out;
  int64_t osb, osh;
  float* lse;
  float* weights;
  int64_t wsb, wsh;
  int32_t H, group;
};

__device__ __forceinline__ float e4m3_to_f32(uint32_t code) {
  return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}

// Element d of cache row `row` (element offset).
template <int CT>
__device__ __forceinline__ float cache_elem(const char* p, int64_t row, int d) {
  if constexpr (CT == RP_CACHE_E4M3) return e4m3_to_f32(reinterpret_cast<const uint8_t*>(p)[row + d]);
  else return in_to_f32<CT>(reinterpret_cast<const uint16_t*>(p)[row + d]);
}

template <int QT, int CT, int D>
__global__ __launch_bounds__(kDThreads) void decode_kernel(DecodeArgs a, PagedView c) {
  constexpr int E = (D + kWave - 1) / kWave, kWaves = kDThreads / kWave;
  __shared__ float sm[kWaves], sl[kWaves], so[kWaves][D];
  const int h = blockIdx.x, b = blockIdx.y, kv = h / a.group;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int n = (int)paged_len(c, a.lens[b]);
  const int32_t* table = c.table + b * c.table_stride;
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + e * kWave;
    q[e] = d < D ? in_to_f32<QT>(a.q[b * a.qsb + h * a.qsh + d]) * a.scale : 0.0f;
    o[e] = 0.0f;
  }
  float m = -__builtin_inff(), l = 0.0f;
  for (int j = wave; j < n; j += kWaves) {
    const int32_t page = paged_page(c, table, j);
    if (page < 0) continue;
    const int64_t row = paged_row(c, page, kv, j);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + e * kWave;
      if (d < D) s += q[e] * cache_elem<CT>(c.k, row, d);
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) s += __shfl_xor(s, x, kWave);
    float vs = 1.0f;
    if constexpr (CT == RP_CACHE_E4M3) {
      s *= c.ks[paged_scale(c, page, kv, j)];
      vs = c.vs[paged_scale(c, page, kv, j)];
    }
    const float mn = fmaxf(m, s), base = mn == -__builtin_inff() ? 0.0f : mn;
    const float r = expf(m - base), p = expf(s - base);
    l = l * r + p;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + e * kWave;
      if (d < D) o[e] = o[e] * r + p * (vs * cache_elem<CT>(c.v, row, d));
    }
    m = mn;
  }
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + e * kWave < D) so[wave][lane + e * kWave] = o[e];
  __syncthreads();
  float mt = sm[0], lt = 0.0f;
  for (int w = 1; w < kWaves; ++w) mt = fmaxf(mt, sm[w]);
  const float base = mt == -__builtin_inff() ? 0.0f : mt;
  for (int w = 0; w < kWaves; ++w) lt += sl[w] * expf(sm[w] - base);
  for (int d = threadIdx.x; d < D; d += kDThreads) {
    float x = 0.0f;
    for (int w = 0; w < kWaves; ++w) x += so[w][d] * expf(sm[w] - base);
    x = lt == 0.0f ? 0.0f : x / lt;
    a.out[b * a.osb + h * a.osh + d] =
        QT == kInF16 ? __builtin_bit_cast(uint16_t, (_Float16)x) : (uint16_t)f32_to_bf16_bits(x);
  }
  if (threadIdx.x == 0 && a.lse) a.lse[(int64_t)b * a.H + h] = lt == 0.0f ? -__builtin_inff() : base + logf(lt);
}

// Adds each seen key's weights: a thread per key.
template <int QT, int CT, int D>
__global__ __launch_bounds__(kDThreads) void decode_weights_kernel(DecodeArgs a, PagedView c) {
  const int kv = blockIdx.y, b = blockIdx.z;
  const int j = blockIdx.x * kDThreads + threadIdx.x;
  if (j >= (int)paged_len(c, a.lens[b])) return;
  const int32_t page = paged_page(c, c.table + b * c.table_stride, j);
  if (page < 0) return;
  const int64_t row = paged_row(c, page, kv, j);
  float w = 0.0f;
  for (int i = 0; i < a.group; ++i) {
    const int h = kv * a.group + i;
    float s = 0.0f;
    for (int d = 0; d < D; ++d)
      s += in_to_f32<QT>(a.q[b * a.qsb + h * a.qsh + d]) * a.scale * cache_elem<CT>(c.k, row, d);
    if constexpr (CT == RP_CACHE_E4M3) s *= c.ks[paged_scale(c, page, kv, j)];
    const float lse = a.lse[(int64_t)b * a.H + h];
    w += lse == -__builtin_inff() ? 0.0f : expf(s - lse);
  }
  a.weights[b * a.wsb + kv * a.wsh + j] += w;
}

template <int QT, int CT, int D>
void launch_decode_d(const DecodeArgs& a, const PagedView& c, int64_t B, hipStream_t st) {
  hipLaunchKernelGGL((decode_kernel<QT, CT, D>), dim3((unsigned)a.H, (unsigned)B), dim3(kDThreads),
                     0, st, a, c);
  if (a.weights)
    hipLaunchKernelGGL((decode_weights_kernel<QT, CT, D>),
                       dim3((unsigned)((c.capacity() + kDThreads - 1) / kDThreads),
                            (unsigned)c.heads, (unsigned)B),
                       dim3(kDThreads), 0, st, a, c);
}

template <int QT, int CT>
void launch_decode(const DecodeArgs& a, const PagedView& c, int64_t B, int64_t D, hipStream_t st) {
  if (D == 32) launch_decode_d<QT, CT, 32>(a, c, B, st);
  else if (D == 64) launch_decode_d<QT, CT, 64>(a, c, B, st);
  else if (D == 128) launch_decode_d<QT, CT, 128>(a, c, B, st);
  else launch_decode_d<QT, CT, 256>(a, c, B, st);
}

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" size_t rp_paged_attn_workspace_bytes(int64_t B, int64_t H, const rp_paged_cache* cache,
                                                int64_t max_seq_len, int with_key_weights) {
  (void)max_seq_len;
  if (!cache || B <= 0 || H <= 0) return 0;
  return with_key_weights ? (size_t)(B * H * 4) : 0;
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
  if (!(sm_scale - sm_scale == 0.0f)) {
    rp_set_error("paged_attn_decode: sm_scale must be finite");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B > 65535 || H > 65535) {
    rp_set_error("paged_attn_decode: too many sequences or heads");
    return RP_ERR_UNSUPPORTED;
  }
  if (((qsb | qsh) & 7) != 0 || ((osb | osh) & 3) != 0 ||
      (reinterpret_cast<uintptr_t>(q) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 7) != 0) {
    rp_set_error("paged_attn_decode: q rows must be 16-byte and out rows 8-byte aligned");
    return RP_ERR_UNSUPPORTED;
  }
  if (key_weights && (wsb < 0 || wsh < 0)) {
    rp_set_error("paged_attn_decode: bad key_weights strides");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const size_t want = rp_paged_attn_workspace_bytes(B, H, cache, max_seq_len, key_weights != nullptr);
  if (want > 0 && (!workspace || workspace_bytes < want ||
                   (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)) {
    rp_set_error("paged_attn_decode: workspace of %zu bytes, 256-byte aligned, needed", want);
    return RP_ERR_WORKSPACE;
  }
  if (!lse && key_weights) lse = static_cast<float*>(workspace);
  const DecodeArgs a{static_cast<const uint16_t*>(q), qsb, qsh, seq_lens, sm_scale,
                     static_cast<uint16_t*>(out), osb, osh, lse, key_weights, wsb, wsh,
                     (int32_t)H, (int32_t)(H / cache->heads)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t D = cache->head_dim;
  if (q_dtype == RP_DTYPE_F16) {
    if (fp8) launch_decode<kInF16, RP_CACHE_E4M3>(a, c, B, D, st);
    else launch_decode<kInF16, RP_CACHE_F16>(a, c, B, D, st);
  } else {
    if (fp8) launch_decode<kInBf16, RP_CACHE_E4M3>(a, c, B, D, st);
    else launch_decode<kInBf16, RP_CACHE_BF16>(a, c, B, D, st);
  }
  return paged_launched("paged_attn_decode");
}
