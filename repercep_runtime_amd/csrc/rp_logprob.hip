// Token log probabilities, entropy and the best alternatives of rows of logits.
//
// One workgroup per row: the maximum, then the sums over exp(z - max), then
// the best logits one after another.

#include "rp_common.h"

namespace rp {
namespace {

constexpr int kLThreads = 256;
constexpr int kLWaves = kLThreads / kWave;

struct LogprobArgs {
  const void* x;
  int64_t ld;
  int32_t V, top;
  const int64_t* tokens;
  float temperature;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
};

template <int DT>
__device__ __forceinline__ float logit(const void* x, int64_t i) {
  if constexpr (DT == RP_OUT_F32) return static_cast<const float*>(x)[i];
  else return in_to_f32<DT == RP_OUT_F16 ? kInF16 : kInBf16>(static_cast<const uint16_t*>(x)[i]);
}

// fp32 -> an unsigned key in the same order; -0 as 0, NaN above everything.
__device__ __forceinline__ uint32_t logit_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (x == 0.0f) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int DT>
__global__ __launch_bounds__(kLThreads) void logprob_kernel(LogprobArgs a) {
  __shared__ float red[3][kLWaves];
  __shared__ uint64_t redk[kLWaves];
  const int64_t row = blockIdx.x;
  const int64_t base = row * a.ld;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  float m = -__builtin_inff();
  for (int i = threadIdx.x; i < a.V; i += kLThreads) m = fmaxf(m, logit<DT>(a.x, base + i) / a.temperature);
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  for (int w = 0; w < kLWaves; ++w) m = fmaxf(m, red[0][w]);
  if (m == -__builtin_inff()) m = 0.0f;   // no logit above -inf: every weight is 0
  float s = 0.0f, sz = 0.0f;
  for (int i = threadIdx.x; i < a.V; i += kLThreads) {
    const float z = __builtin_elementwise_maximum(logit<DT>(a.x, base + i) / a.temperature - m, -200.0f);
    const float e = expf(z);
    s += e;
    sz += e * z;
  }
  for (int o = 32; o >= 1; o >>= 1) {
    s += __shfl_xor(s, o, kWave);
    sz += __shfl_xor(sz, o, kWave);
  }
  if (lane == 0) {
    red[1][wave] = s;
    red[2][wave] = sz;
  }
  __syncthreads();
  s = sz = 0.0f;
  for (int w = 0; w < kLWaves; ++w) {
    s += red[1][w];
    sz += red[2][w];
  }
  const bool none = s == 0.0f;
  const float lg = logf(s);
  if (threadIdx.x == 0) {
    const int64_t t = a.tokens[row];
    float lp = 0.0f;
    if (t >= a.V) lp = __builtin_nanf("");
    else if (t >= 0) lp = none ? -__builtin_inff() : logit<DT>(a.x, base + t) / a.temperature - m - lg;
    a.logprobs[row] = lp;
    if (a.entropy) a.entropy[row] = none ? 0.0f : lg - sz / s;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.V; i += kLThreads) {
      const uint64_t key = ((uint64_t)logit_key(logit<DT>(a.x, base + i)) << 32) | (0xffffffffu - (uint32_t)i);
      if (key < last && key > best) best = key;
    }
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, o, kWave);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) redk[wave] = best;
    __syncthreads();
    for (int w = 0; w < kLWaves; ++w) best = redk[w] > best ? redk[w] : best;
    last = best;
    if (threadIdx.x == 0) {
      const int64_t id = 0xffffffffu - (uint32_t)best;
      a.top_ids[row * a.top + k] = id;
      a.top_logprobs[row * a.top + k] =
          none ? -__builtin_inff() : logit<DT>(a.x, base + id) / a.temperature - m - lg;
    }
  }
}

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" size_t rp_token_logprobs_workspace_bytes(int64_t N, int64_t V, int logits_dtype,
                                                    int top) {
  (void)N; (void)V; (void)logits_dtype; (void)top;
  return 0;
}

extern "C" int rp_token_logprobs(const void* logits, int logits_dtype, int64_t N, int64_t V,
                                 int64_t ld, const int64_t* tokens, float temperature, int top,
                                 float* logprobs, float* entropy, float* top_logprobs,
                                 int64_t* top_ids, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!logits || !tokens || !logprobs || (top > 0 && (!top_logprobs || !top_ids))) {
    rp_set_error("token_logprobs: null pointer");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (logits_dtype != RP_OUT_BF16 && logits_dtype != RP_OUT_F16 && logits_dtype != RP_OUT_F32) {
    rp_set_error("token_logprobs: unknown logits dtype %d", logits_dtype);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (N <= 0 || V <= 0 || ld < V) {
    rp_set_error("token_logprobs: bad sizes N=%lld V=%lld ld=%lld", (long long)N, (long long)V,
                 (long long)ld);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (top < 0 || top > RP_LOGPROB_MAX_TOP || top > V) {
    rp_set_error("token_logprobs: top %d not in [0, min(%d, V)]", top, RP_LOGPROB_MAX_TOP);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (!(temperature > 0.0f) || !(temperature - temperature == 0.0f)) {
    rp_set_error("token_logprobs: temperature must be positive and finite");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (N > 0x7fffffff || V > 0x7fffff00) {
    rp_set_error("token_logprobs: too many rows or logits");
    return RP_ERR_UNSUPPORTED;
  }
  (void)workspace; (void)workspace_bytes;
  const LogprobArgs a{logits, ld, (int32_t)V, top, tokens, temperature, logprobs, entropy,
                      top_logprobs, top_ids};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 g((unsigned)N), t(kLThreads);
  if (logits_dtype == RP_OUT_F32) hipLaunchKernelGGL(logprob_kernel<RP_OUT_F32>, g, t, 0, st, a);
  else if (logits_dtype == RP_OUT_F16) hipLaunchKernelGGL(logprob_kernel<RP_OUT_F16>, g, t, 0, st, a);
  else hipLaunchKernelGGL(logprob_kernel<RP_OUT_BF16>, g, t, 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    rp_set_error("token_logprobs: launch failed: %s", hipGetErrorString(e));
    return RP_ERR_LAUNCH;
  }
  return RP_OK;
}
