// Drafted tokens verified against the target's probabilities, by given random
// numbers.
//
// Draft i of a sequence is accepted where u_i q_i(d_i) < p_i(d_i).  Behind the
// first n accepted ones a token is drawn from
//   w = max(p_n - q_n, 0)   (draft n rejected),   w = p_n   (all accepted):
// the lowest token t with w_0 + .. + w_t > u_N (w_0 + .. + w_{V-1}).
// Differences and sums are held in 64 bits: p - q of 32-bit numbers is exact
// there but for far smaller ones, and sums of another order move the border
// of two tokens by 2^-50 of the total, where 32-bit ones would give another
// token for about one draw in a hundred.
//
// Only row n of p and q is read whole (a test takes one value of each of the
// other rows), so the floor is those rows' bytes.  A row is cut into parts of
// kPart tokens: verify_sum_kernel finds n anew in each workgroup (three
// dependent loads, less than a launch) and adds up its part, verify_draw_kernel
// finds the part that the draw falls into and reads that part once more.

#include "rp_common.h"

namespace rp {
namespace {

constexpr int kSumThreads = 256, kPerSum = 16, kPart = kSumThreads * kPerSum;
constexpr int kDrawThreads = 1024, kPerDraw = kPart / kDrawThreads;
constexpr int64_t kMaxV = (int64_t)kPart * kDrawThreads;

struct VerifyArgs {
  const char* target;            // (B, N + 1, V)
  const char* draft;             // (B, N, V), or null: the drafts were certain
  int64_t tsb, tsn, dsb, dsn;    // element strides
  const int64_t* tokens;         // (B, N)
  const float* u;                // (B, N + 1)
  const int32_t* lens;           // (B), or null
  int32_t N, V, parts;
  int64_t* out;                  // (B, N + 1)
  int32_t* accepted;             // (B)
  double2* sums;                 // (B, parts): of w and of p
};

template <int DT>
__device__ __forceinline__ float prob_at(const char* row, int64_t i) {
  if constexpr (DT == RP_OUT_F32) return reinterpret_cast<const float*>(row)[i];
  else return in_to_f32<DT == RP_OUT_F16 ? kInF16 : kInBf16>(reinterpret_cast<const uint16_t*>(row)[i]);
}

// Values i .. i + 3 of a row of V, zeros past its end; rows are aligned to
// their type only.
template <int DT>
__device__ __forceinline__ void prob4(const char* row, int i, int V, float* to) {
  if (i + 4 <= V) {
    if constexpr (DT == RP_OUT_F32) {
      __builtin_memcpy(to, row + (int64_t)i * 4, 16);
    } else {
      uint32_t w[2];
      __builtin_memcpy(w, row + (int64_t)i * 2, 8);
      constexpr int K = DT == RP_OUT_F16 ? kInF16 : kInBf16;
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = in_to_f32<K>(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) to[e] = i + e < V ? prob_at<DT>(row, i + e) : 0.0f;
}

__device__ __forceinline__ int drafted(const VerifyArgs& a, int b) {
  return a.lens ? max(0, min(a.N, a.lens[b])) : a.N;
}

template <int DT>
__device__ __forceinline__ const char* target_row(const VerifyArgs& a, int b, int i) {
  return a.target + (b * a.tsb + i * a.tsn) * (DT == RP_OUT_F32 ? 4 : 2);
}
template <int DT>
__device__ __forceinline__ const char* draft_row(const VerifyArgs& a, int b, int i) {
  return a.draft + (b * a.dsb + i * a.dsn) * (DT == RP_OUT_F32 ? 4 : 2);
}

// How many of a sequence's n drafts are accepted; by one wave, a test a lane.
template <int DT>
__device__ __forceinline__ int count_accepted(const VerifyArgs& a, int b, int n, int lane) {
  for (int i0 = 0; i0 < n; i0 += kWave) {
    const int i = i0 + lane;
    bool ok = false;
    if (i < n) {
      const int64_t t = a.tokens[(int64_t)b * a.N + i];
      const float u = a.u[(int64_t)b * (a.N + 1) + i];
      if (t >= 0 && t < a.V) {
        const float p = prob_at<DT>(target_row<DT>(a, b, i), t);
        const float q = a.draft ? prob_at<DT>(draft_row<DT>(a, b, i), t) : 1.0f;
        ok = (double)u * (double)q < (double)p;       // the product is exact
      }
    }
    const uint64_t no = __ballot(!ok);
    if (no) return min(i0 + __builtin_ctzll(no), n);
  }
  return n;
}

// The weights that row n is drawn by.  A NaN weighs nothing.
template <int DT>
struct Weights {
  const char* p;
  const char* q;                 // null: nothing is taken off but at `one`
  int64_t one;                   // a certain draft that was rejected, or -1
  int V;

  __device__ __forceinline__ Weights(const VerifyArgs& a, int b, int n, bool rejected) {
    p = target_row<DT>(a, b, n);
    q = rejected && a.draft ? draft_row<DT>(a, b, n) : nullptr;
    one = rejected && !a.draft ? a.tokens[(int64_t)b * a.N + n] : -1;
    V = a.V;
  }
  // Weights and probabilities of tokens i .. i + 3.
  __device__ __forceinline__ void four(int i, double* w, double* pp) const {
    float x[4], y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    prob4<DT>(p, i, V, x);
    if (q) prob4<DT>(q, i, V, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e == one) y[e] = 1.0f;
      const double d = (double)x[e] - (double)y[e];
      w[e] = d > 0.0 ? d : 0.0;
      pp[e] = x[e] > 0.0f ? (double)x[e] : 0.0;
    }
  }
};

template <int DT>
__global__ __launch_bounds__(kSumThreads) void verify_sum_kernel(VerifyArgs a) {
  __shared__ double2 wave_sum[kSumThreads / kWave];
  const int part = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & (kWave - 1);
  const int has = drafted(a, b);
  const int n = __builtin_amdgcn_readfirstlane(count_accepted<DT>(a, b, has, lane));
  if (part == 0 && threadIdx.x == 0) a.accepted[b] = n;
  const Weights<DT> row(a, b, n, n < has);
  double sw = 0.0, sp = 0.0;
#pragma unroll
  for (int k = 0; k < kPerSum / 4; ++k) {
    double w[4], p[4];
    row.four(part * kPart + 4 * (k * kSumThreads + (int)threadIdx.x), w, p);
    sw += (w[0] + w[1]) + (w[2] + w[3]);
    sp += (p[0] + p[1]) + (p[2] + p[3]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    sw += __shfl_xor(sw, o, kWave);
    sp += __shfl_xor(sp, o, kWave);
  }
  if (lane == 0) wave_sum[threadIdx.x / kWave] = double2{sw, sp};
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < kSumThreads / kWave; ++w) {
    sw += wave_sum[w].x;
    sp += wave_sum[w].y;
  }
  a.sums[(int64_t)b * a.parts + part] = double2{sw, sp};
}

// The place of a draw among the block's values, one a thread.
struct Draw {
  double wave_sum[kDrawThreads / kWave];
  int first, last;
};

// Sums of the threads' values before each thread's own, and of all.
__device__ __forceinline__ double before(double x, double* total, Draw& sh) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  double inc = x;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const double y = __shfl_up(inc, o, kWave);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == kWave - 1) sh.wave_sum[wave] = inc;
  __syncthreads();
  double base = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kDrawThreads / kWave; ++w) {
    if (w == wave) base = all;
    all += sh.wave_sum[w];
  }
  *total = all;
  const double exc = __shfl_up(inc, 1, kWave);
  return base + (lane == 0 ? 0.0 : exc);
}

// The lowest `at` that a thread offers (>= 0), else the highest `alt`, else -1.
__device__ __forceinline__ int choose(int at, int alt, Draw& sh) {
  if (threadIdx.x == 0) {
    sh.first = 0x7fffffff;
    sh.last = -1;
  }
  __syncthreads();
  if (at >= 0) atomicMin(&sh.first, at);
  if (alt >= 0) atomicMax(&sh.last, alt);
  __syncthreads();
  return sh.first != 0x7fffffff ? sh.first : sh.last;
}

template <int DT>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ Draw sh;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = a.accepted[b];
  bool rejected = n < drafted(a, b);
  const double2 mine = tid < a.parts ? a.sums[(int64_t)b * a.parts + tid] : double2{0.0, 0.0};
  double part_sum = rejected ? mine.x : mine.y, total;
  double lo = before(part_sum, &total, sh);
  if (rejected && total == 0.0) {
    // nothing is left of p beside q: the draw is from p
    rejected = false;
    part_sum = mine.y;
    lo = before(part_sum, &total, sh);
  }
  const double goal = (double)a.u[(int64_t)b * (a.N + 1) + a.N] * total;
  const int part = choose(lo + part_sum > goal ? tid : -1, part_sum > 0.0 ? tid : -1, sh);
  int token = -1;
  if (part >= 0) {
    __syncthreads();
    if (tid == part) sh.wave_sum[0] = lo;
    __syncthreads();
    const double base = sh.wave_sum[0];
    const Weights<DT> row(a, b, n, rejected);
    const int i = part * kPart + kPerDraw * tid;
    double w[4], p[4], all;
    row.four(i, w, p);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = rejected ? w[e] : p[e];
      sum += w[e];
    }
    double at = base + before(sum, &all, sh);
    int first = -1, last = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      at += w[e];
      if (w[e] > 0.0) {
        last = i + e;
        if (first < 0 && at > goal) first = i + e;
      }
    }
    token = choose(first, last, sh);
  }
  for (int i = tid; i <= a.N; i += kDrawThreads)
    a.out[(int64_t)b * (a.N + 1) + i] =
        i < n ? a.tokens[(int64_t)b * a.N + i] : i == n ? (int64_t)token : -1;
}
static_assert(kPerDraw == 4, "a thread draws among four tokens");

inline int64_t verify_parts(int64_t V) { return (V + kPart - 1) / kPart; }

template <int DT>
void launch_verify(const VerifyArgs& a, int64_t B, hipStream_t st) {
  hipLaunchKernelGGL(verify_sum_kernel<DT>, dim3((unsigned)a.parts, (unsigned)B),
                     dim3(kSumThreads), 0, st, a);
  hipLaunchKernelGGL(verify_draw_kernel<DT>, dim3((unsigned)B), dim3(kDrawThreads), 0, st, a);
}

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" size_t rp_verify_drafts_workspace_bytes(int64_t B, int64_t V) {
  // sizes that the call refuses need none
  if (B <= 0 || B > 65535 || V <= 0 || V > kMaxV) return 0;
  return (size_t)(B * verify_parts(V) * 16);
}

extern "C" int rp_verify_drafts(const int64_t* tokens, const int32_t* lens, int64_t B, int64_t N,
                                const void* target, int64_t tsb, int64_t tsn, const void* draft,
                                int64_t dsb, int64_t dsn, int dtype, int64_t V, const float* u,
                                int64_t* out, int32_t* accepted, void* workspace,
                                size_t workspace_bytes, void* stream) {
  if ((!tokens && N != 0) || !target || !u || !out || !accepted) {
    rp_set_error("verify_drafts: null pointer");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (dtype != RP_OUT_BF16 && dtype != RP_OUT_F16 && dtype != RP_OUT_F32) {
    rp_set_error("verify_drafts: unknown dtype %d", dtype);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B <= 0 || N < 0 || V <= 0 || tsb < 0 || tsn < 0 || dsb < 0 || dsn < 0) {
    rp_set_error("verify_drafts: bad sizes or strides B=%lld N=%lld V=%lld", (long long)B,
                 (long long)N, (long long)V);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B > 65535 || N > 65535 || V > kMaxV) {
    rp_set_error("verify_drafts: too many sequences, drafts or tokens");
    return RP_ERR_UNSUPPORTED;
  }
  const int eb = dtype == RP_OUT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(target) % eb != 0 || reinterpret_cast<uintptr_t>(draft) % eb != 0) {
    rp_set_error("verify_drafts: probabilities must be aligned to their type");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const int64_t parts = verify_parts(V);
  if (!workspace || workspace_bytes < (size_t)(B * parts * 16) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255) != 0) {
    rp_set_error("verify_drafts: workspace of %zu bytes, 256-byte aligned, needed",
                 (size_t)(B * parts * 16));
    return RP_ERR_WORKSPACE;
  }
  const VerifyArgs a{static_cast<const char*>(target), static_cast<const char*>(draft), tsb, tsn,
                     dsb, dsn, tokens, u, lens, (int32_t)N, (int32_t)V, (int32_t)parts, out,
                     accepted, static_cast<double2*>(workspace)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == RP_OUT_F32) launch_verify<RP_OUT_F32>(a, B, st);
  else if (dtype == RP_OUT_F16) launch_verify<RP_OUT_F16>(a, B, st);
  else launch_verify<RP_OUT_BF16>(a, B, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    rp_set_error("verify_drafts: launch failed: %s", hipGetErrorString(e));
    return RP_ERR_LAUNCH;
  }
  return RP_OK;
}
