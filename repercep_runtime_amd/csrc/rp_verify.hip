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
// Only row n of p, and of q if draft n was rejected, is read whole (a test takes
// one value of each of the other rows), so the floor is those rows' bytes; small calls are a chain of
// dependent loads.  A block reads tokens in chunks of four a thread and adds up
// each wave's of each chunk (a segment); every wave then finds the segment that
// the draw falls into from the segments' sums, and the one that holds it looks
// among its lanes.
//
// Rows of up to kOne tokens take one launch: verify_one_kernel, a block a
// sequence.  Longer ones are cut into parts of kPart tokens: verify_sum_kernel
// finds n anew in each block (less than a launch) and adds up its part,
// verify_draw_kernel finds the draw's part and reads it once more.
//
// One sequence's four drafts under 32000 tokens take 10 us (two launches and
// scans over the block 18), 256 sequences under 128256 42 us: 4.7 TB/s of p's rows
// and, for the half of them with a draft rejected, q's.

#include "rp_common.h"

namespace rp {
namespace {

constexpr int kOneWaves = 16, kOneChunks = 8, kOne = kOneWaves * kWave * 4 * kOneChunks;
constexpr int kSumThreads = 256, kPart = 4096, kDrawWaves = kSumThreads / kWave;
constexpr int kDrawChunks = kPart / (kSumThreads * 4);
constexpr int64_t kMaxV = 1024 * (int64_t)kPart;

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
  for (int k = 0; k < kDrawChunks; ++k) {
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

// Sums of the lanes' values up to and with each lane's own.
__device__ __forceinline__ double upto(double x, int lane) {
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const double y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
  return x;
}

// Where a draw falls among up to 128 sums, two a lane: the first entry with
// lo + sums up to it > goal, else (rounding, or a goal of all there is and more)
// the last positive one, else -1; and the sums before it.
struct Place {
  int at;
  double before;
};
__device__ __forceinline__ Place place(double x0, double x1, double up, double lo, double goal,
                                       int lane) {
  const double b0 = lo + (up - (x0 + x1)), b1 = b0 + x0;
  const uint64_t in0 = __ballot(b1 > goal && x0 > 0.0), in1 = __ballot(b1 + x1 > goal && x1 > 0.0);
  const uint64_t any0 = __ballot(x0 > 0.0), any1 = __ballot(x1 > 0.0);
  int at = -1;
  if (in0 | in1) {
    const int l = __builtin_ctzll(in0 | in1);
    at = 2 * l + (in0 >> l & 1 ? 0 : 1);
  } else if (any0 | any1) {
    const int l = 63 - __builtin_clzll(any0 | any1);
    at = 2 * l + (any1 >> l & 1 ? 1 : 0);
  }
  const int l = at < 0 ? 0 : at / 2;
  return Place{at, at & 1 ? __shfl(b1, l, kWave) : __shfl(b0, l, kWave)};
}

// Draws a token among the K chunks of a block of W waves that begin at `first`,
// weighed by `row`: with goal(sum of the block's weights) the sum that has to be
// passed.  The wave that holds the token calls found(token); where there is
// nothing to draw every wave calls none().
template <int DT, int W, int K, typename G, typename F, typename N>
__device__ __forceinline__ void draw(const Weights<DT>& row, bool rejected, int first, double lo,
                                     double* sums, G goal, F found, N none) {
  static_assert(W * K <= 2 * kWave, "two segments a lane");
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  double mine[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    double w[4], p[4];
    row.four(first + 4 * (k * W * kWave + tid), w, p);
    const double* x = rejected ? w : p;
    mine[k] = (x[0] + x[1]) + (x[2] + x[3]);
    double s = mine[k];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, kWave);
    if (lane == 0) sums[k * W + wave] = s;
  }
  __syncthreads();
  const double x0 = 2 * lane < W * K ? sums[2 * lane] : 0.0;
  const double x1 = 2 * lane + 1 < W * K ? sums[2 * lane + 1] : 0.0;
  const double up = upto(x0 + x1, lane), all = __shfl(up, kWave - 1, kWave);
  const double want = goal(all);
  const Place seg = place(x0, x1, up, lo, want, lane);
  if (seg.at < 0) return none();
  if (seg.at % W != wave) return;
  // the segment's lanes, four tokens each, once more
  const int k = seg.at / W, i = first + 4 * (k * W * kWave + tid);
  double w[4], p[4];
  row.four(i, w, p);
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < K; ++c) sum = c == k ? mine[c] : sum;
  double at = seg.before + (upto(sum, lane) - sum);
  int in = -1, last = -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double x = rejected ? w[e] : p[e];
    at += x;
    if (x > 0.0) {
      last = i + e;
      if (in < 0 && at > want) in = i + e;
    }
  }
  const uint64_t past = __ballot(in >= 0), some = __ballot(last >= 0);
  const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  const int token = past ? __shfl(in, l, kWave) : __shfl(last, l, kWave);
  if (lane == 0) found(token);
}

// The accepted drafts and the padding behind the drawn token.
__device__ __forceinline__ void write_others(const VerifyArgs& a, int b, int n) {
  for (int i = threadIdx.x; i <= a.N; i += blockDim.x)
    if (i != n) a.out[(int64_t)b * (a.N + 1) + i] = i < n ? a.tokens[(int64_t)b * a.N + i] : -1;
}

template <int DT>
__global__ __launch_bounds__(kOneWaves* kWave) void verify_one_kernel(VerifyArgs a) {
  __shared__ double sums[2][kOneWaves * kOneChunks];
  const int b = blockIdx.x, lane = threadIdx.x & (kWave - 1);
  const int has = drafted(a, b);
  const int n = __builtin_amdgcn_readfirstlane(count_accepted<DT>(a, b, has, lane));
  if (threadIdx.x == 0) a.accepted[b] = n;
  write_others(a, b, n);
  const double u = a.u[(int64_t)b * (a.N + 1) + a.N];
  int64_t* to = a.out + (int64_t)b * (a.N + 1) + n;
  bool again = false;
  auto goal = [&](double all) { return u * all; };
  auto found = [&](int token) { *to = token; };
  const bool rejected = n < has;
  const Weights<DT> row(a, b, n, rejected);
  draw<DT, kOneWaves, kOneChunks>(row, rejected, 0, 0.0, sums[0], goal, found, [&] { again = true; });
  if (!again) return;                                    // the same in every wave
  // nothing is left of p beside q: the draw is from p
  draw<DT, kOneWaves, kOneChunks>(row, false, 0, 0.0, sums[1], goal, found, [&] {
    if (threadIdx.x == 0) *to = -1;
  });
}

template <int DT>
__global__ __launch_bounds__(kSumThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double sums[kDrawWaves * kDrawChunks];
  const int b = blockIdx.x, lane = threadIdx.x & (kWave - 1);
  const int n = a.accepted[b];
  const double u = a.u[(int64_t)b * (a.N + 1) + a.N];
  const double2* parts = a.sums + (int64_t)b * a.parts;
  bool rejected = n < drafted(a, b);
  write_others(a, b, n);
  // every wave adds up the parts, 128 at a time, and looks for the draw's
  double all = 0.0;
  for (;;) {
    for (int i = 0; i < a.parts; i += kWave)
      all += i + lane < a.parts ? (rejected ? parts[i + lane].x : parts[i + lane].y) : 0.0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) all += __shfl_xor(all, o, kWave);
    if (all != 0.0 || !rejected) break;
    rejected = false;                                    // nothing is left of p beside q
  }
  const double goal = u * all;
  Place part{-1, 0.0};
  double lo = 0.0;
  for (int i = 0; i < a.parts; i += 2 * kWave) {
    const int j = i + 2 * lane;
    const double2 none = {0.0, 0.0};
    const double2 y0 = j < a.parts ? parts[j] : none, y1 = j + 1 < a.parts ? parts[j + 1] : none;
    const double x0 = rejected ? y0.x : y0.y, x1 = rejected ? y1.x : y1.y;
    const double up = upto(x0 + x1, lane), sum = __shfl(up, kWave - 1, kWave);
    const Place p = place(x0, x1, up, lo, goal, lane);
    if (p.at >= 0) part = Place{i + p.at, p.before};
    lo += sum;
    if (lo > goal) break;
  }
  int64_t* to = a.out + (int64_t)b * (a.N + 1) + n;
  const Weights<DT> row(a, b, n, rejected);
  auto found = [&](int token) { *to = token; };
  auto none = [&] {
    if (threadIdx.x == 0) *to = -1;
  };
  if (part.at < 0) return none();
  draw<DT, kDrawWaves, kDrawChunks>(row, rejected, part.at * kPart, part.before, sums,
                                    [&](double) { return goal; }, found, none);
}

// 0: one launch.
inline int64_t verify_parts(int64_t V) { return V <= kOne ? 0 : (V + kPart - 1) / kPart; }

template <int DT>
void launch_verify(const VerifyArgs& a, int64_t B, hipStream_t st) {
  if (a.parts == 0) {
    hipLaunchKernelGGL(verify_one_kernel<DT>, dim3((unsigned)B), dim3(kOneWaves * kWave), 0, st, a);
    return;
  }
  hipLaunchKernelGGL(verify_sum_kernel<DT>, dim3((unsigned)a.parts, (unsigned)B),
                     dim3(kSumThreads), 0, st, a);
  hipLaunchKernelGGL(verify_draw_kernel<DT>, dim3((unsigned)B), dim3(kSumThreads), 0, st, a);
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
  const int64_t eb = dtype == RP_OUT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(target) % eb != 0 || reinterpret_cast<uintptr_t>(draft) % eb != 0) {
    rp_set_error("verify_drafts: probabilities must be aligned to their type");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const int64_t parts = verify_parts(V);
  if (parts > 0 && (!workspace || workspace_bytes < (size_t)(B * parts * 16) ||
                    (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)) {
    rp_set_error("verify_drafts: workspace of %zu bytes, 256-byte aligned, needed",
                 (size_t)(B * parts * 16));
    return RP_ERR_WORKSPACE;
  }
  // a block's waves write out while others still read the drafts
  const RowSet in[] = {whole(tokens, 8 * B * N),
                       whole(lens, 4 * B),
                       whole(u, 4 * B * (N + 1)),
                       {target, eb * V, {{B, eb * tsb}, {N + 1, eb * tsn}, {1, 0}}},
                       {draft, eb * V, {{B, eb * dsb}, {N, eb * dsn}, {1, 0}}}};
  const RowSet to[] = {whole(out, 8 * B * (N + 1)), whole(accepted, 4 * B)};
  if (outputs_meet(to, in, 0)) {
    rp_set_error("verify_drafts: an output shares memory with another array");
    return RP_ERR_INVALID_ARGUMENT;
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
