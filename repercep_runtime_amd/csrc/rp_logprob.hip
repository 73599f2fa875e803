// Token log probabilities, entropy and the best alternatives of rows of logits.
//
// The floor is one read of the logits, and 5 TB/s of 16-bit logits leave the
// VALU about 15 lane operations each, so a row is read once, into registers,
// and everything is computed from there:
//   M = max x,  t = x c - M c  (c = log2(e) / temperature),
//   s = n + r = sum 2^t (n: largest logits left out of r),  u = sum 2^t t,
//   log p(x) = ln 2 t - log(s),  entropy = log(s) - ln 2 u / s.
// t is one fma, so logits far from zero lose nothing; t below -200 (2^t = 0)
// is held there, so a masked logit adds 0 and not 0 * inf.
//
// The best `top` logits cost no pass of their own.  The threads' maxima,
// folded to 64 groups, give M and, as their top-th largest, a bound that at
// least `top` logits reach; the few that do are collected in LDS and ranked
// by counting, on keys of the logit and its token so that no two are equal.
// Should more reach it than the buffer holds (a row of equal logits, a sorted
// one), or a NaN or infinity upset the order, the best are taken one by one.
//
// A workgroup holds up to 64 logits a thread.  Longer rows are split over
// workgroups; logprob_join_kernel merges their sums and their best.
//
// Bound by the VALU beside HBM: 4096 rows of 128256 16-bit logits take 268 us
// with 20 alternatives (3.9 TB/s); 11 instructions a logit, of which the
// exponential counts four times.  Rows of 16-bit logits with no more than
// `top` above zero take their maxima twice: a fifth more time.

#include <type_traits>

#include "rp_common.h"

namespace rp {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxThreads = 512;
constexpr int kHits = 128;                     // vectors collected per workgroup
constexpr int kMaxParts = 64, kMaxV = kMaxParts * kMaxThreads * 64;
constexpr int kJoinRows = 4, kJoinThreads = kJoinRows * kWave;
constexpr double kLn2 = 0.693147180559945309417;

struct LogprobArgs {
  const char* x;
  int64_t ld;
  int32_t V, top, parts, chunk;
  float c;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  f32x4* sums;              // (N, parts): M, n, r, u of each part
  uint64_t* keys;           // (N, parts, top)
};

// fp32 -> an unsigned key in the same order; -0 as 0, NaN above everything.
__device__ __forceinline__ uint32_t logit_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (x == 0.0f) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);   // NaN's key is a NaN's bits
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;

__device__ __forceinline__ uint64_t full_key(float x, int32_t id) {
  return ((uint64_t)logit_key(x) << 32) | (0xffffffffu - (uint32_t)id);
}

template <int DT>
__device__ __forceinline__ float logit_at(const char* row, int64_t i) {
  if constexpr (DT == RP_OUT_F32) return reinterpret_cast<const float*>(row)[i];
  else return in_to_f32<DT == RP_OUT_F16 ? kInF16 : kInBf16>(reinterpret_cast<const uint16_t*>(row)[i]);
}

// Whether fp32(M c) is within 2^-4 of M c: then t is one fma about it, and the
// sums are moved to M c afterwards.  A low temperature or a row of lowest
// values takes (x - M) c.
__device__ __forceinline__ bool near(float m, float c) { return fabsf(m * c) < 0x1p20f; }

// What a row's sums say of it: its log probabilities and entropy.  s = n + r:
// n largest logits weigh 1 each, the rest r together, kept apart so that a
// row that is all but certain keeps its small entropy and log probability.
struct Row {
  double base;
  float n, r, u, c, lg;
  __device__ __forceinline__ Row(float m, float n_, float r_, float u_, float c_)
      : base((double)m * (double)c_), n(n_), r(r_), u(u_), c(c_), lg(log1pf(n_ - 1.0f + r_)) {}
  __device__ __forceinline__ bool none() const { return n == 0.0f && r == 0.0f; }
  __device__ __forceinline__ float logprob(float x) const {
    if (none()) return -__builtin_inff();
    // in 64 bits: a lowest value's log probability is finite
    return (float)(((double)x * (double)c - base) * kLn2 - (double)lg);
  }
  __device__ __forceinline__ float entropy() const {
    return none() ? 0.0f : lg - (float)kLn2 * u / (n + r);
  }
};

template <int DT>
__device__ __forceinline__ float token_logit(const LogprobArgs& a, const char* row, int64_t t) {
  return t >= 0 && t < a.V ? logit_at<DT>(row, t) : 0.0f;
}
__device__ __forceinline__ void write_row(const LogprobArgs& a, const Row& r, int64_t row,
                                          int64_t token, float x) {
  a.logprobs[row] = token < 0 ? 0.0f : token >= a.V ? __builtin_nanf("") : r.logprob(x);
  if (a.entropy) a.entropy[row] = r.entropy();
}
__device__ __forceinline__ void write_top(const LogprobArgs& a, const Row& r, int64_t row, int rank,
                                          uint64_t key) {
  a.top_ids[row * a.top + rank] = 0xffffffffu - (uint32_t)key;
  a.top_logprobs[row * a.top + rank] = r.logprob(key_logit((uint32_t)(key >> 32)));
}

// max that propagates NaN (v_maximum3_f32)
__device__ __forceinline__ float nmax(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

__device__ __forceinline__ uint32_t pk_max_i16(uint32_t a, uint32_t b) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(i16x2, a),
                                                                __builtin_bit_cast(i16x2, b)));
}
// The larger of two 16-bit logits as signed integers, as a float.
template <int DT>
__device__ __forceinline__ float half_max(uint32_t w) {
  const int lo = (int16_t)(w & 0xffffu), hi = (int)w >> 16;
  const uint32_t x = (uint32_t)(lo > hi ? lo : hi) & 0xffffu;
  return DT == RP_OUT_F16 ? f16_to_f32(x) : bf16_to_f32(x);
}
// 16-bit logits whose t may leave fp32's range (c up to 2^20): -2^100 and below, fp16's -inf
template <int DT>
constexpr uint32_t kLow16 = DT == RP_OUT_F16 ? 0xfc00u : 0xf180u;

// One part of one row.  T threads, NV 16-byte vectors each, and a logit more
// for what lies before the part's first 16-byte border and behind its last.
template <int DT, int T, int NV>
__global__ __launch_bounds__(T) void logprob_kernel(LogprobArgs a) {
  constexpr int EB = DT == RP_OUT_F32 ? 4 : 2, EPV = 16 / EB, WAVES = T / kWave;
  constexpr int GROUP = T / kWave;                  // threads per group: 64 groups
  constexpr bool PACKED = EB == 2;
  __shared__ float group_max[kWave];
  __shared__ float wave_sum[2][WAVES];
  __shared__ u32x4 hit[kHits];                      // vectors that reach the bound
  __shared__ int32_t hit_at[kHits];                 // their first logits
  __shared__ uint64_t found[kHits * EPV + 2 * EPV];
  __shared__ uint64_t wave_best[WAVES];
  __shared__ int hits, count, best_count;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const char* xr = a.x + row * a.ld * EB;
  const int c0 = part * a.chunk, c1 = min(a.V, c0 + a.chunk);
  const int skew = (int)((reinterpret_cast<uintptr_t>(xr + (int64_t)c0 * EB) & 15) / EB);
  const int a0 = min(c1, c0 + (skew ? EPV - skew : 0));     // the vectors' logits: [a0, a1)
  const int a1 = a0 + (c1 - a0) / EPV * EPV;
  if (tid == 0) hits = count = best_count = 0;

  const u32x4* src = reinterpret_cast<const u32x4*>(xr + (int64_t)a0 * EB);
  const int nvec = (a1 - a0) / EPV;
  constexpr uint32_t kFill = DT == RP_OUT_F32 ? 0xff800000u : DT == RP_OUT_F16 ? 0xfc00fc00u : 0xff80ff80u;
  u32x4 raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    raw[v] = u32x4{kFill, kFill, kFill, kFill};
    if (tid + v * T < nvec) raw[v] = __builtin_nontemporal_load(src + tid + v * T);
  }
  // threads 0 .. EPV-1: the part's head, EPV .. 2 EPV-1: its tail
  const int edge = tid < EPV ? c0 + tid : a1 + tid - EPV;
  const bool has_edge = tid < EPV ? edge < a0 : tid < 2 * EPV && edge < c1;
  const float extra = has_edge ? logit_at<DT>(xr, edge) : -__builtin_inff();
  const int64_t token = a.tokens[row];
  const float xt = tid == 0 && a.parts == 1 ? token_logit<DT>(a, xr, token) : 0.0f;

  auto value = [&](int v, int e) -> float {
    if constexpr (EB == 4) return __uint_as_float(raw[v][e]);
    else if constexpr (DT == RP_OUT_F16) return f16_to_f32(e & 1 ? raw[v][e / 2] >> 16 : raw[v][e / 2] & 0xffffu);
    else return __uint_as_float(e & 1 ? raw[v][e / 2] & 0xffff0000u : raw[v][e / 2] << 16);
  };
  // The logits are unpacked anew in each phase: kept unpacked they would take
  // the registers of another workgroup, whose loads hide this one's arithmetic.
  auto forget = [&](int v) { asm volatile("" : "+v"(raw[v])); };
  auto phase = [&]() {
#pragma unroll
    for (int v = 0; v < NV; ++v) forget(v);
  };

  // Maxima of each vector and of the thread.  Of 16-bit logits, two at a time
  // as signed integers: right where any has a clear sign bit.  Of others (-0
  // among them) it is some logit, not above the true maximum, which is at most
  // 0; so a bound above 0 and what reaches it are right, and any other bound
  // sends the part through the exact maxima below.  As unsigned integers the
  // largest is the most negative logit (or a NaN of that sign).
  uint32_t vec16[NV], low16 = 0;
  float vec_max[NV], mine = -__builtin_inff();
  if constexpr (PACKED) {
    uint32_t top16 = kFill;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      vec16[v] = pk_max_i16(pk_max_i16(raw[v][0], raw[v][1]), pk_max_i16(raw[v][2], raw[v][3]));
      top16 = v == 0 ? vec16[0] : pk_max_i16(top16, vec16[v]);
#pragma unroll
      for (int i = 0; i < 4; ++i) low16 = pk_max_u16(low16, raw[v][i]);
    }
    mine = half_max<DT>(top16);
    low16 = umax32(low16 & 0xffffu, low16 >> 16);
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      vec_max[v] = value(v, 0);
#pragma unroll
      for (int e = 1; e < EPV; ++e) vec_max[v] = nmax(vec_max[v], value(v, e));
      mine = nmax(mine, vec_max[v]);
    }
  }
  mine = nmax(mine, extra);
  float gm, m;
  auto exchange = [&]() {
    gm = mine;
#pragma unroll
    for (int o = 1; o < GROUP; o *= 2) gm = nmax(gm, __shfl_xor(gm, o, kWave));
    if (tid % GROUP == 0) group_max[tid / GROUP] = gm;
    __syncthreads();
    gm = group_max[lane];
    m = gm;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = nmax(m, __shfl_xor(m, o, kWave));
  };
  exchange();
  phase();
  // the bound: the top-th largest group maximum, its low bits dropped
  float bound = __builtin_inff();
  auto find_bound = [&]() {
    const uint32_t k = logit_key(gm);
    uint32_t b = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t cand = b | 1u << bit;
      if (__popcll(__ballot(k >= cand)) >= a.top) b = cand;
    }
    bound = key_logit(b < kKeyNegInf ? kKeyNegInf : b);
  };
  if (a.top > 0) find_bound();
  if constexpr (PACKED) {
    if (m < 0.0f || bound <= 0.0f) {                // the same in every thread
      __syncthreads();
      mine = extra;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        forget(v);
        // eight sign bits: the largest logit is the least unsigned integer
        const uint32_t lo = pk_min_u16(pk_min_u16(raw[v][0], raw[v][1]),
                                       pk_min_u16(raw[v][2], raw[v][3]));
        if ((vec16[v] & 0x80008000u) == 0x80008000u)
          vec16[v] = min(lo & 0xffffu, lo >> 16) * 0x10001u;
        mine = nmax(mine, half_max<DT>(vec16[v]));
        __builtin_amdgcn_sched_barrier(0);
      }
      exchange();
      if (a.top > 0) find_bound();
    }
    phase();
  }
  const float m0 = m == -__builtin_inff() ? 0.0f : m;
  if (mine >= bound) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if constexpr (PACKED) {
        if (half_max<DT>(vec16[v]) < bound) continue;
      } else {
        if (vec_max[v] < bound) continue;
      }
      if (tid + v * T >= nvec) continue;             // the fill reaches a bound of -inf
      const int at = atomicAdd(&hits, 1);
      if (at < kHits) {
        hit[at] = raw[v];
        hit_at[at] = a0 + (tid + v * T) * EPV;
      }
    }
    if (has_edge && extra >= bound) found[atomicAdd(&count, 1)] = full_key(extra, edge);
  }
  phase();

  float s = 0.0f, u = 0.0f;
  auto weigh = [&](auto power) {                      // power(x) gives t

#pragma unroll
    for (int v = 0; v < NV; ++v) {
      forget(v);                                      // or the branches' common unpacking moves up
      float s1 = 0.0f, u1 = 0.0f;                     // short sums, then theirs
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const float t = power(value(v, e));
        const float p = __builtin_amdgcn_exp2f(t);
        s1 += p;
        u1 = __builtin_fmaf(p, t, u1);
      }
      s += s1;
      u += u1;
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const float base = m0 * a.c;
  const bool fma = near(m0, a.c);
  const float shift = fma ? __builtin_fmaf(m0, a.c, -base) : 0.0f;     // exact
  auto exact = [&](float x) { return nmax((x - m0) * a.c, -200.0f); };
  if (!fma)
    weigh(exact);
  else if (!PACKED || a.c > 0x1p20f || __any(low16 >= kLow16<DT>))
    weigh([&](float x) { return nmax(__builtin_fmaf(x, a.c, -base), -200.0f); });
  else
    weigh([&](float x) { return __builtin_fmaf(x, a.c, -base); });
  if (wave == 0) {                                    // the edges are in its first 16 lanes
    const float t = nmax(fma ? __builtin_fmaf(extra, a.c, -base) : exact(extra), -200.0f);
    const float p = __builtin_amdgcn_exp2f(t);
    s += p;
    u = __builtin_fmaf(p, t, u);
  }
  auto total = [&]() {                                // of the workgroup, in every thread
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      s += __shfl_xor(s, o, kWave);
      u += __shfl_xor(u, o, kWave);
    }
    if (lane == 0) {
      wave_sum[0][wave] = s;
      wave_sum[1][wave] = u;
    }
    __syncthreads();
    s = u = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      s += wave_sum[0][w];
      u += wave_sum[1][w];
    }
  };
  total();
  const bool odd = s != s;                            // a NaN or +inf: no distribution
  // from powers about fp32(M c) to powers about M c
  const float f = __builtin_amdgcn_exp2f(-shift);
  u = f * __builtin_fmaf(-shift, s, u);
  float n_best = s == 0.0f ? 0.0f : 1.0f, r_sum = s == 0.0f ? 0.0f : f * s - 1.0f;
  if (!odd && s > 0.0f && r_sum < 0x1p-8f) {          // the same in every thread
    // All but certain: 1 + r keeps too little of r, so the others are summed
    // again without the logits that equal M.
    int equal = 0;
    s = u = 0.0f;
    // from memory: this path is rare, and registers kept for it would cost the
    // others
#pragma unroll 8
    for (int i = c0 + tid; i < c1; i += T) {
      const float x = logit_at<DT>(xr, i), t = exact(x);
      const float p = x == m0 ? 0.0f : __builtin_amdgcn_exp2f(t);
      equal += x == m0;
      s += p;
      u = __builtin_fmaf(p, t, u);
    }
    if (equal) atomicAdd(&best_count, equal);
    __syncthreads();                                  // the first sums have been read
    total();
    n_best = (float)best_count;
    r_sum = s;
  }
  // made where it is used: its logarithm is a few dozen instructions
  auto whole_row = [&]() { return Row(m0, n_best, odd ? __builtin_nanf("") : r_sum, u, a.c); };
  if (tid == 0) {
    if (a.parts == 1) write_row(a, whole_row(), row, token, xt);
    else a.sums[row * a.parts + part] = f32x4{m0, n_best, odd ? __builtin_nanf("") : r_sum, u};
  }
  if (a.top == 0) return;
  uint64_t* keys = a.keys + (row * a.parts + part) * a.top;
  if (!odd && hits <= kHits) {
    for (int i = tid; i < hits * EPV; i += T) {
      const int v = i / EPV, e = i % EPV;
      float x;
      if constexpr (EB == 4) x = reinterpret_cast<const float*>(hit)[i];
      else x = in_to_f32<DT == RP_OUT_F16 ? kInF16 : kInBf16>(reinterpret_cast<const uint16_t*>(hit)[i]);
      if (x >= bound) found[atomicAdd(&count, 1)] = full_key(x, hit_at[v] + e);
    }
    __syncthreads();
    const int n = count;
    for (int i = tid; i < n; i += T) {
      const uint64_t key = found[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += found[j] > key;
      if (rank < a.top) {
        if (a.parts == 1) write_top(a, whole_row(), row, rank, key);
        else keys[rank] = key;
      }
    }
    // a part shorter than `top` leaves the rest to the other parts
    if (a.parts > 1)
      for (int i = n + tid; i < a.top; i += T) keys[i] = 0;
    return;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (int i = c0 + tid; i < c1; i += T) {        // from memory: this path is rare
      const uint64_t key = full_key(logit_at<DT>(xr, i), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, o, kWave);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) wave_best[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) best = wave_best[w] > best ? wave_best[w] : best;
    last = best;
    if (tid == 0) {
      if (a.parts > 1) keys[k] = best;
      else if (best) write_top(a, whole_row(), row, k, best);
    }
  }
}

// Merges the parts of a row, a wave each.
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void logprob_join_kernel(LogprobArgs a, int64_t rows) {
  extern __shared__ uint64_t join_keys[];          // kJoinRows * parts * top
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t row = (int64_t)blockIdx.x * kJoinRows + wave;
  const int n = a.parts * a.top;
  uint64_t* keys = join_keys + wave * n;
  if (row < rows)
    for (int i = lane; i < n; i += kWave) keys[i] = a.keys[row * n + i];
  __syncthreads();
  if (row >= rows) return;
  const int64_t token = a.tokens[row];
  const float xt = lane == 0 ? token_logit<DT>(a, a.x + row * a.ld * (DT == RP_OUT_F32 ? 4 : 2), token) : 0.0f;
  // a part a lane; one of nothing but -inf has no maximum
  static_assert(kMaxParts <= kWave, "a row's parts fit a wave");
  const f32x4 p = lane < a.parts ? a.sums[row * a.parts + lane] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const float whole = p[1] + p[2];
  const bool some = whole != 0.0f;
  float m = some ? p[0] : -__builtin_inff();
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = nmax(m, __shfl_xor(m, o, kWave));
  float nb = 0.0f, s = 0.0f, u = 0.0f;
  if (some) {
    const float t = nmax((float)((double)p[0] * (double)a.c - (double)m * (double)a.c), -200.0f);
    const float f = __builtin_amdgcn_exp2f(t);
    nb = t == 0.0f ? p[1] : 0.0f;                    // the parts that hold the row's maximum
    s = t == 0.0f ? p[2] : whole * f;
    u = f * __builtin_fmaf(whole, t, p[3]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    nb += __shfl_xor(nb, o, kWave);
    s += __shfl_xor(s, o, kWave);
    u += __shfl_xor(u, o, kWave);
  }
  const Row r(m, nb, s, u, a.c);
  for (int i = lane; i < n; i += kWave) {
    const uint64_t key = keys[i];
    if (key == 0) continue;
    // a part's keys fall: how many of each are above this one, by bisection
    int rank = 0;
    for (int q = 0; q < a.parts && rank < a.top; ++q) {
      const uint64_t* part = keys + q * a.top;
      int above = 0;
#pragma unroll
      for (int step = RP_LOGPROB_MAX_TOP; step >= 1; step /= 2)
        if (above + step <= a.top && part[above + step - 1] > key) above += step;
      rank += above;
    }
    if (rank < a.top) write_top(a, r, row, rank, key);
  }
  if (lane == 0) write_row(a, r, row, token, xt);
}

// Threads, vectors a thread and logits a part, by the row's length: one part
// where 512 threads of 64 logits hold the row, fewer logits a thread for short
// rows.  Of 4096 rows of 128256 parts of 32064 on 512 threads were the fastest:
// parts of 16032 on 256 took 1% more, 1024 threads of 32 logits 8% more.
struct LogprobPlan {
  int threads, vectors, parts, chunk;
};

inline LogprobPlan logprob_plan(int64_t V, int dtype) {
  const int epv = dtype == RP_OUT_F32 ? 4 : 8, per = 64 / epv;
  LogprobPlan p;
  p.threads = V > 256 * 64 ? 512 : 256;
  p.vectors = V > 256 * 32 ? per : V > 256 * 8 ? per / 2 : per / 8;
  const int64_t most = (int64_t)p.threads * p.vectors * epv;
  p.parts = (int)((V + most - 1) / most);
  p.chunk = (int)(((V + p.parts - 1) / p.parts + epv - 1) / epv * epv);
  p.parts = (int)((V + p.chunk - 1) / p.chunk);
  return p;
}

inline size_t logprob_sums_bytes(int64_t N, int parts) {
  return (size_t)((N * parts * 16 + 255) / 256 * 256);
}

template <int DT>
void launch_logprob(const LogprobArgs& a, const LogprobPlan& p, int64_t N, hipStream_t st) {
  constexpr int P = DT == RP_OUT_F32 ? 16 : 8;       // vectors of 64 logits
  auto go = [&](auto t, auto nv) {
    hipLaunchKernelGGL((logprob_kernel<DT, decltype(t)::value, decltype(nv)::value>),
                       dim3((unsigned)(N * p.parts)), dim3(p.threads), 0, st, a);
  };
  using std::integral_constant;
  if (p.threads == 512) go(integral_constant<int, 512>{}, integral_constant<int, P>{});
  else if (p.vectors == P) go(integral_constant<int, 256>{}, integral_constant<int, P>{});
  else if (p.vectors == P / 2) go(integral_constant<int, 256>{}, integral_constant<int, P / 2>{});
  else go(integral_constant<int, 256>{}, integral_constant<int, P / 8>{});
  if (p.parts > 1)
    hipLaunchKernelGGL(logprob_join_kernel<DT>, dim3((unsigned)((N + kJoinRows - 1) / kJoinRows)),
                       dim3(kJoinThreads), (size_t)(kJoinRows * p.parts * a.top * 8), st, a, N);
}

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" size_t rp_token_logprobs_workspace_bytes(int64_t N, int64_t V, int logits_dtype,
                                                    int top) {
  // sizes that the call refuses need none
  if (N <= 0 || N > 0x7fffffff / kMaxParts || V <= 0 || V > kMaxV || top < 0 ||
      top > RP_LOGPROB_MAX_TOP)
    return 0;
  const LogprobPlan p = logprob_plan(V, logits_dtype);
  return p.parts == 1 ? 0 : logprob_sums_bytes(N, p.parts) + (size_t)(N * p.parts * top * 8);
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
  if (N <= 0 || V <= 0 || (ld < V && ld != 0)) {
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
  const float c = (float)(1.4426950408889634 / (double)temperature);
  if (!(c - c == 0.0f)) {
    rp_set_error("token_logprobs: temperature too small");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (V > kMaxV || N > 0x7fffffff / kMaxParts) {
    rp_set_error("token_logprobs: too many rows or logits");
    return RP_ERR_UNSUPPORTED;
  }
  const int eb = logits_dtype == RP_OUT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % eb != 0) {
    rp_set_error("token_logprobs: logits must be aligned to their type");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const LogprobPlan p = logprob_plan(V, logits_dtype);
  if (N * p.parts * p.threads > kMaxGridThreads) {
    rp_set_error("token_logprobs: too many rows");
    return RP_ERR_UNSUPPORTED;
  }
  const size_t sums = logprob_sums_bytes(N, p.parts);
  const size_t want = p.parts == 1 ? 0 : sums + (size_t)(N * p.parts * top * 8);
  if (want > 0 && (!workspace || workspace_bytes < want ||
                   (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)) {
    rp_set_error("token_logprobs: workspace of %zu bytes, 256-byte aligned, needed", want);
    return RP_ERR_WORKSPACE;
  }
  char* ws = static_cast<char*>(workspace);
  const LogprobArgs a{static_cast<const char*>(logits), ld, (int32_t)V, top, p.parts, p.chunk, c,
                      tokens, logprobs, entropy, top_logprobs, top_ids,
                      reinterpret_cast<f32x4*>(ws), reinterpret_cast<uint64_t*>(ws + (want ? sums : 0))};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (logits_dtype == RP_OUT_F32) launch_logprob<RP_OUT_F32>(a, p, N, st);
  else if (logits_dtype == RP_OUT_F16) launch_logprob<RP_OUT_F16>(a, p, N, st);
  else launch_logprob<RP_OUT_BF16>(a, p, N, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    rp_set_error("token_logprobs: launch failed: %s", hipGetErrorString(e));
    return RP_ERR_LAUNCH;
  }
  return RP_OK;
}
