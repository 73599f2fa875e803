// A paged key-value cache's writer and its eviction by attention weight.
//
// * append_kernel: new K and V rows to their pages, as they are or through
//   the row-wise e4m3fn quantizer (rp_rowwise_dev.h).  D / 8 lanes hold one
//   row, a 16-byte vector each, so a row is read once, its maximum found by a
//   butterfly and its codes written once.  Bound by HBM: 131 MB of rows into
//   69 MB of codes and scales in 48 us (4.2 TB/s).
// * evict_select_kernel: which rows of one (sequence, kv head) stay: the
//   budget-th largest weight by a radix select over order-preserving integer
//   keys, then one ordered pass that ranks the kept rows and writes their
//   positions and weights.
// * evict_move_kernel: the kept rows moved to the front, in place.

#include "rp_paged_dev.h"
#include "rp_rowwise_dev.h"

namespace rp {
namespace {

constexpr int kPThreads = 256;
// Rows a group of lanes takes where there are workgroups enough (4096 of one
// row a group, sixteen a CU): 16 ragged prompts of up to 4000 rows, 8 heads
// of 128 into e4m3fn pages, take 51 us with two, 55 with one and 53 with four;
// such calls read and write past the caches: 48 us (200 MB; 40 us at the rate
// of a large copy).
constexpr int kAppendUnroll = 2;
constexpr int64_t kManyRows = 4096;

struct AppendArgs {
  const uint16_t* k;
  const uint16_t* v;
  int64_t ksb, ksh, kss, vsb, vsh, vss;
  const int32_t* start;
  const int32_t* lengths;
  int32_t S;
};

template <bool STREAM, typename T>
__device__ __forceinline__ void put(T x, char* to) {
  if constexpr (STREAM) __builtin_nontemporal_store(x, reinterpret_cast<T*>(to));
  else *reinterpret_cast<T*>(to) = x;
}

template <bool STREAM>
__device__ __forceinline__ u32x4r get(const uint16_t* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4r*>(p));
  else return *reinterpret_cast<const u32x4r*>(p);
}

// One row of K or V from registers to its place.
template <int DT, bool FP8, int TPR, bool STREAM>
__device__ __forceinline__ void append_row(const u32x4r& x, char* cache, float* scale, int64_t row,
                                           int64_t srow, int t) {
  if constexpr (FP8) {
    uint32_t m = absmax8(x);
#pragma unroll
    for (int o = TPR / 2; o >= 1; o >>= 1) m = umax32(m, (uint32_t)__shfl_xor((int)m, o, kWave));
    float qm, dq;
    rowwise_scales<DT>(m, &qm, &dq);
    if (row >= 0) {
      const uint2 o = quant8<DT>(x, qm);
      put<STREAM>(u32x2r{o.x, o.y}, cache + row + 8 * t);
      if (t == 0) scale[srow] = dq;
    }
  } else if (row >= 0) {
    put<STREAM>(x, cache + 2 * row + 16 * t);
  }
}

// U rows of K and U of V per thread group, their loads all on the way before
// the first is used.
template <int DT, bool FP8, int TPR, int U>
__global__ __launch_bounds__(kPThreads) void append_kernel(AppendArgs a, PagedView c) {
  constexpr int RPB = kPThreads / TPR;
  const int b = blockIdx.y, t = threadIdx.x % TPR;
  const int n = a.lengths ? min(a.lengths[b], a.S) : a.S;
  const int32_t* table = c.table + b * c.table_stride;
  u32x4r x[U], y[U];
  int64_t row[U], srow[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const uint32_t r = (blockIdx.x * U + j) * RPB + threadIdx.x / TPR;
    // a head's rows are neighbours in a page
    const int h = (int)(r / (uint32_t)a.S), i = (int)(r % (uint32_t)a.S);
    const int64_t pos = (int64_t)a.start[b] + i;
    const int32_t page = h < c.heads && i < n ? paged_page(c, table, pos) : -1;
    x[j] = y[j] = u32x4r{0u, 0u, 0u, 0u};
    row[j] = srow[j] = -1;
    if (page >= 0) {
      x[j] = get<(U > 1)>(a.k + b * a.ksb + h * a.ksh + i * a.kss + 8 * t);
      y[j] = get<(U > 1)>(a.v + b * a.vsb + h * a.vsh + i * a.vss + 8 * t);
      row[j] = paged_row(c, page, h, pos);
      if constexpr (FP8) srow[j] = paged_scale(c, page, h, pos);
    }
  }
#pragma unroll
  for (int j = 0; j < U; ++j) {
    append_row<DT, FP8, TPR, (U > 1)>(x[j], c.k, c.ks, row[j], srow[j], t);
    append_row<DT, FP8, TPR, (U > 1)>(y[j], c.v, c.vs, row[j], srow[j], t);
  }
}

template <int DT, bool FP8>
void launch_append(const AppendArgs& a, const PagedView& c, int64_t B, int64_t D, hipStream_t st) {
  const int64_t rows = (int64_t)a.S * c.heads;
  auto go = [&](auto one, auto many, int64_t tpr) {
    const int64_t rpb = kPThreads / tpr;
    const bool u = rows * B >= kManyRows * rpb;
    const int64_t per = u ? kAppendUnroll * rpb : rpb;
    hipLaunchKernelGGL(u ? many : one, dim3((unsigned)((rows + per - 1) / per), (unsigned)B),
                       dim3(kPThreads), 0, st, a, c);
  };
  constexpr int U = kAppendUnroll;
  if (D == 32) go(append_kernel<DT, FP8, 4, 1>, append_kernel<DT, FP8, 4, U>, 4);
  else if (D == 64) go(append_kernel<DT, FP8, 8, 1>, append_kernel<DT, FP8, 8, U>, 8);
  else if (D == 128) go(append_kernel<DT, FP8, 16, 1>, append_kernel<DT, FP8, 16, U>, 16);
  else go(append_kernel<DT, FP8, 32, 1>, append_kernel<DT, FP8, 32, U>, 32);
}

// ------------------------------------------------------------------ eviction

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;

// fp32 -> an unsigned key in the same order; -0 as 0, NaN above everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w);
  if (w != w) return 0xffffffffu;
  if (w == 0.0f) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictArgs {
  const int32_t* lens;
  const float* weights;
  int64_t wsb, wsh;
  int32_t budget, recent;
  int32_t* new_lens;
  float* new_weights;
  int64_t W;
  int32_t* src;        // (B, heads, budget): the position each kept row comes from
  int32_t* first;      // (B, heads): ranks below it are their own positions
  bool aligned;        // every row of weights lies on a 16-byte border
};

struct SelectShared {
  uint32_t hist[kBins];
  uint32_t pick[2];                // the digit, the keys above it
  uint32_t wave_count[kSelThreads / kWave];
  uint64_t wave_rank[kSelThreads / kWave];
  int first;
};

// Bound by its chain of passes, a few dependent latencies each: 11.6 us at
// 1100 rows, 16.2 at 256 caches' heads of up to 8192 (256 threads instead of
// 1024 take 12.7 us at 1100).
//
// One workgroup per (sequence, kv head).  Each thread owns `per` consecutive
// positions, four at a time (KEEP > 0: at most KEEP, held in registers; 0: read
// again in each pass).  The border key is found eleven bits at a time: a histogram of the
// digit among the keys that share the digits found so far, and the bin in
// which the count from above passes `need`.  A scan of each thread's rows above
// and on the border then ranks the kept rows in one go.
template <int KEEP>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a, PagedView c) {
  __shared__ SelectShared sh;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t g = (int64_t)b * c.heads + h;
  const int n = (int)paged_len(c, a.lens[b]);
  const float* w = a.weights + b * a.wsb + h * a.wsh;
  float* out = a.new_weights + g * a.W;
  if (tid == 0 && h == 0) a.new_lens[b] = min(n, a.budget);
  if (n <= a.budget) {
    for (int64_t i = tid; i < a.W; i += kSelThreads) out[i] = i < n ? w[i] : 0.0f;
    if (tid == 0) a.first[g] = a.budget;
    return;
  }
  for (int64_t i = a.budget + tid; i < a.W; i += kSelThreads) out[i] = 0.0f;
  const int per = (int)(((int64_t)n + 4 * kSelThreads - 1) / (4 * kSelThreads) * 4);
  const int from = (int)min((int64_t)n, (int64_t)tid * per), to = min(n, from + per);
  auto load4 = [&](int i) -> f32x4 {                // positions i .. i + 3, those before `to`
    if (a.aligned && i + 4 <= to) return *reinterpret_cast<const f32x4*>(w + i);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < to ? w[i + e] : 0.0f;
    return v;
  };
  f32x4 x[KEEP > 0 ? KEEP / 4 : 1];
  if constexpr (KEEP > 0) {
#pragma unroll
    for (int q = 0; q < KEEP / 4; ++q) x[q] = load4(from + 4 * q);
  }
  // calls f(position, weight) for each of the thread's rows, in order
  auto each = [&](auto f) {
    auto four = [&](int i, f32x4 v) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < to) f(i + e, v[e]);
    };
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int q = 0; q < KEEP / 4; ++q) four(from + 4 * q, x[q]);
    } else {
      for (int i = from; i < to; i += 4) four(i, load4(i));
    }
  };

  const int old = n - a.recent;
  uint32_t need = (uint32_t)(a.budget - a.recent);   // of the first `old`; < old
  const bool choose = need > 0;
  uint32_t key = 0;
  if (choose) {
    constexpr int kLow[3] = {21, 10, 0}, kWidth[3] = {11, 11, 10};
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      const int low = kLow[d];
      const uint32_t bins = 1u << kWidth[d], digit = bins - 1;
      for (int i = tid; i < kBins; i += kSelThreads) sh.hist[i] = 0;
      __syncthreads();
      each([&](int i, float v) {
        const uint32_t u = weight_key(v);
        const bool same = d == 0 || u >> (low + kWidth[d]) == key >> (low + kWidth[d]);
        if (i < old && same) atomicAdd(&sh.hist[(u >> low) & digit], 1u);
      });
      __syncthreads();
      // thread t counts the BPT bins from BPT (kSelThreads - 1 - t) up, the last thread the lowest
      constexpr int BPT = kBins / kSelThreads;
      const int bin = BPT * (kSelThreads - 1 - tid);
      uint32_t cnt[BPT], own = 0;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        cnt[i] = sh.hist[bin + i];
        own += cnt[i];
      }
      uint32_t sum = own;
#pragma unroll
      for (int o = 1; o < kWave; o *= 2) {
        const uint32_t v = __shfl_up((int)sum, o, kWave);
        if (lane >= o) sum += v;
      }
      if (lane == kWave - 1) sh.wave_count[wave] = sum;
      __syncthreads();
      uint32_t above = sum - own;                    // keys in bins over this thread's
#pragma unroll
      for (int q = 0; q < kSelThreads / kWave; ++q)
        if (q < wave) above += sh.wave_count[q];
#pragma unroll
      for (int i = BPT - 1; i >= 0; --i) {
        if (above < need && need <= above + cnt[i]) {
          sh.pick[0] = (uint32_t)(bin + i);
          sh.pick[1] = above;
        }
        above += cnt[i];
      }
      __syncthreads();
      key |= sh.pick[0] << low;
      need -= sh.pick[1];
    }
  }
  // need: how many of the rows on the border stay
  auto over = [&](int i, uint32_t u) { return i >= old || (choose && u > key); };
  auto tie = [&](int i, uint32_t u) { return i < old && choose && u == key; };
  uint32_t overs = 0, ties = 0;
  each([&](int i, float v) {
    const uint32_t u = weight_key(v);
    overs += over(i, u);
    ties += tie(i, u);
  });
  const uint64_t own = (uint64_t)overs << 32 | ties;
  uint64_t sum = own;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const uint64_t v = __shfl_up((unsigned long long)sum, o, kWave);
    if (lane >= o) sum += v;
  }
  if (lane == kWave - 1) sh.wave_rank[wave] = sum;
  if (tid == 0) sh.first = a.budget;
  __syncthreads();
  sum -= own;
#pragma unroll
  for (int q = 0; q < kSelThreads / kWave; ++q)
    if (q < wave) sum += sh.wave_rank[q];
  uint32_t ro = (uint32_t)(sum >> 32), rt = (uint32_t)sum;
  int32_t* src = a.src + g * a.budget;
  int first = a.budget;
  each([&](int i, float v) {
    const uint32_t u = weight_key(v);
    const bool o = over(i, u), t = tie(i, u);
    if (o || (t && rt < need)) {
      const uint32_t rank = ro + min(rt, need);
      src[rank] = i;
      out[rank] = v;
    } else {
      first = min(first, i);
    }
    ro += o;
    rt += t;
  });
  if (first < a.budget) atomicMin(&sh.first, first);
  __syncthreads();
  if (tid == 0) a.first[g] = sh.first;
}

// Moves the kept rows of one (sequence, kv head) to their ranks, one slice of
// 16-byte columns of K or of V (or the row scales) per workgroup.  A row only
// moves down and ranks rise with positions, so tiles of rows in order need no
// second buffer: every row that a tile overwrites is one that this tile or an
// earlier one has read, or one that goes.  A tile's places are looked up while
// the one before it is on its way.  Bound by the order of a cache's tiles and by
// HBM taking single rows: 32 caches of 8 heads cut to 2048 e4m3fn rows of 128
// move 2 x 120 MB in 64 us (3.8 TB/s).
constexpr int kMoveThreads = 1024, kMoveUnroll = 4;

template <bool STREAM, typename T, typename Offset>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const PagedView& c,
                                          const int32_t* src, const int32_t* table, int h,
                                          int begin, int r, int step, T* base, Offset offset) {
  int64_t at[kMoveUnroll], to[kMoveUnroll];
  auto find = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int row = r0 + u * step + r;
      at[u] = to[u] = -1;
      if (row >= a.budget) continue;
      const int32_t from = src[row];
      const int32_t pf = paged_page(c, table, from), pt = paged_page(c, table, row);
      if (pf < 0 || pt < 0) continue;
      at[u] = offset(pf, from);
      to[u] = offset(pt, row);
    }
  };
  find(begin);
  for (int r0 = begin; r0 < a.budget; r0 += step * kMoveUnroll) {
    T x[kMoveUnroll];
    int64_t dst[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      dst[u] = to[u];
      x[u] = T{};
      if (at[u] >= 0) x[u] = *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + at[u]);
    }
    find(r0 + step * kMoveUnroll);
    // every load of the tile has to be back before any store of it
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) asm volatile("" : "+v"(x[u]));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u)
      if (dst[u] >= 0) put<STREAM>(x[u], reinterpret_cast<char*>(base) + dst[u]);
  }
}

// LINES: slices of whole 128-byte lines, written past the caches (32 caches of
// 8 heads cut to 2048 rows: 77 us a call against 82).
template <bool LINES>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a, PagedView c,
                                                                  int slices, int lanes) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t g = (int64_t)b * c.heads + h;
  const int begin = a.first[g];
  if (begin >= a.budget) return;
  const int32_t* src = a.src + g * a.budget;
  const int32_t* table = c.table + b * c.table_stride;
  const int kind = blockIdx.x / slices;     // 0: K, 1: V, 2: the scales
  if (kind == 2) {
    // K's in the first half of the threads, V's in the second
    float* s = threadIdx.x < kMoveThreads / 2 ? c.ks : c.vs;
    move_rows<false>(a, c, src, table, h, begin, threadIdx.x & (kMoveThreads / 2 - 1),
                     kMoveThreads / 2, s,
              [&](int32_t p, int64_t pos) { return paged_scale(c, p, h, pos) * 4; });
    return;
  }
  u32x4r* base = reinterpret_cast<u32x4r*>(kind == 0 ? c.k : c.v);
  const int eb = c.ks ? 1 : 2;
  const int col = ((blockIdx.x % slices) * lanes + threadIdx.x % lanes) * 16;
  move_rows<LINES>(a, c, src, table, h, begin, threadIdx.x / lanes, kMoveThreads / lanes, base,
            [&](int32_t p, int64_t pos) { return paged_row(c, p, h, pos) * eb + col; });
}

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" int64_t rp_selftest_paged_row(const rp_paged_cache* cache, int64_t head, int64_t pos) {
  PagedView c;
  if (paged_view("selftest_paged_row", cache, &c) != RP_OK || head < 0 || head >= c.heads)
    return -1;
  const int32_t page = paged_page(c, c.table, pos);
  return page < 0 ? -1 : paged_row(c, page, head, pos);
}

extern "C" int rp_paged_kv_append(const void* k, const void* v, int x_dtype, int64_t B, int64_t S,
                                  int64_t ksb, int64_t ksh, int64_t kss, int64_t vsb, int64_t vsh,
                                  int64_t vss, const rp_paged_cache* cache, const int32_t* start,
                                  const int32_t* lengths, void* stream) {
  if (!k || !v || !start) {
    rp_set_error("paged_kv_append: null pointer");
    return RP_ERR_INVALID_ARGUMENT;
  }
  PagedView c;
  int rc = paged_view("paged_kv_append", cache, &c);
  if (rc != RP_OK) return rc;
  if (x_dtype != RP_DTYPE_BF16 && x_dtype != RP_DTYPE_F16) {
    rp_set_error("paged_kv_append: unknown input dtype %d", x_dtype);
    return RP_ERR_INVALID_ARGUMENT;
  }
  const bool fp8 = cache->dtype == RP_CACHE_E4M3;
  if (!fp8 && (cache->dtype == RP_CACHE_F16) != (x_dtype == RP_DTYPE_F16)) {
    rp_set_error("paged_kv_append: a 16-bit cache takes rows of its own dtype");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B <= 0 || S <= 0) {
    rp_set_error("paged_kv_append: non-positive size B=%lld S=%lld", (long long)B, (long long)S);
    return RP_ERR_INVALID_ARGUMENT;
  }
  // head_dim / 8 threads take kAppendUnroll rows of so many
  if (B > 65535 || S > 0x7fffffff / cache->heads ||
      (S * cache->heads / kAppendUnroll + kPThreads) * (cache->head_dim / 8) > kMaxGridThreads) {
    rp_set_error("paged_kv_append: too many sequences or rows");
    return RP_ERR_UNSUPPORTED;
  }
  if (((ksb | ksh | kss | vsb | vsh | vss) & 7) != 0 ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0) {
    rp_set_error("paged_kv_append: new rows must be 16-byte aligned");
    return RP_ERR_UNSUPPORTED;
  }
  rc = paged_writable("paged_kv_append", cache);
  if (rc != RP_OK) return rc;
  const AppendArgs a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                     ksb, ksh, kss, vsb, vsh, vss, start, lengths, (int32_t)S};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t D = cache->head_dim;
  if (!fp8) launch_append<kInBf16, false>(a, c, B, D, st);
  else if (x_dtype == RP_DTYPE_F16) launch_append<kInF16, true>(a, c, B, D, st);
  else launch_append<kInBf16, true>(a, c, B, D, st);
  return paged_launched("paged_kv_append");
}

extern "C" size_t rp_paged_evict_workspace_bytes(int64_t B, const rp_paged_cache* cache,
                                                 int64_t budget) {
  // sizes that the call refuses need none; no more than the table's positions stay
  if (!cache || B <= 0 || B > 65535 || budget <= 0 || cache->heads <= 0 || cache->heads > 65535 ||
      cache->page_size <= 0 || cache->max_pages <= 0 ||
      cache->max_pages > (1 << 30) / cache->page_size)
    return 0;
  const int64_t cap = cache->max_pages * cache->page_size;
  budget = budget < cap ? budget : cap;
  return (size_t)((B * cache->heads * 4 + 255) / 256 * 256 + B * cache->heads * budget * 4);
}

extern "C" int rp_paged_kv_evict(const rp_paged_cache* cache, const int32_t* seq_lens, int64_t B,
                                 const float* weights, int64_t wsb, int64_t wsh, int64_t budget,
                                 int64_t recent, int32_t* new_lens, float* new_weights, int64_t W,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (!seq_lens || !weights || !new_lens || !new_weights) {
    rp_set_error("paged_kv_evict: null pointer");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (new_lens == seq_lens || new_weights == weights) {
    rp_set_error("paged_kv_evict: new_lens and new_weights are not the inputs");
    return RP_ERR_INVALID_ARGUMENT;
  }
  PagedView c;
  int rc = paged_view("paged_kv_evict", cache, &c);
  if (rc != RP_OK) return rc;
  if (B <= 0 || budget <= 0 || recent < 0 || recent > budget) {
    rp_set_error("paged_kv_evict: needs B > 0 and 0 <= recent <= budget, budget > 0 (B=%lld "
                 "budget=%lld recent=%lld)", (long long)B, (long long)budget, (long long)recent);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B > 65535) {
    rp_set_error("paged_kv_evict: too many sequences");
    return RP_ERR_UNSUPPORTED;
  }
  if (wsb < 0 || wsh < 0 || W < c.capacity()) {
    rp_set_error("paged_kv_evict: weights need a place for each of %lld positions (got %lld)",
                 (long long)c.capacity(), (long long)W);
    return RP_ERR_INVALID_ARGUMENT;
  }
  // a budget past the table's end cuts nothing: the workspace need not hold it
  budget = budget < c.capacity() ? budget : c.capacity();
  recent = recent < budget ? recent : budget;
  const size_t want = rp_paged_evict_workspace_bytes(B, cache, budget);
  if (!workspace || workspace_bytes < want || (reinterpret_cast<uintptr_t>(workspace) & 255)) {
    rp_set_error("paged_kv_evict: workspace of %zu bytes, 256-byte aligned, needed", want);
    return RP_ERR_WORKSPACE;
  }
  rc = paged_writable("paged_kv_evict", cache);
  if (rc != RP_OK) return rc;
  int32_t* first = static_cast<int32_t*>(workspace);
  int32_t* src = first + (B * c.heads * 4 + 255) / 256 * 64;
  const EvictArgs a{seq_lens, weights, wsb, wsh, (int32_t)budget, (int32_t)recent, new_lens,
                    new_weights, W, src, first,
                    ((wsb | wsh) & 3) == 0 && (reinterpret_cast<uintptr_t>(weights) & 15) == 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)c.heads, (unsigned)B);
  auto select = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kSelThreads), 0, st, a, c);
  };
  if (c.capacity() <= 8 * kSelThreads) select(evict_select_kernel<8>);
  else if (c.capacity() <= 32 * kSelThreads) select(evict_select_kernel<32>);
  else select(evict_select_kernel<0>);
  const int row_bytes = (int)cache->head_dim * cache_elem_bytes(cache->dtype);
  // slices of whole 128-byte lines where that leaves a workgroup for each CU
  // (32 caches x 8 heads of e4m3fn: 84 us, 98 us in half lines), else of 64
  // bytes (one cache of 8 heads: 16 us, 18 us in whole lines)
  const bool lines = row_bytes >= 128 && B * c.heads * 2 * (row_bytes / 128) >= 256;
  const int lanes = lines ? 8 : row_bytes >= 64 ? 4 : row_bytes / 16;
  const int slices = row_bytes / (16 * lanes);
  auto move = [&](auto kernel) {
    hipLaunchKernelGGL(kernel,
                       dim3((unsigned)(2 * slices + (c.ks ? 1 : 0)), (unsigned)c.heads, (unsigned)B),
                       dim3(kMoveThreads), 0, st, a, c, slices, lanes);
  };
  if (lines) move(evict_move_kernel<true>);
  else move(evict_move_kernel<false>);
  return paged_launched("paged_kv_evict");
}
