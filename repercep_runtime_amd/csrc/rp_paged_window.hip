// Attention of each sequence's last tokens over a paged key-value cache: which
// kernel takes a call, how its keys are split, the join of the parts, and the
// entry point.

#include <algorithm>

#include "rp_paged_window.h"

namespace rp {
namespace {

// Joins the parts of 256 / (64 W) rows, W waves a row: each part's mean counts
// by its sum about the largest base.  Half a wave or more takes a part's columns.
template <int QT, int D, int W>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a, int64_t rows) {
  constexpr int COLS = D / 4, GR = W * kWave / COLS;     // lanes a part, parts at a time
  __shared__ f32x4 sums[256];
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + threadIdx.x / (W * kWave);
  const int tid = threadIdx.x % (W * kWave), lane = threadIdx.x & (kWave - 1);
  const int col = tid % COLS, gr = tid / COLS;
  const bool in = row < rows;
  const int64_t bh = in ? row / a.S : 0;
  const int i = in ? (int)(row % a.S) : 0;
  const float2* ml = a.ml + (in ? row : 0) * a.splits;
  float base = neg_inf(), sum = 0.0f;
  for (int s = lane; s < a.splits; s += kWave)
    if (ml[s].y != 0.0f) base = fmaxf(base, ml[s].x);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) base = fmaxf(base, __shfl_xor(base, o, kWave));
  const float b0 = base == neg_inf() ? 0.0f : base;
  for (int s = lane; s < a.splits; s += kWave)
    if (ml[s].y != 0.0f) sum += ml[s].y * __builtin_amdgcn_exp2f(ml[s].x - b0);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.part + (in ? row : 0) * a.splits * D) + col;
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = gr; s < a.splits; s += GR) {
    const float2 p = ml[s];
    if (p.y == 0.0f) continue;                           // a part without keys wrote nothing
    x += part[(int64_t)s * COLS] * (p.y * __builtin_amdgcn_exp2f(p.x - b0) * inv);
  }
  sums[threadIdx.x] = x;
  __syncthreads();
  if (gr != 0 || !in) return;
#pragma unroll
  for (int g = 1; g < GR; ++g) x += sums[threadIdx.x + g * COLS];
  const int64_t b = bh / a.H, h = bh % a.H;
  uint16_t* out = a.out + b * a.osb + h * a.osh + (int64_t)i * a.oss + 4 * col;
  if (sum == 0.0f) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  *reinterpret_cast<u32x2*>(out) = u32x2{pack_out<QT>(x[0], x[1]), pack_out<QT>(x[2], x[3])};
  if (col == 0 && a.lse)
    a.lse[row] = sum == 0.0f ? neg_inf() : (b0 + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <int QT>
void launch_join(const WindowArgs& a, int64_t D, int64_t rows, hipStream_t st) {
  auto go = [&](auto one, auto four) {
    if (a.splits <= 16)
      hipLaunchKernelGGL(one, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, rows);
    else
      hipLaunchKernelGGL(four, dim3((unsigned)rows), dim3(256), 0, st, a, rows);
  };
  if (D == 32) go(window_join_kernel<QT, 32, 1>, window_join_kernel<QT, 32, 4>);
  else if (D == 64) go(window_join_kernel<QT, 64, 1>, window_join_kernel<QT, 64, 4>);
  else if (D == 128) go(window_join_kernel<QT, 128, 1>, window_join_kernel<QT, 128, 4>);
  else go(window_join_kernel<QT, 256, 1>, window_join_kernel<QT, 256, 4>);
}

constexpr int64_t kMaxSplits = 256;
// see kStreamBytes of rp_paged_attn.hip
constexpr int64_t kStreamBytes = 256 << 20;
// few_kernel: rows of a kv head up to which a call is bound by its keys' bytes.
// 16 sequences of 8000 keys, 8 kv heads of 128: 64 rows 142 us (prompt_kernel
// takes 128 rows in 154), 128 rows 268 us; e4m3fn 64 rows 100 us.
constexpr int64_t kFewRows = 64;
// and its workgroups: two a CU, what its registers hold.  Of 16-bit keys one a CU
// takes nearly the card's rate (93 us against 90 with half as many), but ragged
// batches need the parts: 16 sequences of 640 to 8000 e4m3fn keys 72 us on 256
// workgroups, 48 on 512, 58 on 1024.
constexpr int64_t kFewGroups = 512;
constexpr int64_t kFewPartBytes = 128 << 10;

// prompt_kernel: workgroups that fill the card (its LDS and registers hold one a
// CU), and the keys that are worth a part of their own: 256 where all rows see
// nearly all of them, 512 where a prompt's tiles see from few to all.  64 tokens of
// 2000 keys, 8 kv heads, 60 us in parts of 1024, 33 of 512, 28 of 256, 30 of 128;
// prompts of 512 tokens 22 us unsplit, 32 in parts of 256; of 2048, 2 kv heads, 53,
// 43 and 54 us in parts of 1024, 512 and 256.
constexpr int64_t kPromptGroups = 256, kPromptPartKeys = 512, kAfterPartKeys = 256;

struct Layout : WindowLaunch {
  int64_t tiles, splits, room;
  size_t ml, total;                                     // byte offsets: parts first
};

// (std::min on the host: HIP's own takes int there.)
inline Layout window_layout(int64_t B, int64_t H, int64_t S, const rp_paged_cache* c,
                            int64_t window, int64_t sinks, int64_t max_seq_len) {
  const int64_t cap = c->max_pages * c->page_size, group = H / c->heads;
  const int64_t longest = max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
  const int64_t groups = B * c->heads, all = S * group;
  const int64_t key_bytes =
      2 * (c->head_dim * cache_elem_bytes(c->dtype) + (c->dtype == RP_CACHE_E4M3 ? 4 : 0));
  Layout l;
  l.columns = all > kFewRows ? 0 : all <= 16 || c->head_dim == 256 ? 1 : 2;
  // Tiles of 256 rows where they are many or their keys can be split, of 128
  // otherwise: prompts of 1024 tokens, 8 kv heads, 40 us in 128 workgroups, 36 in
  // 256 of half the rows; 512 tokens after 15488 keys 162 us in 64 x 4 workgroups,
  // 232 with half the rows.  (A head dim of 256 leaves no registers for eight waves.)
  const bool many = groups * ((all + 255) / 256) >= kPromptGroups;
  l.waves = c->head_dim < 256 && all > 128 && (many || longest >= 2048) ? 8 : 4;
  const int64_t rows = l.columns ? 16 * l.columns : 32 * l.waves;
  l.tiles = (all + rows - 1) / rows;
  // a tile's keys: its tokens', the window's before them, the sinks
  const int64_t tokens = std::min(S, rows / group + 2);
  int64_t keys = longest;
  const int64_t past = std::min(window, longest) + std::min(sinks, longest);
  if (window > 0 && past + tokens < keys) keys = past + tokens;
  const int64_t blocks = groups * l.tiles;
  l.room = 0;
  l.stream = false;
  if (l.columns) {
    // No more parts of a sequence than four times an even share.  Sequences within
    // a window are alike, so one workgroup a CU is enough: 256 groups of 1056 keys
    // 27 us unsplit, 32 in two parts.
    l.room = kFewGroups / (c->heads * l.tiles);
    l.splits = std::min({1 + l.room - B, 4 * ((l.room + B - 1) / B), keys * key_bytes / kFewPartBytes});
    if (keys < longest && blocks >= kFewGroups / 2) l.splits = 1;
    // a second row tile finds V in the caches
    l.stream = l.tiles == 1 && groups * keys * key_bytes > kStreamBytes;
  } else if (blocks >= kPromptGroups) {
    l.splits = 1;
  } else {
    // One workgroup a CU; two where tiles of a prompt see few keys and many: 4096
    // tokens on one kv head 113 us unsplit, 81 in four parts.
    l.splits = keys >= 4 * S
        ? std::min(kPromptGroups / blocks, keys / kAfterPartKeys)
        : std::min((2 * kPromptGroups + blocks - 1) / blocks, keys / kPromptPartKeys);
  }
  l.splits = std::max((int64_t)1, std::min(l.splits, kMaxSplits));
  const int64_t parts = l.splits > 1 ? B * H * S * l.splits : 0;
  l.ml = (size_t)(parts * c->head_dim * 4);
  l.total = l.ml + (size_t)(parts * 8);
  return l;
}

}  // namespace
}  // namespace rp

using namespace rp;

extern "C" size_t rp_paged_window_workspace_bytes(int64_t B, int64_t H, int64_t S,
                                                  const rp_paged_cache* cache, int64_t window,
                                                  int64_t sinks, int64_t max_seq_len) {
  // sizes that the call refuses need none
  if (!cache || B <= 0 || B > 65535 || H <= 0 || H > 65535 || S <= 0 || cache->heads <= 0 ||
      cache->heads > H || cache->page_size <= 0 || cache->max_pages <= 0 ||
      cache->max_pages > (1 << 30) / cache->page_size || cache->head_dim <= 0 ||
      cache->head_dim > 256 || max_seq_len < 0 || window < 0 || sinks < 0 ||
      S > 0x7fffffff / (H / cache->heads) || B * cache->heads > 0x7fffffff / S)
    return 0;
  return window_layout(B, H, S, cache, window, sinks, max_seq_len).total;
}

extern "C" int rp_paged_attn_window(const void* q, int q_dtype, int64_t B, int64_t H, int64_t S,
                                    int64_t qsb, int64_t qsh, int64_t qss,
                                    const rp_paged_cache* cache, const int32_t* seq_lens,
                                    const int32_t* q_lens, int64_t window, int64_t sinks,
                                    float sm_scale, void* out, int64_t osb, int64_t osh,
                                    int64_t oss, float* lse, int64_t max_seq_len, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (!q || !out || !seq_lens) {
    rp_set_error("paged_attn_window: null pointer");
    return RP_ERR_INVALID_ARGUMENT;
  }
  PagedView c;
  const int rc = paged_view("paged_attn_window", cache, &c);
  if (rc != RP_OK) return rc;
  if (q_dtype != RP_DTYPE_BF16 && q_dtype != RP_DTYPE_F16) {
    rp_set_error("paged_attn_window: unknown q dtype %d", q_dtype);
    return RP_ERR_INVALID_ARGUMENT;
  }
  const bool fp8 = cache->dtype == RP_CACHE_E4M3;
  if (!fp8 && (cache->dtype == RP_CACHE_F16) != (q_dtype == RP_DTYPE_F16)) {
    rp_set_error("paged_attn_window: a 16-bit cache has q's dtype");
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (B <= 0 || S <= 0 || H <= 0 || H % cache->heads != 0 || max_seq_len < 0 || window < 0 ||
      sinks < 0) {
    rp_set_error("paged_attn_window: needs B, S > 0, H a multiple of the cache's %lld heads and "
                 "window, sinks, max_seq_len >= 0 (B=%lld S=%lld H=%lld)", (long long)cache->heads,
                 (long long)B, (long long)S, (long long)H);
    return RP_ERR_INVALID_ARGUMENT;
  }
  const float c2 = sm_scale * kLog2e;              // scores in powers of two
  if (!(c2 - c2 == 0.0f)) {
    rp_set_error("paged_attn_window: sm_scale and sm_scale * log2(e) must be finite");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const int64_t group = H / cache->heads;
  if (B > 65535 || H > 65535 || cache->stride_row > (1 << 25) || S > 0x7fffffff / group - 512 ||
      B * cache->heads > 0x7fffffff / S) {
    rp_set_error("paged_attn_window: too many sequences, heads or tokens, or rows too far apart");
    return RP_ERR_UNSUPPORTED;
  }
  if (fp8 && c.shift >= 4 &&
      ((reinterpret_cast<uintptr_t>(c.ks) | reinterpret_cast<uintptr_t>(c.vs)) & 15) != 0) {
    rp_set_error("paged_attn_window: scales must be 16-byte aligned");
    return RP_ERR_UNSUPPORTED;
  }
  if (((qsb | qsh | qss) & 7) != 0 || ((osb | osh | oss) & 3) != 0 ||
      (reinterpret_cast<uintptr_t>(q) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 7) != 0) {
    rp_set_error("paged_attn_window: q rows must be 16-byte and out rows 8-byte aligned");
    return RP_ERR_UNSUPPORTED;
  }
  if (!rows_apart(cache->head_dim, {{B, osb}, {H, osh}, {S, oss}})) {
    rp_set_error("paged_attn_window: out rows overlap");
    return RP_ERR_INVALID_ARGUMENT;
  }
  const Layout l = window_layout(B, H, S, cache, window, sinks, max_seq_len);
  const int64_t groups = B * cache->heads;
  if (groups * l.tiles * l.splits * 8 * kWave > kMaxGridThreads ||
      (l.splits > 1 && B * H * S * 256 > kMaxGridThreads)) {
    rp_set_error("paged_attn_window: too many sequences, heads or tokens");
    return RP_ERR_UNSUPPORTED;
  }
  if (l.total > 0 && (!workspace || workspace_bytes < l.total ||
                      (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)) {
    rp_set_error("paged_attn_window: workspace of %zu bytes, 256-byte aligned, needed", l.total);
    return RP_ERR_WORKSPACE;
  }
  // A row of q is read by the workgroup that writes its row of out, or before any
  // is written, so out can take q's place.
  const int64_t D = cache->head_dim, eb = cache_elem_bytes(cache->dtype);
  const int64_t scales = fp8 ? 4 * cache->num_pages * cache->heads * cache->page_size : 0;
  const Dim pages{cache->num_pages, cache->stride_page * eb},
      heads{cache->heads, cache->stride_head * eb}, slots{cache->page_size, cache->stride_row * eb};
  const RowSet in[] = {{q, 2 * D, {{B, 2 * qsb}, {H, 2 * qsh}, {S, 2 * qss}}},
                       {cache->k, D * eb, {pages, heads, slots}},
                       {cache->v, D * eb, {pages, heads, slots}},
                       whole(cache->k_scale, scales),
                       whole(cache->v_scale, scales),
                       {cache->block_table, 4 * cache->max_pages, {{B, 4 * cache->table_stride}, {1, 0}, {1, 0}}},
                       whole(seq_lens, 4 * B),
                       whole(q_lens, 4 * B)};
  const RowSet to[] = {{out, 2 * D, {{B, 2 * osb}, {H, 2 * osh}, {S, 2 * oss}}},
                       whole(lse, 4 * B * H * S)};
  if (outputs_meet(to, in, 1)) {
    rp_set_error("paged_attn_window: an output shares memory with another array, or with q at "
                 "other strides");
    return RP_ERR_INVALID_ARGUMENT;
  }
  char* ws = static_cast<char*>(workspace);
  WindowArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.qsb = qsb;
  a.qsh = qsh;
  a.qss = qss;
  a.lens = seq_lens;
  a.qlens = q_lens;
  // not 0, beside which a masked score of -inf would be NaN: 2^-149 of a score
  // is less than 2^-21
  a.c = c2 == 0.0f ? 0x1p-149f : c2 < 0.0f ? -c2 : c2;
  a.flip = c2 < 0.0f ? 0x80008000u : 0u;
  // bf16 weights where sums overflow: of at most as many keys as the table has
  // places, 1 in all; fp16 ones: up to 2^15
  a.lift = cache->dtype == RP_CACHE_F16
      ? kSlack - 15.0f
      : kSlack + (float)(64 - __builtin_clzll((unsigned long long)c.capacity()));
  a.window = window == 0 || window > 0x7fffffff ? 0x7fffffff : (int32_t)window;
  a.sinks = (int32_t)std::min(sinks, (int64_t)0x7fffffff);
  a.out = static_cast<uint16_t*>(out);
  a.osb = osb;
  a.osh = osh;
  a.oss = oss;
  a.lse = lse;
  a.H = (int32_t)H;
  a.group = (int32_t)group;
  a.S = (int32_t)S;
  a.tiles = (int32_t)l.tiles;
  a.splits = (int32_t)l.splits;
  a.room = (int32_t)l.room;
  a.groups = groups;
  a.part = reinterpret_cast<float*>(ws);
  a.ml = reinterpret_cast<float2*>(ws + l.ml);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (q_dtype == RP_DTYPE_F16) {
    if (fp8) launch_window<kInF16, RP_CACHE_E4M3>(a, c, D, l, st);
    else launch_window<kInF16, RP_CACHE_F16>(a, c, D, l, st);
    if (l.splits > 1) launch_join<kInF16>(a, D, B * H * S, st);
  } else {
    if (fp8) launch_window<kInBf16, RP_CACHE_E4M3>(a, c, D, l, st);
    else launch_window<kInBf16, RP_CACHE_BF16>(a, c, D, l, st);
    if (l.splits > 1) launch_join<kInBf16>(a, D, B * H * S, st);
  }
  return paged_launched("paged_attn_window");
}
