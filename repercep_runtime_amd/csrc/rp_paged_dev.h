// The paged key-value cache as the kernels see it, its row lookup and the
// host checks that its entry points share.  But for PagedView itself,
// everything here has internal linkage.
#pragma once

#include "rp_common.h"

namespace rp {

struct PagedView {
  char* k;
  char* v;
  float* ks;                       // null for 16-bit caches
  float* vs;
  const int32_t* table;
  int64_t table_stride;
  int64_t sp, sh, sr;              // element strides of page, head, row
  int32_t num_pages, heads, max_pages, shift;   // page_size = 1 << shift

  __host__ __device__ int64_t capacity() const { return (int64_t)max_pages << shift; }
  __host__ __device__ int32_t page_mask() const { return (1 << shift) - 1; }
};

namespace {

// The page that holds position `pos` of the sequence whose table entries
// begin at `row`; -1 where there is none: the position is past the table, or
// its entry is no page.
__host__ __device__ __forceinline__ int32_t paged_page(const PagedView& c, const int32_t* row,
                                                       int64_t pos) {
  const int64_t i = pos >> c.shift;
  if (pos < 0 || i >= c.max_pages) return -1;
  const int32_t p = row[i];
  return p >= 0 && p < c.num_pages ? p : -1;
}

// Element offset of a row, and its index in the scale arrays.
__host__ __device__ __forceinline__ int64_t paged_row(const PagedView& c, int32_t page,
                                                      int64_t head, int64_t pos) {
  return page * c.sp + head * c.sh + (pos & (((int64_t)1 << c.shift) - 1)) * c.sr;
}
__host__ __device__ __forceinline__ int64_t paged_scale(const PagedView& c, int32_t page,
                                                        int64_t head, int64_t pos) {
  return ((page * (int64_t)c.heads + head) << c.shift) + (pos & (((int64_t)1 << c.shift) - 1));
}

// A sequence's length as the kernels use it.
__device__ __forceinline__ int64_t paged_len(const PagedView& c, int32_t n) {
  return n < 0 ? 0 : min((int64_t)n, c.capacity());
}

inline int cache_elem_bytes(int64_t dtype) { return dtype == RP_CACHE_E4M3 ? 1 : 2; }

// Checks a descriptor and fills `v`; RP_OK or the error to return.
inline int paged_view(const char* what, const rp_paged_cache* c, PagedView* v) {
  if (!c || !c->k || !c->v || !c->block_table) {
    rp_set_error("%s: null pointer", what);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (c->dtype != RP_CACHE_BF16 && c->dtype != RP_CACHE_F16 && c->dtype != RP_CACHE_E4M3) {
    rp_set_error("%s: unknown cache dtype %lld", what, (long long)c->dtype);
    return RP_ERR_INVALID_ARGUMENT;
  }
  const bool fp8 = c->dtype == RP_CACHE_E4M3;
  if (fp8 != (c->k_scale != nullptr) || fp8 != (c->v_scale != nullptr)) {
    rp_set_error("%s: an e4m3 cache needs k_scale and v_scale, a 16-bit one takes none", what);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (c->num_pages <= 0 || c->heads <= 0 || c->page_size <= 0 || c->max_pages <= 0 ||
      c->table_stride < 0) {
    rp_set_error("%s: non-positive cache size", what);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
    rp_set_error("%s: head dim %lld not in {32, 64, 128, 256}", what, (long long)c->head_dim);
    return RP_ERR_UNSUPPORTED;
  }
  if ((c->page_size & (c->page_size - 1)) != 0 || c->page_size > 65536) {
    rp_set_error("%s: page size %lld is not a power of two up to 65536", what,
                 (long long)c->page_size);
    return RP_ERR_UNSUPPORTED;
  }
  if (c->num_pages > 0x7fffffff || c->max_pages > (1 << 30) / c->page_size ||
      c->heads > 65535) {
    rp_set_error("%s: too many pages, positions or heads", what);
    return RP_ERR_UNSUPPORTED;
  }
  const int64_t eb = cache_elem_bytes(c->dtype);
  if (c->stride_page < 0 || c->stride_head < 0 || c->stride_row < c->head_dim) {
    rp_set_error("%s: bad cache strides", what);
    return RP_ERR_INVALID_ARGUMENT;
  }
  if ((c->stride_page * eb | c->stride_head * eb | c->stride_row * eb) % 16 != 0 ||
      ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) != 0) {
    rp_set_error("%s: cache rows must be 16-byte aligned", what);
    return RP_ERR_UNSUPPORTED;
  }
  v->k = static_cast<char*>(c->k);
  v->v = static_cast<char*>(c->v);
  v->ks = c->k_scale;
  v->vs = c->v_scale;
  v->table = c->block_table;
  v->table_stride = c->table_stride;
  v->sp = c->stride_page;
  v->sh = c->stride_head;
  v->sr = c->stride_row;
  v->num_pages = (int32_t)c->num_pages;
  v->heads = (int32_t)c->heads;
  v->max_pages = (int32_t)c->max_pages;
  v->shift = __builtin_ctzll((unsigned long long)c->page_size);
  return RP_OK;
}

// Refuses a cache of which two rows share memory, K's and V's among them, for
// the calls that write it.
inline int paged_writable(const char* what, const rp_paged_cache* c) {
  const int64_t eb = cache_elem_bytes(c->dtype);
  const uintptr_t k = reinterpret_cast<uintptr_t>(c->k), v = reinterpret_cast<uintptr_t>(c->v);
  if (!rows_apart(c->head_dim * eb, {{c->num_pages, c->stride_page * eb},
                                     {c->heads, c->stride_head * eb},
                                     {c->page_size, c->stride_row * eb},
                                     {2, (int64_t)(k < v ? v - k : k - v)}})) {
    rp_set_error("%s: cache rows overlap", what);
    return RP_ERR_INVALID_ARGUMENT;
  }
  return RP_OK;
}

inline int paged_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    rp_set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return RP_ERR_LAUNCH;
  }
  return RP_OK;
}

}  // namespace
}  // namespace rp
