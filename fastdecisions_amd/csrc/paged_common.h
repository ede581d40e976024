// What the kernels of the paged cache share: the host's checks of an
// fd_paged_cache and the device's way from (request, key) to memory.
#pragma once

#include "../../include/fd_cache.h"
#include "fd_common.h"

namespace {

// A cache as the kernels see it: K and V (and their scales) lie at the same offsets of two pools.
struct PagedView {
  unsigned char* k;
  unsigned char* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t page, head, row;      // strides in bytes
  int64_t s_page, s_head;
  const int32_t* table;
  const int32_t* lens;
  int64_t table_stride;
  int n_pages, max_pages, shift;  // page_size == 1 << shift
};

inline int fill_view(const char* what, const fd_paged_cache* c, bool needs_lens, PagedView* out) {
  FD_REQUIRE(c != nullptr, FD_ERR_INVALID_ARGUMENT, "%s: the cache must be non-null", what);
  FD_REQUIRE(c->k && c->v && c->page_table && (c->cache_lens || !needs_lens), FD_ERR_INVALID_ARGUMENT,
             "%s: the cache's tensors, page table and lengths must be non-null", what);
  FD_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, FD_ERR_UNSUPPORTED,
             "%s: head_dim must be 64, 128 or 256 (got %d)", what, c->head_dim);
  FD_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
             FD_ERR_UNSUPPORTED, "%s: page_size must be a power of two in [16, 256] (got %d)", what, c->page_size);
  FD_REQUIRE(c->dtype == FD_DTYPE_BF16 || c->dtype == FD_DTYPE_E4M3, FD_ERR_INVALID_ARGUMENT,
             "%s: the cache's dtype must be FD_DTYPE_BF16 or FD_DTYPE_E4M3", what);
  FD_REQUIRE(c->n_pages >= 1 && c->max_pages >= 1 && c->kv_heads >= 1, FD_ERR_INVALID_ARGUMENT,
             "%s: n_pages, max_pages and kv_heads must be >= 1", what);
  FD_REQUIRE(static_cast<int64_t>(c->max_pages) * c->page_size < (1LL << 27), FD_ERR_UNSUPPORTED,
             "%s: a request holds fewer than 2^27 keys", what);
  const bool fp8 = c->dtype == FD_DTYPE_E4M3;
  FD_REQUIRE(!fp8 || (c->k_scale && c->v_scale), FD_ERR_INVALID_ARGUMENT, "%s: an E4M3 cache needs its scales", what);
  const int64_t elem = fp8 ? 1 : 2;
  const int64_t* st = c->k_strides;
  const int64_t* ss = c->k_scale_strides;
  FD_REQUIRE(st[0] == c->v_strides[0] && st[1] == c->v_strides[1] && st[2] == c->v_strides[2] &&
                 (!fp8 || (ss[0] == c->v_scale_strides[0] && ss[1] == c->v_scale_strides[1])),
             FD_ERR_UNSUPPORTED, "%s: the strides of K and V must be the same", what);
  FD_REQUIRE(st[0] * elem % 16 == 0 && st[1] * elem % 16 == 0 && st[2] * elem % 16 == 0, FD_ERR_ALIGNMENT,
             "%s: the cache's rows must be 16-byte aligned", what);
  FD_REQUIRE(st[2] >= 0 && st[2] < (1 << 20) && st[0] >= 0 && st[0] < (1LL << 35), FD_ERR_UNSUPPORTED,
             "%s: cache row strides must be in [0, 2^20), page strides in [0, 2^35)", what);
  FD_REQUIRE(!fp8 || (ss[0] >= 0 && ss[0] < (1LL << 31)), FD_ERR_UNSUPPORTED,
             "%s: scale page strides must be in [0, 2^31)", what);
  FD_REQUIRE(fd_aligned16(c->k) && fd_aligned16(c->v), FD_ERR_ALIGNMENT, "%s: the cache must be 16-byte aligned", what);
  out->k = static_cast<unsigned char*>(c->k);
  out->v = static_cast<unsigned char*>(c->v);
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->page = st[0] * elem;
  out->head = st[1] * elem;
  out->row = st[2] * elem;
  out->s_page = ss[0];
  out->s_head = ss[1];
  out->table = c->page_table;
  out->lens = c->cache_lens;
  out->table_stride = c->table_stride;
  out->n_pages = c->n_pages;
  out->max_pages = c->max_pages;
  out->shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
  return FD_OK;
}

// New tokens [start, end) of the T axis of request r, clamped to [0, seq_len]: a
// malformed offset table cannot move an access outside the tensors.
__device__ __forceinline__ void request_rows(const int32_t* cu, int r, int seq_len, int* start, int* end) {
  if (cu == nullptr) {
    *start = 0;
    *end = seq_len;
  } else {
    *start = min(max(cu[r], 0), seq_len);
    *end = min(max(cu[r + 1], *start), seq_len);
  }
}

__device__ __forceinline__ int request_keys(const PagedView& c, int r) {
  return min(max(c.lens[r], 0), c.max_pages << c.shift);
}

// Scale byte -> 2^(byte - 127).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

}  // namespace
