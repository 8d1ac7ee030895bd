// What the kernels over a paged key/value cache share: the cache as they see
// it and the host's checks of the caller's description.
#pragma once

#include "abi_internal.h"
#include "slr_common.h"

namespace ssl {

// Strides in elements. A page number read from the table is used only after
// `has` accepted it.
struct PagedCache {
  char *k, *v;
  int64_t layer_stride, page_stride, head_stride, slot_stride;
  int64_t pages;
  const int32_t* table;
  int64_t table_stride;
  int layers, kv_heads, page, log2_page, head_dim;
  int seqs, cols;

  __device__ __forceinline__ bool has(int32_t page_no) const {
    return (uint32_t)page_no < (uint32_t)pages;
  }
};

// Checks `c` (the pools only where `pools`) and fills `out`.
int paged_cache(const char* what, const ssl_paged_cache& c, int64_t struct_bytes, bool pools,
                PagedCache* out);

}  // namespace ssl
