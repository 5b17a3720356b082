// Shared pieces of the paged cache's kernels (paged.hip, paged_attn.hip).
#pragma once

#include "bfly_common.h"
#include "../../include/butterfly_amd_paged.h"

namespace bfly {

// Pages [num_pages, hkv, page_size, head_dim] with strides in bytes; the row of a page in 64 bits.
struct PagePtr {
  char* base;
  int64_t page, head;
  int row_bytes;
  __device__ __forceinline__ char* row(int64_t id, int h, int r) const {
    return base + id * page + h * head + r * row_bytes;
  }
};

// The host's checks of page_size, num_pages and the six page strides (elements); BFLY_OK or an error.
int paged_check_pages(const char* what, int64_t num_pages, int page_size, int64_t esize, int64_t k_page,
                      int64_t k_head, int64_t k_row, int64_t v_page, int64_t v_head, int64_t v_row);

}  // namespace bfly
