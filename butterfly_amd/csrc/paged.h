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

// The host's checks of a pair of page tensors (elements of `esize` bytes); BFLY_OK or an error.
int paged_check_pages(const char* what, const bfly_pages_t& p, int64_t esize);

inline PagePtr page_ptr(void* base, int64_t page, int64_t head, int64_t row, int64_t esize) {
  return PagePtr{static_cast<char*>(base), page * esize, head * esize, (int)(row * esize)};
}
inline PagePtr k_page_ptr(const bfly_pages_t& p, int64_t esize) {
  return page_ptr(p.k, p.k_page_stride, p.k_head_stride, p.k_row_stride, esize);
}
inline PagePtr v_page_ptr(const bfly_pages_t& p, int64_t esize) {
  return page_ptr(p.v, p.v_page_stride, p.v_head_stride, p.v_row_stride, esize);
}

}  // namespace bfly
