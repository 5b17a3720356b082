// Shared pieces of the 4-bit paged cache's kernels (paged_q4.hip, paged_q4_attn.hip).
#pragma once

#include "paged.h"
#include "../../include/butterfly_amd_paged_q4.h"

namespace bfly {

// The four tensors of a pair of 4-bit pages, strides in bytes.
struct Q4Ptr {
  PagePtr kc, ks, vc, vs;
};
inline Q4Ptr q4_ptr(const bfly_q4_pages_t& p) {
  return Q4Ptr{page_ptr(p.k_codes, p.k_codes_page, p.k_codes_head, p.k_codes_row, 1),
               page_ptr(p.k_scales, p.k_scales_page, p.k_scales_head, p.k_scales_row, 1),
               page_ptr(p.v_codes, p.v_codes_page, p.v_codes_head, p.v_codes_row, 1),
               page_ptr(p.v_scales, p.v_scales_page, p.v_scales_head, p.v_scales_row, 1)};
}

// The host's checks of such pages; BFLY_OK or an error.
int q4_check_pages(const char* what, const bfly_q4_pages_t& p, int64_t head_dim);
inline bool q4_aligned(const bfly_q4_pages_t& p) {
  return aligned16(p.k_codes) && aligned16(p.k_scales) && aligned16(p.v_codes) && aligned16(p.v_scales);
}
inline bool q4_given(const bfly_q4_pages_t& p) { return p.k_codes && p.k_scales && p.v_codes && p.v_scales; }

}  // namespace bfly
