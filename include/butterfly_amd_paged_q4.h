/*
 * butterfly_amd paged serving in 4 bits -- C ABI of the paged key-value cache (butterfly_amd_paged.h) whose
 * rows are held as 4-bit affine codes: rows into pages, rows out of them, one-token attention over them.
 *
 * The layers that the swap leaves dense keep the host model's cache (bna/integrations/qwen_mlx.py:1822-1846),
 * which the reference may hold quantised (bna/integrations/mlx_kv_quant.py); these are its counterpart here
 * over pages of this build's own layout.
 *
 * Conventions are those of butterfly_amd_paged.h, and:
 *   - a row of head_dim elements is head_dim / group groups of `group` (32 or 64) consecutive elements.  An
 *     element is code * scale + bias, code 0..15, with a bf16 scale and bias for each group:
 *       bias = bf16(min), scale = bf16(max((max - min) / 15, 1e-8)) (each by way of fp32),
 *       code = (x - bias) / scale rounded to the nearest, to the even one of two, and held within 0..15,
 *     computed in 64 bits.  A group with an infinity or NaN, or whose bias or scale is none in bf16, has scale and bias NaN and
 *     codes 0: it reads as NaN.
 *   - codes: [num_pages, hkv, page_size, head_dim / 2] bytes, two codes a byte, the lower one first.  The n-th
 *     of 16 equal pieces of a row holds the n-th sixteenth (group / 16 codes) of every group, group by group.
 *   - scales: [num_pages, hkv, page_size, head_dim / group] pairs (scale, bias) of bf16.
 *   - codes and scales have strides of their own for page, head and row, in bytes: those of the codes are
 *     multiples of 16, those of the scales multiples of their row (4 * head_dim / group bytes, 16 at the
 *     most), base addresses 16-byte aligned.
 *   - head_dim 64, 128 or 256.
 */
#ifndef BUTTERFLY_AMD_PAGED_Q4_H_
#define BUTTERFLY_AMD_PAGED_Q4_H_

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct bfly_q4_pages {
  void* k_codes;
  void* k_scales;
  void* v_codes;
  void* v_scales;
  int64_t num_pages, page_size, group;
  int64_t k_codes_page, k_codes_head, k_codes_row;      /* strides in bytes */
  int64_t k_scales_page, k_scales_head, k_scales_row;
  int64_t v_codes_page, v_codes_head, v_codes_row;
  int64_t v_scales_page, v_scales_head, v_scales_row;
} bfly_q4_pages_t;

/*
 * Device: rows k, v [rows, hkv, head_dim] (fp32 or bf16; row and head strides in elements, multiples of 16
 * bytes) quantised into their slots.  A row whose slot is negative or beyond the pages is passed over; of two
 * rows with one slot it is not defined which stays, element by element.
 */
typedef struct bfly_paged_q4_append_args {
  const void* k;
  const void* v;
  int64_t dtype, rows, hkv, head_dim;
  int64_t k_row_stride, k_head_stride, v_row_stride, v_head_stride;
  const int64_t* slots;
  bfly_q4_pages_t pages;
} bfly_paged_q4_append_args_t;
int bfly_paged_q4_append(const bfly_paged_q4_append_args_t* args, hipStream_t stream);

/*
 * Device: bfly_paged_q4_append with the per-head RMSNorm of q and k and rotate-half RoPE on the way, as
 * bfly_paged_rope_append (butterfly_amd_paged.h).  q_out is computed in fp32; k up to its codes in 64 bits, so
 * that they do not depend on the order of a sum.  A position outside the table gives NaN in q_out and in k.
 */
typedef struct bfly_paged_q4_rope_append_args {
  const void* q;
  const void* k;
  const void* v;
  int64_t dtype, rows, hq, hkv, head_dim;
  int64_t q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride, v_head_stride;
  const void* q_weight;
  const void* k_weight;
  double eps;
  const float* cos;
  const float* sin;
  int64_t table_rows, rotary_dim;
  const int64_t* positions;
  const int64_t* slots;
  void* q_out;
  bfly_q4_pages_t pages;
} bfly_paged_q4_rope_append_args_t;
int bfly_paged_q4_rope_append(const bfly_paged_q4_rope_append_args_t* args, hipStream_t stream);

/*
 * Device: the first `tokens` rows of every request as dense k, v [requests, hkv, tokens, head_dim] (fp32 or
 * bf16, contiguous): code * scale + bias in fp32, rounded once.  A row whose block table entry is outside the
 * pages reads as NaN.  tokens at most table_width * page_size.
 */
typedef struct bfly_paged_q4_read_args {
  int64_t dtype, requests, hkv, head_dim, tokens;
  const int32_t* block_table;
  int64_t table_width, table_stride;
  void* k;
  void* v;
  bfly_q4_pages_t pages;
} bfly_paged_q4_read_args_t;
int bfly_paged_q4_read(const bfly_paged_q4_read_args_t* args, hipStream_t stream);

/*
 * Device: one new token of every request over its pages: bfly_paged_attention (butterfly_amd_paged.h) with
 * q and out in `dtype` (fp32 or bf16) and the keys and values as the codes stand for.
 * Queries of 2^110 and more, or of 2^107 and more times |scale|, and scales of v of 2^80 and more, may give
 * infinities or NaN; values whose weighted sum passes 2^124 may give infinities.
 * workspace: bfly_paged_q4_attention_workspace_bytes bytes, 16-byte aligned (it need not be cleared; calls
 * that overlap need one each).
 */
int64_t bfly_paged_q4_attention_workspace_bytes(int dtype, int64_t requests, int hq, int hkv, int head_dim,
                                                int64_t table_width, int page_size, int window);
typedef struct bfly_paged_q4_attention_args {
  const void* q;
  int64_t dtype, requests, hq, hkv, head_dim;
  int64_t q_request_stride, q_head_stride;
  bfly_q4_pages_t pages;
  const int32_t* block_table;
  int64_t table_width, table_stride;
  const int32_t* lengths;
  int64_t window;
  double scale;
  void* out;
  float* l;
  float* m;
  void* workspace;
  int64_t workspace_bytes;
} bfly_paged_q4_attention_args_t;
int bfly_paged_q4_attention(const bfly_paged_q4_attention_args_t* args, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* BUTTERFLY_AMD_PAGED_Q4_H_ */
