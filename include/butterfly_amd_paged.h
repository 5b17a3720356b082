/*
 * butterfly_amd paged serving -- C ABI of the paged key-value cache for the layers that keep dense
 * attention: one step's bookkeeping on the device, rows into pages, and one-token attention over pages.
 *
 * The swap leaves every layer it is not asked to replace on its stock attention (bna/integrations/
 * qwen_mlx.py:1822-1846, qwen_torch.py:1652-1700), whose cache the reference leaves to the host model;
 * so none of these has a counterpart in the reference's own code.
 *
 * Conventions are those of butterfly_amd.h (caller-owned device pointers, work enqueued on `stream`,
 * nothing allocates or synchronises, 0 or a negative BFLY_ERR_*), and:
 *   - arguments come in one struct a call, every member eight bytes wide (a caller in another language
 *     packs them in order).
 *   - pages are [num_pages, hkv, page_size, head_dim] with strides (in elements) of their own for page,
 *     head and row; head_dim is contiguous.  Base addresses are 16-byte aligned, strides multiples of
 *     16 bytes.  page_size is a power of two from 16 to 1024.
 *   - a slot is page * page_size + row of the page.  block_table is [requests, table_width] int32 with
 *     rows table_stride elements apart: entry j holds positions [j * page_size, (j + 1) * page_size).
 *     Entries behind a request's last page are neither read nor defined.
 *   - every index that is read on the device is checked there: none of them can lead outside the tensors.
 */
#ifndef BUTTERFLY_AMD_PAGED_H_
#define BUTTERFLY_AMD_PAGED_H_

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct bfly_pages {
  void* k;
  void* v;
  int64_t num_pages;
  int64_t page_size;
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
} bfly_pages_t;

/* Error codes of state[1] (bfly_paged_plan); the lowest that applies is kept. */
#define BFLY_PAGED_BAD_LENGTH 1 /* a length that is negative or beyond its table row */
#define BFLY_PAGED_TABLE_FULL 2 /* a request would outgrow its table row */
#define BFLY_PAGED_ROWS 3       /* the counts sum to more than num_rows */
#define BFLY_PAGED_NO_PAGES 4   /* the free list holds too few pages */
#define BFLY_PAGED_FREE_LIST 5  /* the free list's count is outside its array, or would be */

/*
 * Device: one step's bookkeeping.  Request b holds lengths[b] tokens; counts[b] > 0 appends that many,
 * counts[b] < 0 takes back the last -counts[b] (all of them at the most), 0 leaves it as it is.
 *   - free_pages [free_capacity] is a stack of state[0] page ids.  Pages that requests no longer need go
 *     on top of it (the first of them, in request order, topmost), then the pages that others need are
 *     taken from the top in request order and written to block_table.  So a step and the same step with
 *     its counts negated leave the free list as it was.
 *   - lengths_out [requests], state_out [2] = {free pages, error}; both may be the inputs themselves.
 *   - starts [requests + 1]: the first row of each request among the call's rows (exclusive sums of the
 *     positive counts).  slots and positions [num_rows] int64: where row starts[b] + i of request b goes
 *     and its position lengths[b] + i; rows behind the last have slot -1 and position 0.
 *   - rows_each > 0 (num_rows = requests * rows_each): every request has rows_each rows of its own instead,
 *     starts[b] = b * rows_each, for a batch in which some stay idle; no count may exceed it (code
 *     BFLY_PAGED_ROWS), and rows behind a request's count have slot -1 and position 0.
 *   - When something does not fit (codes above), or state[1] is already set, nothing changes: lengths,
 *     free list and table stay, state_out keeps the count and holds the code, starts are 0 and every slot
 *     is -1.  The code stays until the caller clears it.
 *   - workspace: (requests + 1) * 12 bytes, 4-byte aligned.
 * The tensors do not overlap otherwise.  requests at most 2^24; num_rows and free_capacity below 2^31.
 */
typedef struct bfly_paged_plan_args {
  int32_t* block_table;
  int64_t requests, table_width, table_stride;
  const int32_t* lengths;
  const int32_t* counts;
  int32_t* free_pages;
  int64_t free_capacity;
  const int32_t* state;
  int64_t page_size, num_rows, rows_each;
  int32_t* lengths_out;
  int32_t* state_out;
  int32_t* starts;
  int64_t* slots;
  int64_t* positions;
  void* workspace;
  int64_t workspace_bytes;
} bfly_paged_plan_args_t;
int bfly_paged_plan(const bfly_paged_plan_args_t* args, hipStream_t stream);

/*
 * Device: rows k, v [rows, hkv, head_dim] (row and head strides in elements, multiples of 16 bytes) into
 * their slots.  A row whose slot is negative or beyond the pages is passed over.  Of two rows with one
 * slot it is not defined which stays, element by element.  Any head_dim of whole 16-byte pieces.
 */
typedef struct bfly_paged_append_args {
  const void* k;
  const void* v;
  int64_t dtype, rows, hkv, head_dim;
  int64_t k_row_stride, k_head_stride, v_row_stride, v_head_stride;
  const int64_t* slots;
  bfly_pages_t pages;
} bfly_paged_append_args_t;
int bfly_paged_append(const bfly_paged_append_args_t* args, hipStream_t stream);

/*
 * Device: bfly_paged_append for a decoder's projection rows, with the per-head RMSNorm of q and k (weights
 * [head_dim] in the rows' type, or both NULL for none) and rotate-half RoPE on the way: position p of a row
 * picks row p of cos / sin [table_rows, rotary_dim] (fp32, contiguous); elements from rotary_dim on are not rotated.
 * q_out [rows, hq, head_dim] (contiguous) is written for every row, k and v go to their slots.  fp32 from
 * the inputs to the one rounding of each output.  A position outside the table gives NaN in q_out and in k.
 * head_dim 64, 128 or 256; rotary_dim a multiple of 16, at most head_dim.
 */
typedef struct bfly_paged_rope_append_args {
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
  bfly_pages_t pages;
} bfly_paged_rope_append_args_t;
int bfly_paged_rope_append(const bfly_paged_rope_append_args_t* args, hipStream_t stream);

/*
 * Device: one new token of every request over its pages.  q [requests, hq, head_dim] with request and head
 * strides (multiples of 16 bytes); query head h reads kv head h / (hq / hkv).  The token sees positions
 * [max(0, lengths[b] - window), lengths[b]) (window 0: all of them; its own key is the last).
 * out [requests, hq, head_dim] (contiguous); l and m [requests, hq] (both NULL, or fp32: the sum of
 * exp(score - m) and the largest score, as the stream entries of butterfly_amd.h give them).
 * A request without tokens (length <= 0) gives 0, 0 and -1e30.  A length beyond its table row, or a page
 * id outside the pages among those it reads, gives NaN in out, l and m of that request.
 * head_dim 64, 128 or 256.  workspace: bfly_paged_attention_workspace_bytes bytes, 16-byte aligned (it need
 * not be cleared; calls that overlap need one each).
 */
int64_t bfly_paged_attention_workspace_bytes(int dtype, int64_t requests, int hq, int hkv, int head_dim,
                                             int64_t table_width, int page_size, int window);
typedef struct bfly_paged_attention_args {
  const void* q;
  int64_t dtype, requests, hq, hkv, head_dim;
  int64_t q_request_stride, q_head_stride;
  bfly_pages_t pages;
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
} bfly_paged_attention_args_t;
int bfly_paged_attention(const bfly_paged_attention_args_t* args, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* BUTTERFLY_AMD_PAGED_H_ */
