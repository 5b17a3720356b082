// One new token of every request over its pages (include/butterfly_amd_paged.h).
//
//   s_t = scale q . k_t for the positions t it sees, m = max s_t, l = sum exp(s_t - m),
//   o = (sum exp(s_t - m) v_t) / l, with running m and l over one pass of the keys.
#include "paged.h"

namespace bfly {

constexpr float kPagedNeg = -1e30f;   // the largest score of a request without tokens

struct PagedAttnArgs {
  const char* q;
  PagePtr kp, vp;
  const int32_t* table;
  const int32_t* lengths;
  void* out;
  float* l;
  float* m;
  int64_t q_req, q_head, table_stride;   // bytes, bytes, elements
  int64_t capacity;
  int num_pages, hq, hkv, shift, window;
  float scale;
};

// A workgroup per (request, query head): wave w takes keys w, w + 4, ..., a lane D / 64 elements.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_attn_kernel(PagedAttnArgs a) {
  constexpr int E = D / 64;
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kvh = h / (a.hq / a.hkv);
  const int len = a.lengths[b];
  const bool off_table = (int64_t)len > a.capacity;
  const int n = len <= 0 || off_table ? 0 : len;
  const int lo = a.window > 0 && n > a.window ? n - a.window : 0;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
  const T* qr = reinterpret_cast<const T*>(a.q + b * a.q_req + h * a.q_head);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = to_f32(qr[lane * E + e]);
    acc[e] = 0.f;
  }
  bool bad = off_table;
  for (int t = lo + wave; t < n; t += 4) {
    int page = a.table[b * a.table_stride + (t >> a.shift)];
    if (page < 0 || page >= a.num_pages) {
      bad = true;
      page = 0;
    }
    const int r = t & ((1 << a.shift) - 1);
    const T* k = reinterpret_cast<const T*>(a.kp.row(page, kvh, r));
    const T* v = reinterpret_cast<const T*>(a.vp.row(page, kvh, r));
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], to_f32(k[lane * E + e]), s);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    s *= a.scale;
    const float nm = fmaxf(m, s);
    const float ref = nm == -INFINITY ? 0.f : nm;
    const float c = expf(m - ref), p = expf(s - ref);
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(p, to_f32(v[lane * E + e]), acc[e] * c);
    m = nm;
  }
  __shared__ float sm[4], sl[4], so[4][D];
  __shared__ int sbad;
  if (threadIdx.x == 0) sbad = 0;
  __syncthreads();
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
    if (bad) sbad = 1;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[wave][lane * E + e] = acc[e];
  __syncthreads();
  const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float ref = mm == -INFINITY ? 0.f : mm;
  float w[4], ll = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = expf(sm[i] - ref);
    ll += w[i] * sl[i];
  }
  const int64_t row = (int64_t)b * a.hq + h;
  const bool nan = sbad != 0;
  for (int c = threadIdx.x; c < D; c += 256) {
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) y += w[i] * so[i][c];
    y = nan ? __builtin_nanf("") : n > lo ? y / ll : 0.f;
    static_cast<T*>(a.out)[row * D + c] = from_f32<T>(y);
  }
  if (threadIdx.x == 0 && a.l != nullptr) {
    a.l[row] = nan ? __builtin_nanf("") : n > lo ? ll : 0.f;
    a.m[row] = nan ? __builtin_nanf("") : n > lo ? mm : kPagedNeg;
  }
}

}  // namespace bfly

using namespace bfly;

extern "C" int64_t bfly_paged_attention_workspace_bytes(int64_t requests, int hq, int hkv, int head_dim,
                                                        int64_t table_width, int page_size, int window) {
  (void)requests; (void)hq; (void)hkv; (void)head_dim; (void)table_width; (void)page_size; (void)window;
  return 0;
}

extern "C" int bfly_paged_attention(const void* q, int dtype, int64_t requests, int hq, int hkv, int head_dim,
                                    int64_t q_request_stride, int64_t q_head_stride, const void* k_pages,
                                    const void* v_pages, int64_t num_pages, int page_size, int64_t k_page_stride,
                                    int64_t k_page_head_stride, int64_t k_page_row_stride, int64_t v_page_stride,
                                    int64_t v_page_head_stride, int64_t v_page_row_stride, const int32_t* block_table,
                                    int64_t table_width, int64_t table_stride, const int32_t* lengths, int window,
                                    float scale, void* out, float* l, float* m, void* workspace,
                                    int64_t workspace_bytes, hipStream_t stream) {
  BFLY_CHECK_ARG(dtype == BFLY_DTYPE_F32 || dtype == BFLY_DTYPE_BF16, "unsupported dtype %d", dtype);
  const int64_t es = dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(requests >= 0 && hq > 0 && hkv > 0 && hq % hkv == 0, "bad head counts hq=%d hkv=%d", hq, hkv);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("bfly_paged_attention: head_dim=%d unsupported (64, 128, 256)", head_dim);
    return BFLY_ERR_UNSUPPORTED;
  }
  const int rc = paged_check_pages("bfly_paged_attention", num_pages, page_size, es, k_page_stride, k_page_head_stride,
                                   k_page_row_stride, v_page_stride, v_page_head_stride, v_page_row_stride);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(window >= 0, "window must not be negative");
  BFLY_CHECK_ARG(table_width >= 0 && table_width <= INT32_MAX && (requests <= 1 || table_stride >= 0), "bad block table shape");
  BFLY_CHECK_ARG(q_request_stride >= 0 && q_head_stride >= 0 && q_request_stride * es % 16 == 0 && q_head_stride * es % 16 == 0,
                 "q strides must be multiples of 16 bytes");
  if (requests == 0) return BFLY_OK;
  BFLY_CHECK_ARG(q && k_pages && v_pages && lengths && out, "null pointer");
  BFLY_CHECK_ARG(table_width == 0 || block_table, "null pointer");
  BFLY_CHECK_ARG((l == nullptr) == (m == nullptr), "both l and m or neither");
  BFLY_CHECK_ARG(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out), "pointers must be 16-byte aligned");
  BFLY_CHECK_ARG(requests <= 65535, "at most 65535 requests");
  PagedAttnArgs a{};
  a.q = static_cast<const char*>(q);
  a.kp = {static_cast<char*>(const_cast<void*>(k_pages)), k_page_stride * es, k_page_head_stride * es, (int)(k_page_row_stride * es)};
  a.vp = {static_cast<char*>(const_cast<void*>(v_pages)), v_page_stride * es, v_page_head_stride * es, (int)(v_page_row_stride * es)};
  a.table = block_table; a.lengths = lengths; a.out = out; a.l = l; a.m = m;
  a.q_req = q_request_stride * es; a.q_head = q_head_stride * es; a.table_stride = table_stride;
  a.shift = __builtin_ctz(page_size); a.capacity = table_width << a.shift;
  a.num_pages = (int)num_pages; a.hq = hq; a.hkv = hkv; a.window = window; a.scale = scale;
  const dim3 grid((unsigned)hq, (unsigned)requests), block(256);
#define BFLY_PAGED(T, D) hipLaunchKernelGGL((paged_attn_kernel<T, D>), grid, block, 0, stream, a)
  if (dtype == BFLY_DTYPE_BF16) {
    if (head_dim == 64) BFLY_PAGED(__bf16, 64);
    else if (head_dim == 128) BFLY_PAGED(__bf16, 128);
    else BFLY_PAGED(__bf16, 256);
  } else {
    if (head_dim == 64) BFLY_PAGED(float, 64);
    else if (head_dim == 128) BFLY_PAGED(float, 128);
    else BFLY_PAGED(float, 256);
  }
#undef BFLY_PAGED
  BFLY_CHECK_LAUNCH("bfly_paged_attention");
  return BFLY_OK;
}
