// Paged key-value cache on gfx950: a step's bookkeeping on the device (pages, block table, slots,
// positions), rows into pages, and the decoder's q/k norm + RoPE on the way there.  The contracts are
// include/butterfly_amd_paged.h's; no counterpart in the reference's own code (the layers that the swap
// leaves dense keep the host model's cache, bna/integrations/qwen_mlx.py:1822-1846).
#include "paged.h"

namespace bfly {

// --------------------------------------------------------------------------- bookkeeping
// With P(x) = ceil(x / page), a request b that goes from old to new tokens gives back pages
// P(new)..P(old) - 1 or takes pages P(old)..P(new) - 1.  Every request's place among the rows, the given
// and the taken pages is an exclusive sum over the requests before it: one scan of three counts.
//
// plan_kernel is one workgroup: each thread sums a run of requests, one scan over the threads, then the
// writes.  Sums saturate at 2^32 - 1 (saturating addition of counts is associative, so the scan may
// regroup them), which is above every limit they are held against.
struct PlanArgs {
  int32_t* table;
  const int32_t* lengths;
  const int32_t* counts;
  int32_t* free_pages;
  const int32_t* state;
  int32_t* lengths_out;
  int32_t* state_out;
  int32_t* starts;
  int64_t* slots;
  int64_t* positions;
  int32_t* taken;          // [requests + 1]: pages taken by the requests before
  int32_t* given;          // [requests + 1]: pages given back by them
  int32_t* before;         // [requests + 1]: rows added by them
  int64_t table_stride, capacity;   // capacity: tokens a table row holds
  int requests, shift, free_capacity, num_rows;
  int fixed;               // rows that every request has (idle ones too), or 0: rows packed
};

struct PlanSum {
  uint32_t rows, give, take;
};
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ PlanSum operator+(PlanSum a, PlanSum b) {
  return {add_sat(a.rows, b.rows), add_sat(a.give, b.give), add_sat(a.take, b.take)};
}

struct PlanStep {
  int old_len, new_len, count;   // count: rows added
  int p_old, p_new;
  bool bad, full;
};
__device__ __forceinline__ PlanStep plan_step(const PlanArgs& a, int b) {
  PlanStep s;
  const int64_t n = a.lengths[b], c = a.counts[b], pages = ((int64_t)1 << a.shift) - 1;
  const int64_t m = n + c > 0 ? n + c : 0;
  s.bad = n < 0 || n > a.capacity;
  s.full = m > a.capacity;
  const bool ok = !s.bad && !s.full;
  s.old_len = ok ? (int)n : 0;
  s.new_len = ok ? (int)m : 0;
  s.count = ok && c > 0 ? (int)c : 0;
  s.p_old = (int)((s.old_len + pages) >> a.shift);
  s.p_new = (int)((s.new_len + pages) >> a.shift);
  return s;
}

// The b with sums[b] <= i < sums[b + 1] (0 <= i < sums[requests]).
__device__ __forceinline__ int plan_find(const int32_t* sums, int requests, int i) {
  int lo = 0, hi = requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid + 1] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Row i of the call: the request it belongs to (by binary search in the sums `starts`, or, with a fixed number of
// rows each, by division), its position, and its page: one the request has, or the one it takes, which the
// page's first row also writes to the table.
__device__ __forceinline__ void plan_row(const PlanArgs& a, const int32_t* starts, const int32_t* taken,
                                         const int32_t* new_len, int i, bool ok, int64_t stack) {
  int64_t slot = -1, pos = 0;
  int lo = 0, off_row = 0;                           // the row's request, and which of its rows it is
  if (ok && a.fixed > 0) {
    lo = i / a.fixed;                                // (num_rows = requests * fixed)
    off_row = i - lo * a.fixed;
    ok = off_row < starts[lo + 1] - starts[lo];
  } else if (ok && i < starts[a.requests]) {
    lo = plan_find(starts, a.requests, i);
    off_row = i - starts[lo];
  } else {
    ok = false;
  }
  if (ok) {
    const int count = starts[lo + 1] - starts[lo], old_len = new_len[lo] - count;
    pos = (int64_t)old_len + off_row;
    const int p_old = (int)(((int64_t)old_len + (1 << a.shift) - 1) >> a.shift), j = (int)(pos >> a.shift);
    const int off = (int)(pos & ((1 << a.shift) - 1));
    int32_t* entry = a.table + lo * a.table_stride + j;
    int page;
    if (j < p_old) {
      page = *entry;
    } else {
      page = a.free_pages[stack - 1 - (taken[lo] + (j - p_old))];
      if (off == 0) *entry = page;
    }
    slot = ((int64_t)page << a.shift) + off;
  }
  a.slots[i] = slot;
  a.positions[i] = pos;
}

constexpr int kPlanMaxThreads = 1024;
constexpr int kPlanLds = 2048;     // requests whose sums the one-launch form keeps in LDS

template <bool kRows>
__global__ void __launch_bounds__(kPlanMaxThreads) plan_kernel(PlanArgs a) {
  __shared__ PlanSum part[kPlanMaxThreads / 64];
  __shared__ int flags;
  __shared__ int32_t s_starts[kRows ? kPlanLds + 1 : 1], s_taken[kRows ? kPlanLds + 1 : 1], s_given[kRows ? kPlanLds + 1 : 1],
      s_new[kRows ? kPlanLds : 1];
  const int t = threadIdx.x, nt = blockDim.x, lane = t & 63, wave = t >> 6;
  const int per = (a.requests + nt - 1) / nt;
  const int b0 = t * per < a.requests ? t * per : a.requests;
  const int b1 = b0 + per < a.requests ? b0 + per : a.requests;
  const int top = a.state[0], held = a.state[1];
  if (t == 0) flags = 0;
  __syncthreads();
  PlanSum mine{0, 0, 0};
  int bad = 0;
  for (int b = b0; b < b1; ++b) {
    const PlanStep s = plan_step(a, b);
    bad |= s.bad ? 1 : s.full ? 2 : a.fixed > 0 && s.count > a.fixed ? 4 : 0;
    mine = mine + PlanSum{(uint32_t)s.count, (uint32_t)(s.p_old > s.p_new ? s.p_old - s.p_new : 0),
                          (uint32_t)(s.p_new > s.p_old ? s.p_new - s.p_old : 0)};
  }
  PlanSum up = mine;                                // inclusive over the wave
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const PlanSum v{__shfl_up(up.rows, o), __shfl_up(up.give, o), __shfl_up(up.take, o)};
    if (lane >= o) up = up + v;
  }
  if (lane == 63) part[wave] = up;
  if (bad) atomicOr(&flags, bad);
  __syncthreads();
  PlanSum before{0, 0, 0}, total{0, 0, 0};
  for (int w = 0; w < nt / 64; ++w) {
    if (w == wave) before = total;
    total = total + part[w];
  }
  {
    // the sum before this thread: its inclusive sum without its own (exact where nothing saturated;
    // where something did, the call refuses below and the sums are not used)
    before = before + PlanSum{up.rows - mine.rows, up.give - mine.give, up.take - mine.take};
  }
  const int64_t stack = (int64_t)top + total.give;
  int err = held;
  if (err == 0) {
    if (flags & 1) err = BFLY_PAGED_BAD_LENGTH;
    else if (flags & 2) err = BFLY_PAGED_TABLE_FULL;
    else if (flags & 4 || total.rows > (uint32_t)a.num_rows) err = BFLY_PAGED_ROWS;
    else if (stack < (int64_t)total.take) err = BFLY_PAGED_NO_PAGES;
    else if (top < 0 || top > a.free_capacity || stack > a.free_capacity) err = BFLY_PAGED_FREE_LIST;
  }
  const bool ok = err == 0;
  int32_t* rows = kRows ? s_starts : a.before;
  int32_t* taken = kRows ? s_taken : a.taken;
  int32_t* given = kRows ? s_given : a.given;
  // lengths may be updated in place: a thread reads its own requests before it writes them
  PlanSum at = before;
  for (int b = b0; b < b1; ++b) {
    const int32_t raw = a.lengths[b];
    const PlanStep s = plan_step(a, b);
    a.lengths_out[b] = ok ? s.new_len : raw;
    a.starts[b] = ok ? (a.fixed > 0 ? b * a.fixed : (int)at.rows) : 0;
    rows[b] = (int)at.rows;
    if constexpr (kRows) {
      s_new[b] = s.new_len;
    }
    taken[b] = (int)at.take;
    given[b] = (int)at.give;
    at = at + PlanSum{(uint32_t)s.count, (uint32_t)(s.p_old > s.p_new ? s.p_old - s.p_new : 0),
                      (uint32_t)(s.p_new > s.p_old ? s.p_new - s.p_old : 0)};
  }
  if (t == 0) {
    a.starts[a.requests] = ok ? (a.fixed > 0 ? a.requests * a.fixed : (int)total.rows) : 0;
    rows[a.requests] = (int)total.rows;
    taken[a.requests] = (int)total.take;
    given[a.requests] = (int)total.give;
  }
  __syncthreads();                                  // state is read by every thread before it is written
  if (t == 0) {
    a.state_out[0] = ok ? (int)(stack - total.take) : top;
    a.state_out[1] = err;
  }
  if (ok && total.give != 0) {
    // the pages that are given back, a thread each: one request may leave with thousands
    const int32_t* len = kRows ? s_new : a.lengths_out;
    for (int i = t; i < (int)total.give; i += nt) {
      const int b = plan_find(given, a.requests, i);
      const int j = (int)(((int64_t)len[b] + (1 << a.shift) - 1) >> a.shift) + i - given[b];
      a.free_pages[stack - 1 - i] = a.table[b * a.table_stride + j];
    }
    __syncthreads();
  }
  if constexpr (kRows)
    for (int i = t; i < a.num_rows; i += nt) plan_row(a, s_starts, s_taken, s_new, i, ok, stack);
}

// The rows of a call with many of them, after plan_kernel<false>: a thread each.
__global__ void __launch_bounds__(256) plan_rows_kernel(PlanArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.num_rows) return;
  const bool ok = a.state_out[1] == 0;
  plan_row(a, a.before, a.taken, a.lengths_out, i, ok, (int64_t)a.state_out[0] + a.taken[a.requests]);
}

// --------------------------------------------------------------------------- rows into pages
// 16-byte pieces, a thread each: `per` pieces make a head's row.  Bound by the rows' bytes, read once and
// written once.
struct AppendArgs {
  const char* k;
  const char* v;
  const int64_t* slots;
  PagePtr kp, vp;
  int64_t k_row, k_head, v_row, v_head;   // bytes
  int64_t limit;                          // num_pages * page_size
  unsigned pieces;                        // of k (and of v), below 2^31
  unsigned hkv, per;
  int shift;
};

__global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs a) {
  unsigned i = blockIdx.x * 256u + threadIdx.x;     // below 2^32: 2^31 pieces of each at most
  const bool is_v = i >= a.pieces;
  if (is_v) i -= a.pieces;
  if (i >= a.pieces) return;
  const unsigned item = i / a.per, pc = i - item * a.per;
  const unsigned r = item / a.hkv, h = item - r * a.hkv;
  const int64_t row = r;
  const int64_t slot = a.slots[row];
  if (slot < 0 || slot >= a.limit) return;
  const char* src = is_v ? a.v + row * a.v_row + h * a.v_head : a.k + row * a.k_row + h * a.k_head;
  const PagePtr& p = is_v ? a.vp : a.kp;
  const uint4 x = *reinterpret_cast<const uint4*>(src + 16 * pc);
  *reinterpret_cast<uint4*>(p.row(slot >> a.shift, h, (int)(slot & ((1 << a.shift) - 1))) + 16 * pc) = x;
}

// --------------------------------------------------------------------------- norm, RoPE, rows into pages
// A group of LPR lanes holds one head's row of a token, E = 16 bytes of it a lane: mean square by
// shuffles inside the group, weight, then rotate-half with the lane that holds the other half
// (rotary / 2 elements away, whole lanes since rotary is a multiple of 16).  fp32 from the loads to the
// one rounding of each output: y = x * rsqrt(mean x^2 + eps) * w, z = y cos + rotate_half(y) sin.
//
// kHeads = 1: a decode step's few rows, spread as wide as they go; what they write stays in the caches for the
// attention that follows.  kHeads = 4, from kManyHeads heads' rows on: a group takes four heads of a token, so
// four loads are under way over one position's cos and sin, and moves them past the caches.
// Both sides, us (16/4 heads, whole rotation; one head / four; the rule changes at 2731 rows):
//            32 rows     1024         2048         2731         4096         16384
//   bf16  64  2.8 / 5.5   4.4 / 6.5    6.0 / 7.2    6.8 / 7.7    8.9 / 9.0   29.2 / 25.8
//   bf16 128  2.9 / 5.9   6.0 / 7.4    9.0 / 9.5   10.5 / 11.1  16.0 / 15.3  51.6 / 45.3
//   bf16 256  2.9 / 6.3   9.1 / 9.7   16.1 / 14.9  20.7 / 18.9  29.5 / 26.8   102 / 84.6
//   fp32  64  2.5 / 4.6   5.0 / 6.0    7.4 / 7.6    8.7 / 8.8   13.0 / 11.9  41.9 / 39.8
//   fp32 128  2.6 / 4.8   7.7 / 7.7   13.5 / 11.8  16.8 / 15.5  23.7 / 23.3  85.1 / 73.9
//   fp32 256  2.7 / 4.9  13.8 / 12.4  24.5 / 23.7  30.1 / 28.7  44.9 / 40.1   176 / 142
constexpr int64_t kManyHeads = 1 << 16;

struct RopeAppendArgs {
  const char* q;
  const char* k;
  const char* v;
  const void* qw;
  const void* kw;
  const float* cos;
  const float* sin;
  const int64_t* positions;
  const int64_t* slots;
  char* q_out;
  PagePtr kp, vp;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // bytes
  int64_t limit, table_rows;
  unsigned items;                         // rows x groups of heads, below 2^31
  int hq, hkv, shift, rot;
  float eps;
};

template <typename T, int D, int kHeads>
__global__ void __launch_bounds__(256) paged_rope_append_kernel(RopeAppendArgs a) {
  constexpr int E = 16 / sizeof(T), LPR = D / E;   // lanes a row: 8 (bf16, 64) to 64 (fp32, 256)
  typedef T vec __attribute__((ext_vector_type(E)));
  const int gl = threadIdx.x % LPR;
  const unsigned item = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;
  if (item >= a.items) return;                     // whole groups
  const unsigned nh = a.hq + 2 * a.hkv, chunks = (nh + kHeads - 1) / kHeads, r0 = item / chunks;
  const int64_t row = r0;
  const int head0 = (int)(item - r0 * chunks) * kHeads;
  const int64_t slot = a.slots[row], pos = a.positions[row];
  const bool keep = slot >= 0 && slot < a.limit, inside = pos >= 0 && pos < a.table_rows;
  vec x[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int head = head0 + i;
    if (kHeads > 1 && head >= (int)nh) break;
    const bool is_q = head < a.hq, is_v = head >= a.hq + a.hkv;
    const char* src = is_q ? a.q + row * a.q_row + head * a.q_head
                           : is_v ? a.v + row * a.v_row + (head - a.hq - a.hkv) * a.v_head
                                  : a.k + row * a.k_row + (head - a.hq) * a.k_head;
    const vec* p = reinterpret_cast<const vec*>(src + 16 * gl);
    x[i] = kHeads > 1 ? __builtin_nontemporal_load(p) : *p;
  }
  const int half = a.rot / 2 / E;                  // lanes to the other half
  const int lane = threadIdx.x & 63;
  const int other = gl < half ? lane + half : gl < 2 * half ? lane - half : lane;
  const bool turned = gl < 2 * half;
  float c[E], s[E];
  {
    const int64_t at = turned ? (inside ? pos : 0) * a.rot + E * gl : 0;
#pragma unroll
    for (int e4 = 0; e4 < E; e4 += 4) {
      const f32x4 cv = *reinterpret_cast<const f32x4*>(a.cos + at + (turned ? e4 : 0));
      const f32x4 sv = *reinterpret_cast<const f32x4*>(a.sin + at + (turned ? e4 : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e4 + e] = turned ? cv[e] : 1.f;
        s[e4 + e] = gl < half ? -sv[e] : sv[e];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int head = head0 + i;
    if (kHeads > 1 && head >= (int)nh) break;
    const bool is_q = head < a.hq, is_v = head >= a.hq + a.hkv;
    if (!is_q && !keep) continue;
    const int h = is_q ? head : is_v ? head - a.hq - a.hkv : head - a.hq;
    char* dst = is_q ? a.q_out + ((row * a.hq + h) * D) * (int64_t)sizeof(T)
                     : (is_v ? a.vp : a.kp).row(slot >> a.shift, h, (int)(slot & ((1 << a.shift) - 1)));
    if (!is_v) {
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = to_f32(x[i][e]);
      const T* w = static_cast<const T*>(is_q ? a.qw : a.kw);
      if (w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor(ss, o);
        const float r = rsqrtf(ss / (float)D + a.eps);
        const vec wv = *reinterpret_cast<const vec*>(w + E * gl);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = y[e] * r * to_f32(wv[e]);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float z = __shfl(y[e], other);
        const float t = y[e] * c[e] + z * s[e];
        x[i][e] = from_f32<T>(!inside ? __builtin_nanf("") : turned ? t : y[e]);
      }
    }
    vec* p = reinterpret_cast<vec*>(dst + 16 * gl);
    if constexpr (kHeads > 1) __builtin_nontemporal_store(x[i], p);
    else *p = x[i];
  }
}

int paged_check_pages(const char* what, const bfly_pages_t& p, int64_t esize) {
  BFLY_CHECK_ARG(p.page_size >= 16 && p.page_size <= 1024 && (p.page_size & (p.page_size - 1)) == 0,
                 "%s: page_size %lld must be a power of two from 16 to 1024", what, (long long)p.page_size);
  BFLY_CHECK_ARG(p.num_pages > 0 && p.num_pages <= INT32_MAX, "%s: bad num_pages", what);
  for (const int64_t s : {p.k_page_stride, p.k_head_stride, p.k_row_stride, p.v_page_stride, p.v_head_stride, p.v_row_stride})
    BFLY_CHECK_ARG(s >= 0 && s < ((int64_t)1 << 48) && (s * esize) % 16 == 0,
                   "%s: page strides must be multiples of 16 bytes", what);
  // offsets inside a page and head are kept in 32 bits
  BFLY_CHECK_ARG(p.k_row_stride * esize * p.page_size <= INT32_MAX && p.v_row_stride * esize * p.page_size <= INT32_MAX,
                 "%s: row stride too large", what);
  return BFLY_OK;
}

static bool strides16(std::initializer_list<int64_t> st, int64_t esize) {
  for (int64_t s : st)
    if (s < 0 || s >= ((int64_t)1 << 48) || (s * esize) % 16 != 0) return false;
  return true;
}

}  // namespace bfly

using namespace bfly;

extern "C" int bfly_paged_plan(const bfly_paged_plan_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_plan_args_t& x = *args;
  BFLY_CHECK_ARG(x.requests >= 0 && x.requests <= (1 << 24) && x.table_width >= 0 && x.table_width <= INT32_MAX,
                 "bad block table shape");
  BFLY_CHECK_ARG(x.requests <= 1 || x.table_stride >= x.table_width, "block table rows overlap");
  BFLY_CHECK_ARG(x.num_rows >= 0 && x.num_rows <= INT32_MAX && x.free_capacity >= 0 && x.free_capacity <= INT32_MAX,
                 "num_rows and the free list must stay below 2^31");
  BFLY_CHECK_ARG(x.page_size >= 16 && x.page_size <= 1024 && (x.page_size & (x.page_size - 1)) == 0,
                 "page_size %lld must be a power of two from 16 to 1024", (long long)x.page_size);
  BFLY_CHECK_ARG(x.rows_each >= 0 && (x.rows_each == 0 || (x.rows_each <= INT32_MAX && x.num_rows == x.requests * x.rows_each)),
                 "num_rows must be the requests' rows_each");
  BFLY_CHECK_ARG(x.state && x.state_out && x.starts, "null pointer");
  BFLY_CHECK_ARG(x.requests == 0 || (x.lengths && x.counts && x.lengths_out), "null pointer");
  BFLY_CHECK_ARG(x.requests * x.table_width == 0 || x.block_table, "null pointer");
  BFLY_CHECK_ARG(x.free_capacity == 0 || x.free_pages, "null pointer");
  BFLY_CHECK_ARG(x.num_rows == 0 || (x.slots && x.positions), "null pointer");
  BFLY_CHECK_ARG(x.workspace && x.workspace_bytes >= (x.requests + 1) * 12 && (reinterpret_cast<uintptr_t>(x.workspace) & 3) == 0,
                 "workspace too small");
  PlanArgs a{};
  a.table = x.block_table; a.lengths = x.lengths; a.counts = x.counts; a.free_pages = x.free_pages; a.state = x.state;
  a.lengths_out = x.lengths_out; a.state_out = x.state_out; a.starts = x.starts; a.slots = x.slots; a.positions = x.positions;
  a.taken = static_cast<int32_t*>(x.workspace);
  a.given = a.taken + x.requests + 1;
  a.before = a.given + x.requests + 1;
  a.table_stride = x.table_stride;
  a.shift = __builtin_ctzll(x.page_size);
  const int64_t cap = x.table_width << a.shift;
  a.capacity = cap < INT32_MAX ? cap : INT32_MAX;
  a.requests = (int)x.requests; a.free_capacity = (int)x.free_capacity; a.num_rows = (int)x.num_rows;
  a.fixed = (int)x.rows_each;
  const dim3 block(x.requests <= 256 && x.num_rows <= 256 ? 256 : kPlanMaxThreads);
  if (x.requests <= kPlanLds && x.num_rows <= 4096) {
    hipLaunchKernelGGL(plan_kernel<true>, dim3(1), block, 0, stream, a);
  } else {
    hipLaunchKernelGGL(plan_kernel<false>, dim3(1), block, 0, stream, a);
    if (x.num_rows > 0)
      hipLaunchKernelGGL(plan_rows_kernel, dim3((unsigned)((x.num_rows + 255) / 256)), dim3(256), 0, stream, a);
  }
  BFLY_CHECK_LAUNCH("bfly_paged_plan");
  return BFLY_OK;
}

extern "C" int bfly_paged_append(const bfly_paged_append_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_append_args_t& x = *args;
  BFLY_CHECK_ARG(x.dtype == BFLY_DTYPE_F32 || x.dtype == BFLY_DTYPE_BF16, "unsupported dtype %lld", (long long)x.dtype);
  const int64_t es = x.dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(x.rows >= 0 && x.rows <= INT32_MAX && x.hkv > 0 && x.hkv <= 65535 && x.head_dim > 0 && x.head_dim <= 65535,
                 "bad shape");
  BFLY_CHECK_ARG(x.head_dim * es % 16 == 0, "head_dim %lld is not whole 16-byte pieces", (long long)x.head_dim);
  const int rc = paged_check_pages("bfly_paged_append", x.pages, es);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(strides16({x.k_row_stride, x.k_head_stride, x.v_row_stride, x.v_head_stride}, es),
                 "row and head strides must be multiples of 16 bytes");
  if (x.rows == 0) return BFLY_OK;
  BFLY_CHECK_ARG(x.k && x.v && x.slots && x.pages.k && x.pages.v, "null pointer");
  BFLY_CHECK_ARG(aligned16(x.k) && aligned16(x.v) && aligned16(x.pages.k) && aligned16(x.pages.v),
                 "pointers must be 16-byte aligned");
  AppendArgs a{};
  a.k = static_cast<const char*>(x.k); a.v = static_cast<const char*>(x.v); a.slots = x.slots;
  a.kp = k_page_ptr(x.pages, es); a.vp = v_page_ptr(x.pages, es);
  a.k_row = x.k_row_stride * es; a.k_head = x.k_head_stride * es; a.v_row = x.v_row_stride * es; a.v_head = x.v_head_stride * es;
  a.limit = x.pages.num_pages * x.pages.page_size; a.hkv = (unsigned)x.hkv; a.per = (unsigned)(x.head_dim * es / 16);
  a.shift = __builtin_ctzll(x.pages.page_size);
  // (rows < 2^31, hkv and per < 2^16 and 2^14: no overflow)
  BFLY_CHECK_ARG(x.rows * x.hkv * a.per < ((int64_t)1 << 31) - 256, "too many rows");
  a.pieces = (unsigned)(x.rows * x.hkv * a.per);
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)((2 * (int64_t)a.pieces + 255) / 256)), dim3(256), 0, stream, a);
  BFLY_CHECK_LAUNCH("bfly_paged_append");
  return BFLY_OK;
}

extern "C" int bfly_paged_rope_append(const bfly_paged_rope_append_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_rope_append_args_t& x = *args;
  BFLY_CHECK_ARG(x.dtype == BFLY_DTYPE_F32 || x.dtype == BFLY_DTYPE_BF16, "unsupported dtype %lld", (long long)x.dtype);
  const int64_t es = x.dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(x.rows >= 0 && x.rows <= INT32_MAX, "bad shape");
  BFLY_CHECK_ARG(x.hkv > 0 && x.hq > 0 && x.hq <= (1 << 20) && x.hkv <= x.hq && x.hq % x.hkv == 0,
                 "bad head counts hq=%lld hkv=%lld", (long long)x.hq, (long long)x.hkv);
  if (x.head_dim != 64 && x.head_dim != 128 && x.head_dim != 256) {
    set_error("bfly_paged_rope_append: head_dim=%lld unsupported (64, 128, 256)", (long long)x.head_dim);
    return BFLY_ERR_UNSUPPORTED;
  }
  BFLY_CHECK_ARG(x.rotary_dim > 0 && x.rotary_dim <= x.head_dim && x.rotary_dim % 16 == 0,
                 "rotary_dim %lld must be a multiple of 16, at most head_dim", (long long)x.rotary_dim);
  BFLY_CHECK_ARG(x.table_rows > 0, "the cos/sin tables must have rows");
  const int rc = paged_check_pages("bfly_paged_rope_append", x.pages, es);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(strides16({x.q_row_stride, x.q_head_stride, x.k_row_stride, x.k_head_stride, x.v_row_stride,
                            x.v_head_stride}, es),
                 "row and head strides must be multiples of 16 bytes");
  if (x.rows == 0) return BFLY_OK;
  BFLY_CHECK_ARG(x.q && x.k && x.v && x.cos && x.sin && x.positions && x.slots && x.q_out && x.pages.k && x.pages.v,
                 "null pointer");
  BFLY_CHECK_ARG((x.q_weight == nullptr) == (x.k_weight == nullptr), "both norm weights or neither");
  BFLY_CHECK_ARG(aligned16(x.q) && aligned16(x.k) && aligned16(x.v) && aligned16(x.cos) && aligned16(x.sin) && aligned16(x.q_out) &&
                     aligned16(x.pages.k) && aligned16(x.pages.v) && aligned16(x.q_weight) && aligned16(x.k_weight),
                 "pointers must be 16-byte aligned");
  RopeAppendArgs a{};
  a.q = static_cast<const char*>(x.q); a.k = static_cast<const char*>(x.k); a.v = static_cast<const char*>(x.v);
  a.qw = x.q_weight; a.kw = x.k_weight; a.cos = x.cos; a.sin = x.sin; a.positions = x.positions; a.slots = x.slots;
  a.q_out = static_cast<char*>(x.q_out);
  a.kp = k_page_ptr(x.pages, es); a.vp = v_page_ptr(x.pages, es);
  a.q_row = x.q_row_stride * es; a.q_head = x.q_head_stride * es; a.k_row = x.k_row_stride * es;
  a.k_head = x.k_head_stride * es; a.v_row = x.v_row_stride * es; a.v_head = x.v_head_stride * es;
  a.limit = x.pages.num_pages * x.pages.page_size; a.table_rows = x.table_rows; a.hq = (int)x.hq; a.hkv = (int)x.hkv;
  a.shift = __builtin_ctzll(x.pages.page_size); a.rot = (int)x.rotary_dim; a.eps = (float)x.eps;
  const int64_t heads = x.hq + 2 * x.hkv;
  BFLY_CHECK_ARG(x.rows * heads < ((int64_t)1 << 31) - 256, "too many rows");
  const bool many = x.rows * heads >= kManyHeads;
  a.items = (unsigned)(x.rows * (many ? (heads + 3) / 4 : heads));
  const int64_t lanes = x.head_dim * es / 16, blocks = (a.items * lanes + 255) / 256;
  BFLY_CHECK_ARG(blocks < (1 << 24), "too many rows");       // a grid holds fewer than 2^32 threads
  const dim3 grid((unsigned)blocks), block(256);
#define BFLY_ROPE(T, D)                                                                                \
  do {                                                                                                 \
    if (many) hipLaunchKernelGGL((paged_rope_append_kernel<T, D, 4>), grid, block, 0, stream, a);      \
    else hipLaunchKernelGGL((paged_rope_append_kernel<T, D, 1>), grid, block, 0, stream, a);           \
  } while (0)
  if (x.dtype == BFLY_DTYPE_BF16) {
    if (x.head_dim == 64) BFLY_ROPE(__bf16, 64);
    else if (x.head_dim == 128) BFLY_ROPE(__bf16, 128);
    else BFLY_ROPE(__bf16, 256);
  } else {
    if (x.head_dim == 64) BFLY_ROPE(float, 64);
    else if (x.head_dim == 128) BFLY_ROPE(float, 128);
    else BFLY_ROPE(float, 256);
  }
#undef BFLY_ROPE
  BFLY_CHECK_LAUNCH("bfly_paged_rope_append");
  return BFLY_OK;
}
