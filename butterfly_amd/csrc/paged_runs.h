// The schedule that the attention kernels over pages share (paged_attn.hip, paged_q4_attn.hip): which run of which
// request a workgroup takes, from the lengths on the device, and the join of a request's runs.
#pragma once

#include "paged.h"

namespace bfly {

constexpr float kPagedNeg = -1e30f;   // the largest score of a request without tokens
constexpr int kWaves = 4;             // waves of a workgroup, tiles of a round
constexpr int kMaxRuns = 512;         // RunArgs::runs at most
constexpr int kMinRun = 1;            // rounds of a run at least (c)
// A request of several runs has more than c rounds, so fewer than 2 rounds_b / c runs; all of them together, with
// c >= total / runs, fewer than twice the runs: the partials there can be.  (kSlack: the total is a sum of floats.)
constexpr int kSlack = 64;
constexpr int kMaxSlots = 2 * kMaxRuns + kSlack;
constexpr float kLog2e = 1.4426950408889634f;

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

struct RunArgs {
  const int32_t* table;
  const int32_t* lengths;
  void* out;
  float* l;
  float* m;
  float* part;                           // partials: [slot][rows][D], then [slot][rows] m and l
  float* part_ml;
  int4* join;                            // what to join: request, unit, runs, first slot
  int* joins;                            // how many of them
  int64_t table_stride;                  // elements
  int64_t capacity;                      // tokens a table row holds
  int requests, num_pages, hq, hkv, shift, window;
  int group, row_tiles, rows;            // query heads a kv head; 16-row parts of them; rows of a part at most
  int units;                             // hkv * row_tiles
  int runs;                              // in all, where requests and heads leave them
  int whole;                             // rounds that stay one run
  int direct;                            // every request is one run (its table row is that short)
  float scale;
};

// What a request's workgroups do, from its length.
struct Span {
  int lo, n;      // positions seen: [lo, n)
  int t0, tiles;  // tiles that hold them
  int rounds;     // four tiles each
  bool off;       // the length is beyond the table
};
template <int KT>
__device__ __forceinline__ Span span_of(const RunArgs& a, int len) {
  Span s;
  s.off = (int64_t)len > a.capacity;
  s.n = len <= 0 || s.off ? 0 : len;
  s.lo = a.window > 0 && s.n > a.window ? s.n - a.window : 0;
  s.t0 = s.lo / KT;
  s.tiles = s.n > 0 ? (s.n - 1) / KT + 1 - s.t0 : 0;
  s.rounds = (s.tiles + kWaves - 1) / kWaves;
  return s;
}

struct Run {
  int b, len;     // request (-1: none) and its length
  int sub;        // index inside the request
  int splits;     // runs of the request (per unit)
  int slot;       // partials before the request's
  int join;       // (request, unit) pairs of several runs before the request's
  int joins;      // and in all
};

// Sums over the wave's lanes on DPP (row shifts inside 16 lanes, then the rows' last lanes broadcast): lane 63
// of the inclusive scan holds the total.
template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp_shift(int x) { return __builtin_amdgcn_update_dpp(0, x, kCtrl, kRows, 0xf, false); }
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp_shift<0x111, 0xf>(x);     // row_shr:1, 2, 4, 8
  x += dpp_shift<0x112, 0xf>(x);
  x += dpp_shift<0x114, 0xf>(x);
  x += dpp_shift<0x118, 0xf>(x);
  x += dpp_shift<0x142, 0xa>(x);     // row_bcast:15 into rows 1 and 3
  x += dpp_shift<0x143, 0xc>(x);     // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ float wave_total(float x) {
  const auto step = [](float v, int w) { return v + __int_as_float(w); };
  x = step(x, dpp_shift<0x111, 0xf>(__float_as_int(x)));
  x = step(x, dpp_shift<0x112, 0xf>(__float_as_int(x)));
  x = step(x, dpp_shift<0x114, 0xf>(__float_as_int(x)));
  x = step(x, dpp_shift<0x118, 0xf>(__float_as_int(x)));
  x = step(x, dpp_shift<0x142, 0xa>(__float_as_int(x)));
  x = step(x, dpp_shift<0x143, 0xc>(__float_as_int(x)));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// The largest over the wave's lanes, in every lane (col_max4 over the lanes of a row of 16, which hold the
// same then).
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
  return col_max4(x);
}

// kEven: the runs as even as they can be (and fewer of them before they are short).
// The request that item `idx` falls into, where request b has units * splits_b items.  Every wave does it by
// itself: a lane sums a stretch of requests, one scan over the lanes, then the lane of the item walks its stretch.
template <int KT, bool kEven = false>
__device__ __forceinline__ Run plan_run(const RunArgs& a, int64_t idx) {
  if (a.direct) {                                   // no request can have several runs: item = (request, unit)
    const int b = (int)idx / a.units;
    return Run{b, a.lengths[b], (int)idx - b * a.units, 1, 0, 0, 0};
  }
  const int lane = threadIdx.x & 63;
  const int per = (a.requests + 63) >> 6;
  const int b0 = lane * per < a.requests ? lane * per : a.requests;
  const int b1 = b0 + per < a.requests ? b0 + per : a.requests;
  // (up to 64 requests a lane has one, in registers)
  const int len0 = b0 < b1 ? a.lengths[b0] : 0;
  const int first = span_of<KT>(a, len0).rounds;
  const auto each = [&](auto&& f) {
    if (per == 1) {
      if (b0 < b1) f(first);
    } else {
#pragma unroll 4
      for (int b = b0; b < b1; ++b) f(span_of<KT>(a, a.lengths[b]).rounds);
    }
  };
  float total = 0.f;
  each([&](int n) { total += (float)n; });
  total = wave_total(total) * (float)a.units;
  // fewer runs, of two rounds, before as many of one (kEven)
  const int most = __builtin_amdgcn_readfirstlane(kEven && total < 2.f * (float)a.runs ? a.runs / 2 : a.runs);
  // c fills the runs exactly if the requests' last, shorter runs fit among them; else room is left for one each
  const auto over = [&](float to) { return fminf(fmaxf(ceilf(total / to), (float)kMinRun), 1e9f); };
  int c = __builtin_amdgcn_readfirstlane((int)over((float)most));
  const auto runs = [&](int n) { return n > c && n > a.whole ? (int)(((unsigned)n + c - 1) / (unsigned)c) : 1; };
  int items = 0;
  each([&](int n) { items += runs(n); });
  const int64_t pairs = (int64_t)a.requests * a.units;
  if ((int64_t)__builtin_amdgcn_readlane(wave_scan(items), 63) * a.units > most && pairs < most) {
    int fits = __builtin_amdgcn_readfirstlane((int)over((float)(pairs < most / 2 ? most - (int)pairs : most / 2)));
    if (kEven && per == 1) {
      // the least c between the two whose runs fit, or near it: the longest run is the call's time
#pragma unroll 1
      for (int i = 0; i < 5 && fits - c > 1; ++i) {
        const int low = c, mid = c + (fits - c) / 2;
        c = mid;                                    // (what `runs` counts with)
        const int n = b0 < b1 ? runs(first) : 0;
        if ((int64_t)__builtin_amdgcn_readlane(wave_scan(n), 63) * a.units <= most) {
          fits = mid;
          c = low;
        }
      }
    }
    c = fits;
  }
  int slots = 0;                                    // low half: partials; high half: requests that have them (both
  items = 0;                                        // below kMaxSlots in all)
  const auto parts = [](int s) { return s > 1 ? s | 0x10000 : 0; };
  each([&](int n) {
    const int s = runs(n);
    items += s;
    slots += parts(s);
  });
  const int i_up = wave_scan(items), s_up = wave_scan(slots);
  const uint64_t mine = __ballot((int64_t)i_up * a.units > idx);
  Run r{-1, 0, 0, 0, 0, 0, (__builtin_amdgcn_readlane(s_up, 63) >> 16) * a.units};
  if (mine == 0) return r;
  const int owner = __builtin_ctzll(mine);
  int at = __builtin_amdgcn_readlane(i_up - items, owner), slot = __builtin_amdgcn_readlane(s_up - slots, owner);
  for (int b = owner * per;; ++b) {               // (a request of the owner's stretch holds idx)
    const int len = per == 1 ? __builtin_amdgcn_readlane(len0, owner) : a.lengths[b];
    const int s = runs(span_of<KT>(a, len).rounds);
    const int next = at + s;
    if ((int64_t)next * a.units > idx) {
      r.b = b;
      r.len = len;
      r.sub = (int)(idx - (int64_t)at * a.units);
      r.splits = s;
      r.slot = (slot & 0xffff) * a.units;
      r.join = (slot >> 16) * a.units;
      return r;
    }
    at = next;
    slot += parts(s);
  }
}

__device__ __forceinline__ void store4(float* o, f32x4 y, float f) { *reinterpret_cast<f32x4*>(o) = y * f; }
__device__ __forceinline__ void store4(__bf16* o, f32x4 y, float f) {
  y *= f;
  *reinterpret_cast<bf16x4*>(o) = __builtin_convertvector(y, bf16x4);
}

// The statistics of a row from its joined sums.  A row that sees nothing but scores of -inf has no softmax: its sum is
// NaN, as exp(-inf - -inf) gives (its output is 0 / 0).  NaN scores make the sum NaN, and then the maximum, which
// has passed over them (a maximum of +inf makes a NaN sum by itself).
template <typename T>
__device__ __forceinline__ void finish_stats(const RunArgs& a, int64_t row, float m, float l) {
  if (a.l == nullptr) return;
  const bool nan = l != l;
  a.l[row] = m == -INFINITY ? __builtin_nanf("") : l;
  a.m[row] = nan && m != INFINITY ? l : m;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

// The pages of the tile at key `first`: one for each 16 keys.  Keys outside [lo, n) share the page of the nearest key
// inside, so no entry behind the last page (or before the window) is read.
template <int U>
__device__ __forceinline__ void tile_ids(const RunArgs& a, const int32_t* row, int first, const Span& s, int (&id)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    unsigned t = (unsigned)first + 16 * u;
    t = t < (unsigned)s.lo ? s.lo : t > (unsigned)s.n - 1 ? s.n - 1 : t;
    id[u] = row[t >> a.shift];
  }
}
// Whether one of them is outside the pages: it is page 0 then.
template <int U>
__device__ __forceinline__ bool tile_bad(const RunArgs& a, int (&id)[U]) {
  bool bad = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if ((unsigned)id[u] >= (unsigned)a.num_pages) {
      bad = true;
      id[u] = 0;
    }
  }
  return bad;
}
// Where their rows lie.
template <int U>
__device__ __forceinline__ void tile_base(const RunArgs& a, const PagePtr& p, int h, int first, const int (&id)[U],
                                          const char* (&base)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) base[u] = p.row(id[u], h, (first + 16 * u) & ((1 << a.shift) - 1));
}


// Joins the requests of several runs (paged_attn.hip); nothing where there can be none.
void paged_merge(const RunArgs& a, int dtype, int head_dim, hipStream_t stream);

// The rounds (tiles of kt keys, kWaves of them) of a request at most.
inline int64_t most_rounds(int64_t capacity, int window, int kt) {
  const int64_t keys = window > 0 && window < capacity ? (int64_t)window + kt - 1 : capacity;
  return (keys + kWaves * kt - 1) / (kWaves * kt);
}

// Workspace of a call whose requests can have several runs.
inline int64_t run_workspace_bytes(int64_t rows, int64_t head_dim) {
  return (int64_t)kMaxSlots * (rows * (head_dim + 2) * 4 + 16) + 16;
}

// The requests, heads and window of a call; false where the heads are too many.
inline bool run_shape(RunArgs& a, int64_t requests, int64_t hq, int64_t hkv, int64_t page_size, int64_t num_pages,
                      int64_t table_width, int64_t table_stride, int64_t window) {
  a.table_stride = table_stride;
  a.shift = __builtin_ctzll(page_size); a.capacity = table_width << a.shift;
  a.requests = (int)requests; a.num_pages = (int)num_pages; a.hq = (int)hq; a.hkv = (int)hkv;
  a.window = (int)window;
  a.group = a.hq / a.hkv; a.row_tiles = (a.group + 15) / 16; a.rows = a.group < 16 ? a.group : 16;
  if ((int64_t)a.hkv * a.row_tiles > 65535) return false;
  a.units = a.hkv * a.row_tiles;
  return true;
}

// Where the join and the partials lie in the workspace.
inline void run_workspace(RunArgs& a, void* workspace, int64_t head_dim) {
  a.join = static_cast<int4*>(workspace);
  a.joins = reinterpret_cast<int*>(a.join + kMaxSlots);
  a.part = reinterpret_cast<float*>(a.join + kMaxSlots + 1);
  a.part_ml = a.part + (int64_t)kMaxSlots * a.rows * head_dim;
}

// Workgroups of a call: one for each (request, unit), and as many more as the splits make (plan_run).  Sets
// `direct`; `rounds`: the rounds of a request at most.
inline int64_t run_items(RunArgs& a, int64_t rounds) {
  const int64_t pairs = (int64_t)a.requests * a.units;
  a.direct = rounds <= a.whole;
  const int64_t most = pairs * ((rounds + kMinRun - 1) / kMinRun), some = pairs + a.runs + kSlack;
  return a.direct ? pairs : most < some ? most : some;
}

}  // namespace bfly
