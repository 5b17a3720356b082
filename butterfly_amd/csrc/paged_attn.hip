// One new token of every request over its pages (include/butterfly_amd_paged.h).
//
//   s_t = scale q . k_t for the positions t it sees, m = max s_t, l = sum exp(s_t - m),
//   o = (sum exp(s_t - m) v_t) / l, in one pass over the keys with a running m and l.
//
// Work: a request's tiles (32 keys in bf16, 16 in fp32) go in rounds of four, one for each wave of a
// workgroup, and its rounds in runs of at most c, c such that all requests and heads together make about
// 256 runs (512 of d 64).  A workgroup takes one run of one kv head for up to 16 of its query heads; every workgroup finds
// its run from the lengths by itself (plan_run), so the grid needs no host knowledge of them and a long request
// among short ones is split as far as a lone one.  Requests with one run write their output, the others a
// partial (fp32 sums, m, l) that paged_merge_kernel joins.
//
// A wave takes every fourth tile of the run, by itself: no barrier and no LDS until its sums meet the
// other waves'.  S^T = K Q^T and O^T += V^T P^T on the matrix cores (v_mfma_f32_16x16x32_bf16, or
// v_mfma_f32_16x16x4_f32), query heads as columns, so a lane's scores are the operand of the second product as
// they come:
//   * K rows go from memory into the first product's operand registers (lane = key, 16 bytes of d a load).
//   * V rows too (16 lanes take a row, a lane 4 (or 8) keys of one piece of d): the d of an output row is
//     chosen so that the operand is the lane's own words, which v_perm_b32 pairs up by key.
//   * The next tile's K is requested when this one's scores are done, its V after the second product: a wave
//     has 8 to 32 KB under way.
// Rows that hold no token the request sees (behind the last one, before the window) are read with their tile; their
// scores become -inf and their V zero, whatever they hold.
//
// Bound by HBM: keys and values are read once (2 group / size flops a byte for groups of `group` query heads over a kv
// head: 4 for groups of 4 in bf16, 2 in fp32, 1 without groups in bf16, 16 for groups of 16, against some 250 that the
// card's product and copy rates take).  Kernel times: 1.36 GB of 32 requests of up to 131072 tokens 207 us
// (6.6 TB/s; reading alone reaches 7.0 on this card), 262144 tokens of d 256 160 us (6.7); 32768 tokens of one
// request 16.0 us, of which some 3 us are four dependent reads (arguments, lengths, page, K) and the sums' way
// through LDS, and 3.9 us for the join.
//
// The schedule is every workgroup's own work over all lengths: hidden up to some hundreds of requests, and beyond as
// many passes as there are workgroups.  One request of 40000 tokens among requests of 100 (8/2 heads of 128), us: alone
// 17, 64 requests 20, 512 44, 4096 769, 16384 10248; 4096 and 16384 of 100 tokens over tables that hold no more
// (no schedule): 122, 479.  Batches beyond a thousand requests pass short contexts with the first columns of
// their table.
#include "paged.h"

namespace bfly {

constexpr float kPagedNeg = -1e30f;   // the largest score of a request without tokens
// Calls replayed from a graph, us, with 256 / 512 / 1024 runs (d 128 where nothing else stands): one request of 32768 tokens
// 19.1 / 19.7 / 23.6, 131072 tokens x 32 223 / 223 / 222, 262144 tokens of d 256 174 / 177 / 182, 64 of 4096 tokens with 32/8
// heads 174 / 173 / 180; fp32: 32768 tokens 30.9 / 31.8 / 35.9, 8 of 30000 160 / 164 / 165, 4 of 30000 of d 256 163 / 168 / 176.
// c at least 1 / 2: one request of 1024 tokens 9.6 / 11.3, four of up to 4096 in fp32 11.4 / 13.0.
// Two tiles of a wave under way instead of one: 131072 tokens x 32 223 -> 231, 64 of up to 2000 with 32/8 heads 37.9 -> 40.8,
// 262144 tokens of d 256 174 -> 367 (226 registers spill).
// Workgroups of 4 / 8 waves: 131072 tokens x 32 223 / 227, 64 of up to 2000 37.9 / 36.7, one of 1024 9.6 / 15.2, fp32 of d 256
// 164 / 207.
// Tiles of d 64 have half the bytes and half the registers: two runs a CU (512 / 256 runs: 8 requests of 60000 tokens
// 83.7 / 86.6, fp32 8 of 30000 85.4 / 90.4).
constexpr int runs_for(int head_dim) { return head_dim <= 64 ? 512 : 256; }   // in all, where requests and heads leave them
constexpr int kMaxRuns = 512;
constexpr int kMinRun = 1;            // c at least
// Rounds that stay one run, and without a second launch where the tables hold no more: 512 keys (bf16) are done before a
// join of two runs, and the more pairs of request and head (x16 query heads) there are, the longer runs hide behind each
// other.  Measured, half as many / this many / twice as many for all pairs, us: 128 pairs of 1000 tokens 19.8 / 18.0 /
// 18.1; 512 pairs of 2000 tokens 90.7 / 86.5 / 86.8, of up to 2000 (a mixed load) 37.8 / 45.1 / 45.1, of up to 4000
// 58.8 / 58.9 / 84.4, fp32 of up to 2000 62.7 / 62.7 / 98.1; 2048 pairs of up to 3000 164 / 146 (32 rounds either way
// for twice); one request of 1024 tokens 9.6 / 9.6 / 15.3.
// The pairs are the call's, idle requests among them: one request of 4000 tokens among 127 idle ones of 4 kv heads 13.7
// us, alone 10.7.
constexpr int whole_rounds(int64_t pairs) { return pairs >= 2048 ? 32 : pairs >= 512 ? 16 : pairs >= 128 ? 8 : 4; }
// A request of several runs has more than c rounds, so fewer than 2 rounds_b / c runs; all of them together, with
// c >= total / runs_for, fewer than twice runs_for: the partials there can be.  (kSlack: the total is a sum of floats.)
constexpr int kSlack = 64;
constexpr int kMaxSlots = 2 * kMaxRuns + kSlack;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
constexpr int kTile = sizeof(T) == 2 ? 32 : 16;
constexpr int kWaves = 4;             // waves of a workgroup, tiles of a round

typedef __attribute__((ext_vector_type(2))) float f32x2;

struct PagedAttnArgs {
  const char* q;
  PagePtr kp, vp;
  const int32_t* table;
  const int32_t* lengths;
  void* out;
  float* l;
  float* m;
  float* part;                           // partials: [slot][rows][D], then [slot][rows] m and l
  float* part_ml;
  int4* join;                            // what to join: request, unit, runs, first slot
  int* joins;                            // how many of them
  int64_t q_req, q_head, table_stride;   // bytes, bytes, elements
  int64_t capacity;                      // tokens a table row holds
  int requests, num_pages, hq, hkv, shift, window;
  int group, row_tiles, rows;            // query heads a kv head; 16-row parts of them; rows of a part at most
  int units;                             // hkv * row_tiles
  int runs;                              // runs_for(D)
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
__device__ __forceinline__ Span span_of(const PagedAttnArgs& a, int len) {
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

// The request that item `idx` falls into, where request b has units * splits_b items.  Every wave does it by
// itself: a lane sums a stretch of requests, one scan over the lanes, then the lane of the item walks its stretch.
template <int KT>
__device__ __forceinline__ Run plan_run(const PagedAttnArgs& a, int64_t idx) {
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
  // c fills the runs exactly if the requests' last, shorter runs fit among them; else room is left for one each
  const auto over = [&](float to) { return fminf(fmaxf(ceilf(total / to), (float)kMinRun), 1e9f); };
  int c = __builtin_amdgcn_readfirstlane((int)over((float)a.runs));
  const auto runs = [&](int n) { return n > c && n > a.whole ? (int)(((unsigned)n + c - 1) / (unsigned)c) : 1; };
  int items = 0;
  each([&](int n) { items += runs(n); });
  const int64_t pairs = (int64_t)a.requests * a.units;
  if ((int64_t)__builtin_amdgcn_readlane(wave_scan(items), 63) * a.units > a.runs && pairs < a.runs)
    c = __builtin_amdgcn_readfirstlane((int)over((float)(pairs < a.runs / 2 ? a.runs - (int)pairs : a.runs / 2)));
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
__device__ __forceinline__ void finish_stats(const PagedAttnArgs& a, int64_t row, float m, float l) {
  if (a.l == nullptr) return;
  const bool nan = l != l;
  a.l[row] = m == -INFINITY ? __builtin_nanf("") : l;
  a.m[row] = nan && m != INFINITY ? l : m;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
// The word without its bf16 infinities and NaN.
__device__ __forceinline__ uint32_t finite_bf16(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

// V rows are read once, whole lines an instruction, past the caches' replacement: the K half-lines of two
// neighbouring instructions then stay until both have been taken.  Measured, V past the caches / nothing / K and V,
// us: 131072 tokens x 32 223 / 246 / 241, 262144 tokens of d 256 174 / 191 / 172, 64 requests of 4096 tokens 174 / 192 /
// 175, one of 1024 (in the caches) 9.6 / 9.3 / 10.2.
template <typename V>
__device__ __forceinline__ V stream_load(const char* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}

// One wave's sums over its tiles.  acc[i][r] of lane (n = lane & 15, g = lane >> 4): query row n, element
// d_of(i, g, r).
template <typename T, int D>
struct Sweep;

template <int D>
struct Sweep<__bf16, D> {
  static constexpr int KT = 32;
  static constexpr int S = D / 32;                  // K pieces a subtile (and lane)
  static constexpr int W = D == 64 ? 2 : 4;         // words of a V piece
  static constexpr int H = D / (32 * W);            // V pieces a row (and lane): 1, or 2 for 256
  static constexpr int N = D / 16;                  // products a tile, accumulators a lane
  f32x4 acc[N];
  float m, l;                                       // l: this lane's keys only
  u32x4 q[S];
  u32x4 k[2][S];
  uint32_t v[8][H][W];

  // element of acc[i][r]
  static __device__ __forceinline__ int d_of(int i, int g, int r) {
    return (i / (2 * W)) * (32 * W) + (2 * W) * (4 * g + r) + i % (2 * W);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ void load_q(const char* row, int g) {
#pragma unroll
    for (int s = 0; s < S; ++s)
      q[s] = row != nullptr ? *reinterpret_cast<const u32x4*>(row + 64 * s + 16 * g) : u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void load_k(const char* const (&base)[2], int row_bytes, int n, int g) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < S; ++s)
        k[u][s] = *reinterpret_cast<const u32x4*>(base[u] + (uint32_t)(n * row_bytes + 16 * g) + 64 * s);
  }
  __device__ __forceinline__ void load_v(const char* const (&base)[2], int row_bytes, int n, int g) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const char* p = base[j >> 2] + (uint32_t)((4 * g + (j & 3)) * row_bytes + 4 * W * n) + 256 * h;
        if constexpr (W == 4) {
          const u32x4 x = stream_load<u32x4>(p);
#pragma unroll
          for (int w = 0; w < 4; ++w) v[j][h][w] = x[w];
        } else {
          const u32x2 x = stream_load<u32x2>(p);
          v[j][h][0] = x[0];
          v[j][h][1] = x[1];
        }
      }
  }
  __device__ __forceinline__ void scores(float (&s)[8], float scale) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < S; ++i)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[u][i]), __builtin_bit_cast(bf16x8, q[i]), c,
                                                    0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * u + i] = c[i] * scale;
    }
  }
  static __device__ __forceinline__ int key(int i, int g) { return 16 * (i >> 2) + 4 * g + (i & 3); }
  __device__ __forceinline__ void drop_v(int j) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int w = 0; w < W; ++w) v[j][h][w] = 0;
  }
  // The weights enter as two bf16 parts, 16 bits of them: with one part (8 bits) a weight would be off by
  // as much as the output's own rounding, and the second part hides behind the loads (131072 tokens x 32: 223 us
  // with it, 222 without).  kSafe: the second part skips V's infinities and NaN, which the
  // first one has carried into the sums already (p * inf is inf, but the rest of p may be 0).
  template <bool kSafe>
  __device__ __forceinline__ void add(const float (&p)[8]) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = pack_bf16(p[2 * i], p[2 * i + 1]);
      lo[i] = pack_bf16(p[2 * i] - __uint_as_float(hi[i] << 16), p[2 * i + 1] - __uint_as_float(hi[i] & 0xffff0000u));
    }
    const bf16x8 ph = __builtin_bit_cast(bf16x8, u32x4{hi[0], hi[1], hi[2], hi[3]});
    const bf16x8 pl = __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], lo[2], lo[3]});
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int h = i / (2 * W), e = i % (2 * W), w = e >> 1;
      const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
      u32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __builtin_amdgcn_perm(v[2 * j + 1][h][w], v[2 * j][h][w], sel);
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), ph, acc[i], 0, 0, 0);
      if constexpr (kSafe) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = finite_bf16(x[j]);
      }
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), pl, acc[i], 0, 0, 0);
    }
  }
};

template <int D>
struct Sweep<float, D> {
  static constexpr int KT = 16;
  static constexpr int S = D / 16;                  // K pieces a key (and lane)
  static constexpr int H = D / 64;                  // V pieces a row (and lane)
  static constexpr int N = D / 16;
  f32x4 acc[N];
  float m, l;
  f32x4 q[S];
  f32x4 k[S];
  f32x4 v[4][H];

  static __device__ __forceinline__ int d_of(int i, int g, int r) { return (i >> 2) * 64 + 4 * (4 * g + r) + (i & 3); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ void load_q(const char* row, int g) {
#pragma unroll
    for (int s = 0; s < S; ++s)
      q[s] = row != nullptr ? *reinterpret_cast<const f32x4*>(row + 64 * s + 16 * g) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void load_k(const char* const (&base)[1], int row_bytes, int n, int g) {
#pragma unroll
    for (int s = 0; s < S; ++s)
      k[s] = *reinterpret_cast<const f32x4*>(base[0] + (uint32_t)(n * row_bytes + 16 * g) + 64 * s);
  }
  __device__ __forceinline__ void load_v(const char* const (&base)[1], int row_bytes, int n, int g) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int h = 0; h < H; ++h)
        v[j][h] = stream_load<f32x4>(base[0] + (uint32_t)((4 * g + j) * row_bytes + 16 * n) + 256 * h);
  }
  __device__ __forceinline__ void scores(float (&s)[4], float scale) const {
    f32x4 c[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i][e], q[i][e], c[e & 1], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = (c[0][i] + c[1][i]) * scale;
  }
  static __device__ __forceinline__ int key(int i, int g) { return 4 * g + i; }
  __device__ __forceinline__ void drop_v(int j) {
#pragma unroll
    for (int h = 0; h < H; ++h) v[j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  template <bool kSafe>
  __device__ __forceinline__ void add(const float (&p)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j][i >> 2][i & 3], p[j], acc[i], 0, 0, 0);
  }
};

// The pages of tile t: one base per 16 keys, with the page's and the rows' offsets.  Keys outside [lo, n)
// share the page of the nearest key inside, so no entry behind the last page (or before the window) is read.
template <int U>
__device__ __forceinline__ bool tile_pages(const PagedAttnArgs& a, const int32_t* row, int first, const Span& s, int (&id)[U]) {
  bool bad = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    unsigned t = (unsigned)first + 16 * u;
    t = t < (unsigned)s.lo ? s.lo : t > (unsigned)s.n - 1 ? s.n - 1 : t;
    id[u] = row[t >> a.shift];
    if ((unsigned)id[u] >= (unsigned)a.num_pages) {
      bad = true;
      id[u] = 0;
    }
  }
  return bad;
}
template <int U>
__device__ __forceinline__ void tile_base(const PagedAttnArgs& a, const PagePtr& p, int h, int first, const int (&id)[U],
                                          const char* (&base)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) base[u] = p.row(id[u], h, (first + 16 * u) & ((1 << a.shift) - 1));
}

// Tiles t, t + kWaves, ... below t_end.  Returns whether a page id was outside the pages.
template <typename T, int D, bool kSafe>
__device__ __forceinline__ bool sweep(const PagedAttnArgs& a, Sweep<T, D>& w, const int32_t* row, const Span& s, int kvh,
                                      int t, int t_end) {
  constexpr int KT = kTile<T>, U = KT / 16, P = KT / 4;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  w.clear();
  if (t >= t_end) return false;
  int id[U];
  const char* base[U];
  bool bad = tile_pages<U>(a, row, t * KT, s, id);
  tile_base<U>(a, a.kp, kvh, t * KT, id, base);
  w.load_k(base, a.kp.row_bytes, n, g);
  tile_base<U>(a, a.vp, kvh, t * KT, id, base);
  w.load_v(base, a.vp.row_bytes, n, g);
  while (true) {
    const int next = t + kWaves;
    const bool more = next < t_end;
    if (more) bad |= tile_pages<U>(a, row, next * KT, s, id);
    float p[P];
    w.scores(p, a.scale);
    if (more) {
      tile_base<U>(a, a.kp, kvh, next * KT, id, base);
      w.load_k(base, a.kp.row_bytes, n, g);
    }
    const unsigned first = (unsigned)t * KT, lo = s.lo, end = s.n;
    if (first < lo || first + KT > end) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const unsigned at = first + w.key(i, g);
        if (at < lo || at >= end) {
          p[i] = -INFINITY;
          w.drop_v(i);                              // V's piece i is of the same key as score i
        }
      }
    }
    float mx = p[0];
#pragma unroll
    for (int i = 1; i < P; ++i) mx = fmaxf(mx, p[i]);
    mx = col_max4(mx);
    if (__any(mx > w.m)) {
      const float nm = fmaxf(w.m, mx);
      const float f = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((w.m - nm) * kLog2e);
      w.l *= f;
#pragma unroll
      for (int i = 0; i < w.N; ++i) w.acc[i] *= f;
      w.m = nm;
    }
    const float ref = w.m == -INFINITY ? 0.f : w.m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      p[i] = __builtin_amdgcn_exp2f((p[i] - ref) * kLog2e);
      sum += p[i];
    }
    w.l += sum;
    w.template add<kSafe>(p);
    if (!more) return bad;
    tile_base<U>(a, a.vp, kvh, next * KT, id, base);
    w.load_v(base, a.vp.row_bytes, n, g);
    t = next;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(64 * kWaves) paged_attn_kernel(PagedAttnArgs a) {
  constexpr int KT = kTile<T>, LD = D + 4;
  __shared__ float so[kWaves][16 * LD];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ int sbad;
  const Run run = plan_run<KT>(a, blockIdx.x);
  if (run.b < 0) return;
  // (every store comes after the last page id is read: a store before would take those reads off the scalar cache
  // and into the order of the K and V loads, 131072 tokens x 32: 207 -> 280 us)
  const auto leave = [&]() {
    if (blockIdx.x == 0 && threadIdx.x == 0 && !a.direct) *a.joins = run.joins;
  };
  const int b = __builtin_amdgcn_readfirstlane(run.b), splits = __builtin_amdgcn_readfirstlane(run.splits);
  const int sub = __builtin_amdgcn_readfirstlane(run.sub), slot = __builtin_amdgcn_readfirstlane(run.slot) + sub;
  const int unit = sub / splits, split = sub - unit * splits;
  const int kvh = unit / a.row_tiles, part = unit - kvh * a.row_tiles;
  const int rows = a.group - 16 * part < 16 ? a.group - 16 * part : 16;
  const int head0 = kvh * a.group + 16 * part;
  const Span s = span_of<KT>(a, __builtin_amdgcn_readfirstlane(run.len));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)b * a.hq + head0;
  if (s.tiles == 0) {                               // nothing to see, or a length beyond the table
    leave();
    const float y = s.off ? __builtin_nanf("") : 0.f;
    for (int i = threadIdx.x; i < rows * D; i += 64 * kWaves) static_cast<T*>(a.out)[row0 * D + i] = from_f32<T>(y);
    if (a.l != nullptr && threadIdx.x < rows) {
      a.l[row0 + threadIdx.x] = y;
      a.m[row0 + threadIdx.x] = s.off ? y : kPagedNeg;
    }
    return;
  }
  const int each = s.rounds / splits, extra = s.rounds - each * splits;
  const int r0 = split * each + (split < extra ? split : extra), r1 = r0 + each + (split < extra ? 1 : 0);
  const int t0 = s.t0 + kWaves * r0, t1 = s.t0 + (kWaves * r1 < s.tiles ? kWaves * r1 : s.tiles);
  const int32_t* table = a.table + b * a.table_stride;
  if (threadIdx.x == 0) sbad = 0;
  Sweep<T, D> w;
  w.load_q(n < rows ? a.q + b * a.q_req + (int64_t)(head0 + n) * a.q_head : nullptr, g);
  bool bad = sweep<T, D, false>(a, w, table, s, kvh, t0 + wave, t1);
  if constexpr (sizeof(T) == 2) {
    // infinities or NaN in the sums of a row whose weights are finite come from V: once more, with care
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < w.N; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) big = fmaxf(big, w.acc[i][r] - w.acc[i][r] == 0.f ? 0.f : 1.f);
    if (__any(big != 0.f)) bad |= sweep<T, D, true>(a, w, table, s, kvh, t0 + wave, t1);
  }
  const float l = col_sum4(w.l);
  __syncthreads();
  if (n < rows) {
#pragma unroll
    for (int i = 0; i < w.N; i += 4)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(&so[wave][n * LD + w.d_of(i, g, r)]) =
            f32x4{w.acc[i][r], w.acc[i + 1][r], w.acc[i + 2][r], w.acc[i + 3][r]};
    if (g == 0) {
      sm[wave][n] = w.m;
      sl[wave][n] = l;
    }
  }
  if (bad && lane == 0) sbad = 1;
  __syncthreads();
  leave();
  if (splits > 1 && split == 0 && threadIdx.x == 0) a.join[run.join + unit] = int4{b, unit, splits, slot};
  const float poison = sbad ? __builtin_nanf("") : 0.f;
  for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * kWaves) {
    const int r = i / (D / 4), c = 4 * (i % (D / 4));
    float mm = sm[0][r];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) mm = fmaxf(mm, sm[k][r]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    float ll = poison;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float f = __builtin_amdgcn_exp2f((sm[k][r] - ref) * kLog2e);
      // a wave without tiles has no part in it (0 * its sums would do, but for a reference of +inf)
      if (t0 + k < t1) {
        ll += f * sl[k][r];
        y += f * *reinterpret_cast<const f32x4*>(&so[k][r * LD + c]);
      }
    }
    if (splits == 1) {
      store4(static_cast<T*>(a.out) + (row0 + r) * D + c, y, 1.f / ll);
      if (c == 0) finish_stats<T>(a, row0 + r, mm, ll);
    } else {
      const int64_t at = (int64_t)slot * a.rows + r;
      *reinterpret_cast<f32x4*>(a.part + at * D + c) = y;
      if (c == 0) {
        reinterpret_cast<f32x2*>(a.part_ml)[at] = f32x2{mm, ll};
      }
    }
  }
}

// Joins the partials of a request's runs: a workgroup per (request, unit, row, 64 elements) of the list that the runs
// have left.  The runs'
// weights exp(m_i - m) are made once, in LDS; then 16 lanes across the elements, the runs dealt to 16 groups
// of lanes, four loads under way in each.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedAttnArgs a) {
  constexpr int G = 16;
  __shared__ f32x4 sy[G][16];
  __shared__ float weight[kMaxSlots], sl[4], smx[4];
  const int joins = *a.joins;
  const int4 what = a.join[blockIdx.x];             // (what is there behind the last is not looked at)
  if ((int)blockIdx.x >= joins) return;
  const int unit = what.y, splits = what.z;
  const int kvh = unit / a.row_tiles, part = unit - kvh * a.row_tiles, r = blockIdx.y;
  if (16 * part + r >= a.group) return;
  const int64_t slot0 = what.w;
  const int t = threadIdx.x, gr = t >> 4, c = 64 * blockIdx.z + 4 * (t & 15);
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + slot0 * a.rows + r;
  const float* src = a.part + (slot0 * a.rows + r) * D + c;
  const int64_t step = (int64_t)a.rows * D;
  // the first partials are requested beside the maxima that weigh them
  constexpr int kAhead = 4;
  f32x4 ahead[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int i = gr + G * j;
    ahead[j] = i < splits ? *reinterpret_cast<const f32x4*>(src + i * step) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  f32x2 mine = {-INFINITY, 0.f};
  if (t < splits) mine = ml[(int64_t)t * a.rows];
  float mm = mine[0];
  for (int i = t + 256; i < splits; i += 256) mm = fmaxf(mm, ml[(int64_t)i * a.rows][0]);
  mm = wave_max(mm);
  if ((t & 63) == 0) smx[t >> 6] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(smx[0], smx[1]), fmaxf(smx[2], smx[3]));
  const float ref = mm == -INFINITY ? 0.f : mm;
  float l = 0.f;
  for (int i = t; i < splits; i += 256) {
    const f32x2 x = i == t ? mine : ml[(int64_t)i * a.rows];
    const float f = __builtin_amdgcn_exp2f((x[0] - ref) * kLog2e);
    weight[i] = f;
    l += f * x[1];
  }
  l = wave_total(l);
  if ((t & 63) == 0) sl[t >> 6] = l;
  __syncthreads();
  l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (gr + G * j < splits) y += weight[gr + G * j] * ahead[j];
#pragma unroll 4
  for (int i = gr + G * kAhead; i < splits; i += G) y += weight[i] * *reinterpret_cast<const f32x4*>(src + i * step);
  sy[gr][t & 15] = y;
  __syncthreads();
  if (gr != 0) return;
#pragma unroll
  for (int i = 1; i < G; ++i) y += sy[i][t];
  const int64_t row = (int64_t)what.x * a.hq + kvh * a.group + 16 * part + r;
  store4(static_cast<T*>(a.out) + row * D + c, y, 1.f / l);
  if (c == 0) finish_stats<T>(a, row, mm, l);
}

// The rounds of a request at most; only one of more than whole_rounds can have several runs.
static int64_t most_rounds(int64_t capacity, int window, int esize) {
  const int kt = esize == 2 ? kTile<__bf16> : kTile<float>;
  const int64_t keys = window > 0 && window < capacity ? (int64_t)window + kt - 1 : capacity;
  return (keys + kWaves * kt - 1) / (kWaves * kt);
}
template <typename T, int D>
static void launch_paged(const PagedAttnArgs& a, int64_t items, bool splits, hipStream_t stream) {
  hipLaunchKernelGGL((paged_attn_kernel<T, D>), dim3((unsigned)items), dim3(64 * kWaves), 0, stream, a);
  if (splits) {
    const int64_t pairs = (int64_t)a.requests * a.units;
    const unsigned x = (unsigned)(pairs < a.runs ? pairs : a.runs);
    hipLaunchKernelGGL((paged_merge_kernel<T, D>), dim3(x, (unsigned)a.rows, D / 64), dim3(256), 0, stream, a);
  }
}

}  // namespace bfly

using namespace bfly;

extern "C" int64_t bfly_paged_attention_workspace_bytes(int dtype, int64_t requests, int hq, int hkv, int head_dim,
                                                        int64_t table_width, int page_size, int window) {
  if (requests <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || head_dim <= 0 || table_width <= 0 || page_size <= 0) return 0;
  const int64_t group = hq / hkv, rows = group < 16 ? group : 16;
  const int64_t pairs = requests * hkv * ((group + 15) / 16);
  if (most_rounds(table_width * page_size, window, dtype == BFLY_DTYPE_F32 ? 4 : 2) <= whole_rounds(pairs)) return 0;
  return (int64_t)kMaxSlots * (rows * (head_dim + 2) * 4 + 16) + 16;
}

extern "C" int bfly_paged_attention(const bfly_paged_attention_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_attention_args_t& x = *args;
  BFLY_CHECK_ARG(x.dtype == BFLY_DTYPE_F32 || x.dtype == BFLY_DTYPE_BF16, "unsupported dtype %lld", (long long)x.dtype);
  const int64_t es = x.dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(x.requests >= 0 && x.requests <= 65535, "bad number of requests (at most 65535)");
  BFLY_CHECK_ARG(x.hkv > 0 && x.hq > 0 && x.hq <= (1 << 20) && x.hkv <= x.hq && x.hq % x.hkv == 0,
                 "bad head counts hq=%lld hkv=%lld", (long long)x.hq, (long long)x.hkv);
  if (x.head_dim != 64 && x.head_dim != 128 && x.head_dim != 256) {
    set_error("bfly_paged_attention: head_dim=%lld unsupported (64, 128, 256)", (long long)x.head_dim);
    return BFLY_ERR_UNSUPPORTED;
  }
  const int rc = paged_check_pages("bfly_paged_attention", x.pages, es);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(x.window >= 0 && x.window <= INT32_MAX, "bad window");
  BFLY_CHECK_ARG(x.table_width >= 0 && x.table_width <= INT32_MAX && (x.requests <= 1 || x.table_stride >= 0),
                 "bad block table shape");
  BFLY_CHECK_ARG(x.q_request_stride >= 0 && x.q_head_stride >= 0 && x.q_request_stride < ((int64_t)1 << 48) &&
                     x.q_head_stride < ((int64_t)1 << 48) && x.q_request_stride * es % 16 == 0 &&
                     x.q_head_stride * es % 16 == 0,
                 "q strides must be multiples of 16 bytes");
  if (x.requests == 0) return BFLY_OK;
  BFLY_CHECK_ARG(x.q && x.pages.k && x.pages.v && x.lengths && x.out, "null pointer");
  BFLY_CHECK_ARG(x.table_width == 0 || x.block_table, "null pointer");
  BFLY_CHECK_ARG((x.l == nullptr) == (x.m == nullptr), "both l and m or neither");
  BFLY_CHECK_ARG(aligned16(x.q) && aligned16(x.pages.k) && aligned16(x.pages.v) && aligned16(x.out),
                 "pointers must be 16-byte aligned");
  const int64_t need = bfly_paged_attention_workspace_bytes((int)x.dtype, x.requests, (int)x.hq, (int)x.hkv, (int)x.head_dim,
                                                            x.table_width, (int)x.pages.page_size, (int)x.window);
  BFLY_CHECK_ARG(need == 0 || (x.workspace && x.workspace_bytes >= need && aligned16(x.workspace)), "workspace too small");
  PagedAttnArgs a{};
  a.q = static_cast<const char*>(x.q);
  a.kp = k_page_ptr(x.pages, es); a.vp = v_page_ptr(x.pages, es);
  a.table = x.block_table; a.lengths = x.lengths; a.out = x.out; a.l = x.l; a.m = x.m;
  a.q_req = x.q_request_stride * es; a.q_head = x.q_head_stride * es; a.table_stride = x.table_stride;
  a.shift = __builtin_ctzll(x.pages.page_size); a.capacity = x.table_width << a.shift;
  a.requests = (int)x.requests; a.num_pages = (int)x.pages.num_pages; a.hq = (int)x.hq; a.hkv = (int)x.hkv;
  a.window = (int)x.window; a.scale = (float)x.scale;
  a.group = a.hq / a.hkv; a.row_tiles = (a.group + 15) / 16; a.rows = a.group < 16 ? a.group : 16;
  BFLY_CHECK_ARG((int64_t)a.hkv * a.row_tiles <= 65535, "too many heads");
  a.units = a.hkv * a.row_tiles;
  a.join = static_cast<int4*>(x.workspace);
  a.joins = reinterpret_cast<int*>(a.join + kMaxSlots);
  a.part = reinterpret_cast<float*>(a.join + kMaxSlots + 1);
  a.part_ml = a.part + (int64_t)kMaxSlots * a.rows * x.head_dim;
  // runs: one for each (request, unit), and as many more as the splits make (plan_run)
  const int64_t rounds = most_rounds(a.capacity, a.window, (int)es), pairs = x.requests * a.units;
  a.runs = runs_for((int)x.head_dim);
  a.whole = whole_rounds(pairs);
  const bool splits = rounds > a.whole;
  a.direct = !splits;
  const int64_t most = pairs * ((rounds + kMinRun - 1) / kMinRun), some = pairs + a.runs + kSlack;
  const int64_t items = !splits ? pairs : most < some ? most : some;
  BFLY_CHECK_ARG(items < (1 << 24), "too many requests and heads");   // a grid holds fewer than 2^32 threads
#define BFLY_PAGED(T, D) launch_paged<T, D>(a, items, splits, stream)
  if (x.dtype == BFLY_DTYPE_BF16) {
    if (x.head_dim == 64) BFLY_PAGED(__bf16, 64);
    else if (x.head_dim == 128) BFLY_PAGED(__bf16, 128);
    else BFLY_PAGED(__bf16, 256);
  } else {
    if (x.head_dim == 64) BFLY_PAGED(float, 64);
    else if (x.head_dim == 128) BFLY_PAGED(float, 128);
    else BFLY_PAGED(float, 256);
  }
#undef BFLY_PAGED
  BFLY_CHECK_LAUNCH("bfly_paged_attention");
  return BFLY_OK;
}
