// Log probabilities of given tokens, entropy and the top alternatives, from rows of logits
// (bfly_token_logprobs, include/butterfly_amd_decoder.h).
//
//   m = max x, l = sum exp(x - m), s = sum exp(x - m) (x - m):
//   log p(token) = (x_token - m) - log l,   H = log l - s / l,   in one pass with a running m, l and s.
//
// A workgroup takes a row, or (few rows) one of up to 32 parts of a row, in rounds of 64 bytes a thread; a second
// launch joins the parts.  Every thread keeps a reference and sums of its own until the end.  The reference is the
// maximum's whole number of powers of two, r: exp(x - m) counts 2^(x log2 e - r), whose exponent is one fused
// operation and exact up to its one rounding (the constant's own error is common to all terms).
//
// Bound by HBM where there are rows for the card: 2048 of 151936 bf16 (623 MB) 122 us without a top (5.1 TB/s), 133 with the top 20;
// a single such row, top 5, takes 12 us, two launches of 7 and 5.
//
// The top k: the pass leaves each thread's maximum of each round (a segment's) in LDS.  A bound that k threads' maxima reach
// (k / 4 of each wave) is one that the top k reach, so these lie in the segments that do: some k of them, whose elements are
// read once more, one a thread.  Those from the bound on go as 64-bit keys (value's order, then the lower index;
// argmax_key, so all differ) to a list, and a count of larger keys orders it.  Where ties make the list too long, the
// segments go through a bound of whole keys instead (top_by_keys).  This part is loops of few instructions: a row's
// workgroup runs through it once, and unrolled it was bound by fetching them (32 rows of 32003 fp32, top 50: 17 us).
#include "argmax.h"

#include "../../include/butterfly_amd_decoder.h"

namespace bfly {

template <typename T>
constexpr int kLpEach = 64 / sizeof(T);             // elements of a thread in a round
// Threads of a workgroup: one wave for rows of one round of it (4096 rows of 100 bf16: 9.6 us, with four 43; 16384 of 2048 27, 77).
constexpr int kLpWhole = 256, kLpShort = 64;
constexpr int kLpTop = 64;                          // top at most
constexpr int kLpParts = 32;                        // parts of a row at most
constexpr int kLpSlots = 32;                        // rounds whose maxima are kept apart
constexpr int kLpSegments = 512;                    // segments gathered at a time
constexpr float kLpLog2e = 1.4426950408889634f, kLpLn2 = 0.6931471805599453f;
constexpr float kLpFar = -1e30f;                    // below every difference that counts, and finite
constexpr float kLpWide = 1048576.f;                // maxima whose powers of two are whole numbers in fp32

struct LogprobArgs {
  const char* logits;
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int64_t* top_token;
  f32x4* sums;                            // [rows][parts]: m, l, s
  uint64_t* keys;                         // [rows][parts][top]
  int64_t stride;                         // bytes between rows
  int64_t rows;
  int vocab, top, parts, per;             // per: 16-byte vectors of a part
  int slots, fold;                        // kept maxima a thread; rounds of each
};

// --------------------------------------------------------------------------- sums
struct Sums {                                       // relative to m, in nats
  float m, l, s;
  __device__ __forceinline__ void to(float nm) {    // the sums with another maximum (nm >= m)
    const float d = fmaxf(m - nm, kLpFar), f = __builtin_amdgcn_exp2f(d * kLpLog2e);
    s = f * fmaf(l, d, s);
    l *= f;
    m = nm;
  }
  __device__ __forceinline__ void add(Sums o) {
    const float nm = fmaxf(m, o.m);
    to(nm);
    o.to(nm);
    l += o.l;
    s += o.s;
  }
};

// A thread's: l and s (in powers of two) relative to 2^r, or, where the maximum is too large for that (or -inf), to m.
struct Running {
  float m = -INFINITY, r = 0.f, l = 0.f, s = 0.f;
  bool wide = true;
  __device__ __forceinline__ void shift(float d) {  // the sums with a reference of 2^d of the present one
    const float f = __builtin_amdgcn_exp2f(d);
    s = f * fmaf(l, d, s);
    l *= f;
  }
  __device__ __forceinline__ float beyond() const { return wide ? 0.f : fmaf(-m, kLpLog2e, r); }   // r - m log2 e
  __device__ __forceinline__ void refer(float nm) {
    const bool nw = !(fabsf(nm) <= kLpWide);
    const float nr = nw ? 0.f : rintf(nm * kLpLog2e);
    if (nw || wide || nr != r) {
      const float d = beyond() + fmaxf(m - nm, kLpFar) * kLpLog2e - (nw ? 0.f : fmaf(-nm, kLpLog2e, nr));
      shift(d);
    }
    m = nm;
    r = nr;
    wide = nw;
  }
  __device__ __forceinline__ Sums settled() {
    shift(beyond());
    return Sums{m, l, s * kLpLn2};
  }
};

template <int kThreads>
__device__ __forceinline__ Sums block_sums(f32x4* shared, Sums v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v.add(Sums{__shfl_xor(v.m, o), __shfl_xor(v.l, o), __shfl_xor(v.s, o)});
  if constexpr (kThreads == 64) return v;
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = f32x4{v.m, v.l, v.s, 0.f};
  __syncthreads();
  v = Sums{shared[0][0], shared[0][1], shared[0][2]};
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v.add(Sums{shared[w][0], shared[w][1], shared[w][2]});
  return v;
}

// --------------------------------------------------------------------------- the list of keys
// LDS of the top k: sizes by k, so that small ones leave room for more workgroups.
struct TopLds {
  uint64_t* list;                         // [33 k]: k kept and k threads' 32
  uint64_t* few;                          // [few_for(k)]
  uint64_t* most;                         // [kLpThreads]
  uint64_t* bound;
  int* count;                             // of the list
  int* kept;
  int* segments;                          // how many
  uint16_t* segment;                      // [kLpSegments]
  char* ranks;                            // [slots][kLpThreads]
  uint32_t* wave;                         // [4]
  int room, few_room;
  // (k kept and k threads' 32; a few more for the quick way)
  static __host__ __device__ int room_for(int k) { return 33 * k > 256 ? 33 * k : 256; }
  static __host__ __device__ int few_for(int k, int threads) {
    const int most = k * ((room_for(k) + threads - 1) / threads);
    return most > threads ? most : threads;
  }
  static __host__ __device__ int bytes(int k, int threads, int slots, int esize) {
    return 8 * (room_for(k) + few_for(k, threads) + threads + 1) + 4 * 10 + 2 * kLpSegments + slots * threads * esize;
  }
  __device__ __forceinline__ TopLds(char* p, int k, int threads) {
    room = room_for(k);
    few_room = few_for(k, threads);
    list = reinterpret_cast<uint64_t*>(p);
    few = list + room;
    most = few + few_for(k, threads);
    bound = most + threads;
    count = reinterpret_cast<int*>(bound + 1);
    kept = count + 1;
    segments = count + 2;
    wave = reinterpret_cast<uint32_t*>(count + 4);
    segment = reinterpret_cast<uint16_t*>(count + 10);
    ranks = reinterpret_cast<char*>(segment + kLpSegments);
  }
};

// A rank that at least k threads' ranks reach, 0 where they do not (but for the last 6 bits: up to 63 below such a rank).
template <int kThreads>
__device__ __forceinline__ uint32_t rank_bound(const TopLds& sh, uint32_t rank, int k) {
  const int lane = threadIdx.x & 63;
  const auto max_of_wave = [](uint32_t x) {
    const auto step = [](uint32_t v, uint32_t w) { return w > v ? w : v; };
    x = step(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));   // row_shr:1, 2, 4, 8
    x = step(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
    x = step(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
    x = step(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
    x = step(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));   // row_bcast:15, 31
    x = step(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
  };
  uint32_t key = (rank & ~63u) | (63 - lane), last = 0;
  for (int j = (k * 64 + kThreads - 1) / kThreads; j > 0; --j) {
    last = max_of_wave(key);
    if (key == last) key = 0;
  }
  last &= ~63u;
  if constexpr (kThreads > 64) {
    __syncthreads();
    if (lane == 0) sh.wave[threadIdx.x >> 6] = last;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) last = sh.wave[w] < last ? sh.wave[w] : last;
  }
  return last;
}

// The k-th largest of the threads' keys, 0 where fewer than k are above 0 (those differ).
template <int kThreads>
__device__ __forceinline__ uint64_t kth_of_threads(const TopLds& sh, uint64_t mine, int k) {
  const int t = threadIdx.x;
  __syncthreads();
  sh.most[t] = mine;
  if (t == 0) *sh.bound = 0;
  __syncthreads();
  int above = 0;
  if (mine != 0) {
#pragma unroll 8
    for (int j = 0; j < kThreads; ++j) above += sh.most[j] > mine;
    if (above == k - 1) *sh.bound = mine;
  }
  __syncthreads();
  return *sh.bound;
}

// The list's n keys to its k largest in order (0 behind the last).
template <int kThreads>
__device__ __forceinline__ void cut_list(const TopLds& sh, int n, int k) {
  const int t = threadIdx.x;
  const auto gather = [&](uint64_t from) {          // keys from there on to `few`; how many there are
    __syncthreads();
    if (t == 0) *sh.kept = 0;
    __syncthreads();
    for (int i = t; i < n; i += kThreads) {
      const uint64_t x = sh.list[i];
      if (x >= from && x != 0) {
        const int at = atomicAdd(sh.kept, 1);
        if (at < sh.few_room) sh.few[at] = x;
      }
    }
    __syncthreads();
    return *sh.kept;
  };
  uint64_t mine = 0;
  for (int i = t; i < n; i += kThreads) mine = sh.list[i] > mine ? sh.list[i] : mine;
  int kept = gather((uint64_t)rank_bound<kThreads>(sh, (uint32_t)(mine >> 32), k) << 32);
  // (many of one value: by whole keys, k threads' at most)
  if (kept > sh.few_room) kept = gather(kth_of_threads<kThreads>(sh, mine, k));
  if (t == 0) *sh.count = kept < k ? kept : k;
  for (int i = t; i < k; i += kThreads)
    if (i >= kept) sh.list[i] = 0;
  for (int i = t; i < kept; i += kThreads) {
    const uint64_t x = sh.few[i];
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < kept; ++j) above += sh.few[j] > x;
    if (above < k) sh.list[above] = x;
  }
  __syncthreads();
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  if (u == 0xFFFFFFFFu) return __builtin_nanf("");
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
// A value's order alone (argmax_key's upper half); in bf16 its upper 16 bits tell all.
__device__ __forceinline__ uint32_t rank_of(float v) { return (uint32_t)(argmax_key(v, 0) >> 32); }
template <typename T>
struct RankOf {
  typedef uint32_t type;
  static __device__ __forceinline__ uint32_t pack(uint32_t r) { return r; }
};
template <>
struct RankOf<__bf16> {
  typedef uint16_t type;
  static __device__ __forceinline__ uint16_t pack(uint32_t r) { return (uint16_t)(r >> 16); }
};

// A row's results from its sums and its list (in order).
template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs& a, const uint64_t* list, int64_t row, const Sums& v) {
  const float log_l = logf(v.l);
  const int t = threadIdx.x;
  if (t == 0) {
    const int64_t tok = a.tokens[row];
    float y = __builtin_nanf("");
    if (tok >= 0 && tok < a.vocab) y = to_f32(reinterpret_cast<const T*>(a.logits + row * a.stride)[tok]) - v.m - log_l;
    a.logprob[row] = y;
    a.entropy[row] = log_l - v.s / v.l;
  }
  if (t < a.top) {
    const uint64_t key = list[t];
    a.top_logprob[row * a.top + t] = key_value(key) - v.m - log_l;
    a.top_token[row * a.top + t] = argmax_key_index(key);
  }
}

// A row's (or part's) 16-byte vectors: they lie at whole 16 bytes, so `skew` elements of the first are before the row.
template <typename T, int kThreads>
struct RowOf {
  static constexpr int VE = 16 / sizeof(T), NV = kLpEach<T> / VE;   // elements of a vector, vectors of a thread in a round
  static constexpr int kRound = kThreads * NV;
  typedef T Vec __attribute__((ext_vector_type(VE)));
  const T* x;
  int skew, vocab, v0, v1;
  bool stream;                                      // long: past the caches' replacement (short ones are read again there)
  __device__ __forceinline__ RowOf(const LogprobArgs& a, int64_t row, int part) {
    x = reinterpret_cast<const T*>(a.logits + row * a.stride);
    skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    vocab = a.vocab;
    const int vectors = (int)(((int64_t)a.vocab + skew + VE - 1) / VE);
    v0 = part * a.per < vectors ? part * a.per : vectors;
    v1 = v0 + a.per < vectors ? v0 + a.per : vectors;
    // (2048 rows of 151936 bf16, top 5: 123 us, through the caches 134; 8192 of 5000 fp32: 53, past them 58)
    stream = a.per > 4 * kRound;
  }
  // Element i of thread t's in the round at vector `base`; whether it is one.
  __device__ __forceinline__ int at(int base, int t, int i) const { return (base + t + kThreads * (i / VE)) * VE - skew + i % VE; }
  __device__ __forceinline__ bool holds(int base, int t, int i) const {
    const int p = at(base, t, i);
    return base + t + kThreads * (i / VE) < v1 && p >= 0 && p < vocab;
  }
  // thread t's of the round at vector `base`; -inf outside
  __device__ __forceinline__ void load(Vec (&y)[NV], int base, int t) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = base + t + kThreads * i, p = v * VE - skew;
      if (v < v1 && p >= 0 && p + VE <= vocab) {
        const Vec* q = reinterpret_cast<const Vec*>(x + p);
        if (stream) {
          y[i] = __builtin_nontemporal_load(q);
        } else {
          asm("" : "+v"(q));                        // (else both loads become one, of the second kind)
          y[i] = *q;
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) y[i][e] = v < v1 && p + e >= 0 && p + e < vocab ? x[p + e] : (T)-INFINITY;
      }
    }
  }
};

// f(key, index) of every element of `segments` listed segments (slot and thread), dealt to the threads one by one.
template <typename T, int kThreads, typename F>
__device__ __forceinline__ void each_element(const TopLds& sh, const RowOf<T, kThreads>& in, int segments, int fold, int f, F&& g) {
  for (int q = threadIdx.x; q < segments * kLpEach<T>; q += kThreads) {
    const int id = sh.segment[q / kLpEach<T>], tt = id % kThreads, i = q % kLpEach<T>;
    const int base = in.v0 + (id / kThreads * fold + f) * in.kRound;
    if (in.holds(base, tt, i)) g(to_f32(in.x[in.at(base, tt, i)]), in.at(base, tt, i));
  }
}

// The top k of segments whose maxima reach rank `from`, whatever ties there are: slot by slot, through a bound of whole
// keys that at most a round's elements of k threads pass.
template <typename T, int kThreads>
__device__ __forceinline__ void top_by_keys(const LogprobArgs& a, const TopLds& sh, const RowOf<T, kThreads>& in, uint32_t from32,
                                            int slots) {
  typedef typename RankOf<T>::type Rank;
  const Rank* ranks = reinterpret_cast<const Rank*>(sh.ranks);
  const int t = threadIdx.x;
  const Rank from = RankOf<T>::pack(from32);
  uint64_t bound = 0;                               // keys above it count
  __syncthreads();
  if (t == 0) *sh.count = 0;
  for (int slot = 0; slot < slots; ++slot) {
    __syncthreads();
    if (t == 0) *sh.segments = 0;
    __syncthreads();
    // (indices grow with the slot, so a segment below the bound's value, or of it behind the bound's index, is done)
    const Rank rank = ranks[slot * kThreads + t], have = RankOf<T>::pack((uint32_t)(bound >> 32));
    const int first = in.at(in.v0 + slot * a.fold * in.kRound, 0, 0);
    if (rank >= from && (rank > have || (rank == have && (first < 0 || (uint32_t)first < 0xFFFFFFFFu - (uint32_t)bound))))
      sh.segment[atomicAdd(sh.segments, 1)] = (uint16_t)(slot * kThreads + t);
    __syncthreads();
    const int segments = *sh.segments;
    for (int f = 0; segments > 0 && f < a.fold; ++f) {
      uint64_t best = 0;
      each_element<T, kThreads>(sh, in, segments, a.fold, f, [&](float v, int at) {
        const uint64_t key = argmax_key(v, (uint32_t)at);
        if (key > bound && key > best) best = key;
      });
      const uint64_t reach = kth_of_threads<kThreads>(sh, best, a.top);
      if (reach > bound) bound = reach - 1;
      each_element<T, kThreads>(sh, in, segments, a.fold, f, [&](float v, int at) {
        const uint64_t key = argmax_key(v, (uint32_t)at);
        if (key > bound) sh.list[atomicAdd(sh.count, 1)] = key;   // k kept, and k threads' elements of a round
      });
      __syncthreads();
      cut_list<kThreads>(sh, *sh.count, a.top);
      if (*sh.count == a.top) bound = sh.list[a.top - 1];
    }
  }
}

template <typename T, bool kTop, int kThreads>
__global__ void __launch_bounds__(kThreads, 4) logprob_kernel(LogprobArgs a) {
  typedef RowOf<T, kThreads> Row;
  typedef typename RankOf<T>::type Rank;
  extern __shared__ __align__(16) char lds[];
  __shared__ f32x4 shared[kThreads / 64];
  const TopLds sh(lds, a.top, kThreads);
  Rank* ranks = reinterpret_cast<Rank*>(sh.ranks);
  const int t = threadIdx.x;
  const int64_t row = (int64_t)(blockIdx.x / (unsigned)a.parts);
  const int part = (int)(blockIdx.x % (unsigned)a.parts);
  const Row in(a, row, part);
  constexpr int kRound = Row::kRound;
  Running sum;
  typename Row::Vec next[Row::NV];
  in.load(next, in.v0, t);
  if (kTop && t == 0) {
    *sh.count = 0;
    *sh.segments = 0;
  }
  uint32_t most = 0, all = 0;                       // ranks: of the slot's rounds so far, of all
  int slot = 0, round = 0;
  for (int base = in.v0; base < in.v1; base += kRound) {
    float x[kLpEach<T>];
#pragma unroll
    for (int i = 0; i < kLpEach<T>; ++i) x[i] = to_f32(next[i / Row::VE][i % Row::VE]);
    if (base + kRound < in.v1) in.load(next, base + kRound, t);
    // (vectors that no thread has are left out: a last round, a short row)
    const auto vectors = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < Row::NV; ++i)
        if (i == 0 || base + kThreads * i < in.v1) {
#pragma unroll
          for (int e = 0; e < Row::VE; ++e) f(x[Row::VE * i + e], e & 1);
        }
    };
    float mx = x[0];
    vectors([&](float v, int) __attribute__((always_inline)) { mx = fmaxf(mx, v); });
    if (mx > sum.m) sum.refer(mx);
    if (sum.wide && sum.m != -INFINITY) {
#pragma unroll
      for (int i = 0; i < kLpEach<T>; ++i) x[i] -= sum.m;
    }
    float l[2] = {0.f, 0.f}, s[2] = {0.f, 0.f};
    vectors([&](float v, int p) __attribute__((always_inline)) {
      const float z = fmaf(v, kLpLog2e, -sum.r), e = __builtin_amdgcn_exp2f(z);
      l[p] += e;
      s[p] = fmaf(e, fmaxf(z, kLpFar), s[p]);
    });
    const float added = l[0] + l[1];
    sum.l += added;
    sum.s += s[0] + s[1];
    if constexpr (kTop) {
      uint32_t rank = rank_of(mx);
      if (added != added) {                         // (an infinity, or a NaN, which is above)
        typename Row::Vec y[Row::NV];
        in.load(y, base, t);
#pragma unroll
        for (int i = 0; i < kLpEach<T>; ++i) {
          const float v = to_f32(y[i / Row::VE][i % Row::VE]);
          if (v != v) rank = 0xFFFFFFFFu;
        }
      }
      most = rank > most ? rank : most;
      all = rank > all ? rank : all;
      if (++round == a.fold || base + kRound >= in.v1) {
        ranks[slot * kThreads + t] = RankOf<T>::pack(most);
        ++slot;
        round = 0;
        most = 0;
      }
    }
  }
  if constexpr (kTop) {
    __syncthreads();
    constexpr uint32_t kNone = 0x007FFFFFu;         // the rank of -inf
    uint32_t from = in.v0 < in.v1 ? rank_bound<kThreads>(sh, all, a.top) : 0xFFFFFFFFu;
    if (from <= kNone)                              // (mostly -inf: the exact k-th of all threads may be above)
      from = (uint32_t)(kth_of_threads<kThreads>(sh, in.v0 < in.v1 ? (uint64_t)all << 32 | (uint32_t)(kThreads - t) : 0, a.top) >> 32);
    const bool sparse = from <= kNone;              // fewer than k threads have any other: all of those, and the first -inf
    const uint32_t reach = sparse ? kNone + 1 : from;
    for (int i = 0; i < slot; ++i)
      if (ranks[i * kThreads + t] >= RankOf<T>::pack(reach)) {
        const int at = atomicAdd(sh.segments, 1);
        if (at < kLpSegments) sh.segment[at] = (uint16_t)(i * kThreads + t);
      }
    __syncthreads();
    const int segments = *sh.segments;
    const bool fits = segments <= kLpSegments;
    const float least = key_value((uint64_t)reach << 32);
    const auto push = [&](float v, int at) {
      const int to = atomicAdd(sh.count, 1);
      if (to < sh.room) sh.list[to] = argmax_key(v, (uint32_t)at);
    };
    for (int f = 0; fits && f < a.fold; ++f)
      each_element<T, kThreads>(sh, in, segments, a.fold, f, [&](float v, int at) {
        if (!(v < least)) push(v, at);
      });
    if (sparse) {                                   // (where they do not make up k, k -inf are among the first 2 k)
      const int first = in.v0 * Row::VE - in.skew > 0 ? in.v0 * Row::VE - in.skew : 0;
      const int64_t end = (int64_t)in.v1 * Row::VE - in.skew < in.vocab ? (int64_t)in.v1 * Row::VE - in.skew : in.vocab;
      for (int i = t; i < 2 * a.top && first + i < end; i += kThreads) {
        const float v = to_f32(in.x[first + i]);
        if (v == -INFINITY) push(v, first + i);
      }
    }
    __syncthreads();
    if (fits && *sh.count <= sh.room) cut_list<kThreads>(sh, *sh.count, a.top);
    else top_by_keys<T, kThreads>(a, sh, in, from, slot);
  }
  const Sums v = block_sums<kThreads>(shared, sum.settled());
  if (a.parts == 1) {
    write_row<T>(a, sh.list, row, v);
    return;
  }
  const int64_t at = row * a.parts + part;
  if (t == 0) a.sums[at] = f32x4{v.m, v.l, v.s, 0.f};
  if (kTop && t < a.top) a.keys[at * a.top + t] = sh.list[t];
}

template <typename T>
__global__ void __launch_bounds__(kLpWhole) logprob_join_kernel(LogprobArgs a) {
  extern __shared__ __align__(16) char lds[];
  __shared__ f32x4 shared[kLpWhole / 64];
  const TopLds sh(lds, a.top, kLpWhole);
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  Sums sum{-INFINITY, 0.f, 0.f};
  if (t < a.parts) {
    const f32x4 x = a.sums[row * a.parts + t];
    sum = Sums{x[0], x[1], x[2]};
  }
  const int n = a.parts * a.top;                    // (at most 32 k)
  for (int i = t; i < n; i += kLpWhole) sh.list[i] = a.keys[row * n + i];
  __syncthreads();
  if (a.top > 0) cut_list<kLpWhole>(sh, n, a.top);
  sum = block_sums<kLpWhole>(shared, sum);
  write_row<T>(a, sh.list, row, sum);
}
static_assert(kLpParts <= 32 && kLpSlots * kLpWhole <= 1 << 16 && kLpSegments >= kLpWhole && kLpTop <= kLpShort, "");

// Parts of a row: enough workgroups for the card, of at most 8192 elements each where the rows leave so many (kLpParts at most).
// Measured, us, at most 4096 / 8192: one row of 151936 bf16, top 5, 13.2 / 12.4, 32 of them 16.2 / 14.1, 32 of 32003 fp32, top 50,
// 20.1 / 19.3 (at most 2048: 23.3); at least 8192 (one part fewer) / at most, top 20: one row of 151936 14.8 / 12.6, of 32003 13.6 / 13.7.
// Two parts of a row below 16384 are not worth their join, two / one: one row of 8193, top 20, 12.2 / 9.3, of 12000 11.3 / 8.7 (16384,
// in two parts, 11.6), 32 of 12000 13.2 / 10.1, 200 fp32 ones 14.2 / 10.4.  2048 workgroups instead of 1024: 512 rows of 151936
// fp32 58 -> 65, 1024 mostly masked ones of bf16 70 -> 95.
static int parts_for(int64_t rows, int64_t vocab) {
  int64_t parts = 1024 / rows;
  const int64_t most = vocab < 2 * 8192 ? 1 : (vocab + 8191) / 8192;
  parts = parts < most ? parts : most;
  parts = parts < kLpParts ? parts : kLpParts;
  return parts > 1 ? (int)parts : 1;
}

}  // namespace bfly

using namespace bfly;

extern "C" int64_t bfly_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0) return 0;
  const int64_t parts = parts_for(rows, vocab);
  return parts == 1 ? 0 : rows * parts * (16 + 8 * (int64_t)top);
}

extern "C" int bfly_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                   const int64_t* tokens, int top, float* logprobs, float* entropy, float* top_logprobs,
                                   int64_t* top_tokens, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  BFLY_CHECK_ARG(dtype == BFLY_DTYPE_F32 || dtype == BFLY_DTYPE_BF16, "unsupported dtype %d", dtype);
  const int64_t es = dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(rows >= 0 && vocab > 0 && vocab < (1 << 30), "bad shape (1 to 2^30 - 1 logits a row)");
  BFLY_CHECK_ARG(top >= 0 && top <= kLpTop && top <= vocab, "top %d must be 0 to %d, and at most a row's logits", top, kLpTop);
  BFLY_CHECK_ARG(row_stride >= 0 && row_stride < ((int64_t)1 << 48), "bad row stride");
  if (rows == 0) return BFLY_OK;
  BFLY_CHECK_ARG(logits && tokens && logprobs && entropy && (top == 0 || (top_logprobs && top_tokens)), "null pointer");
  BFLY_CHECK_ARG((reinterpret_cast<uintptr_t>(logits) & (es - 1)) == 0, "logits must be aligned to their type");
  LogprobArgs a{};
  a.parts = parts_for(rows, vocab);
  BFLY_CHECK_ARG(rows * a.parts < (1 << 24), "too many rows");       // a grid holds fewer than 2^32 threads
  const int64_t need = bfly_token_logprobs_workspace_bytes(rows, vocab, top);
  BFLY_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)), "workspace too small");
  a.logits = static_cast<const char*>(logits); a.tokens = tokens; a.logprob = logprobs; a.entropy = entropy;
  a.top_logprob = top_logprobs; a.top_token = top_tokens; a.stride = row_stride * es; a.rows = rows; a.vocab = (int)vocab;
  a.top = top;
  a.sums = static_cast<f32x4*>(workspace);
  a.keys = reinterpret_cast<uint64_t*>(a.sums + rows * a.parts);
  const int64_t ve = 16 / es;
  const bool whole = aligned16(logits) && row_stride * es % 16 == 0;   // (else wherever a row's first element lies)
  const int64_t vectors = (vocab + (whole ? ve - 1 : 2 * ve - 2)) / ve;
  a.per = (int)((vectors + a.parts - 1) / a.parts);
  const int threads = a.parts == 1 && vectors <= kLpShort * 4 ? kLpShort : kLpWhole;
  const int64_t rounds = (a.per + threads * 4 - 1) / (threads * 4);
  a.fold = (int)((rounds + kLpSlots - 1) / kLpSlots);
  a.slots = (int)((rounds + a.fold - 1) / a.fold);
  const int lds = top > 0 ? TopLds::bytes(top, threads, a.slots, (int)es) : 0;
  const int join_lds = top > 0 ? TopLds::bytes(top, kLpWhole, 0, 0) : 0;
  const dim3 grid((unsigned)(rows * a.parts)), block(threads);
#define BFLY_LP(T, TOP)                                                                                            \
  do {                                                                                                             \
    if (threads == kLpShort) hipLaunchKernelGGL((logprob_kernel<T, TOP, kLpShort>), grid, block, lds, stream, a);  \
    else hipLaunchKernelGGL((logprob_kernel<T, TOP, kLpWhole>), grid, block, lds, stream, a);                      \
    if (a.parts > 1) hipLaunchKernelGGL((logprob_join_kernel<T>), dim3((unsigned)rows), block, join_lds, stream, a); \
  } while (0)
  if (dtype == BFLY_DTYPE_BF16) {
    if (top > 0) BFLY_LP(__bf16, true);
    else BFLY_LP(__bf16, false);
  } else {
    if (top > 0) BFLY_LP(float, true);
    else BFLY_LP(float, false);
  }
#undef BFLY_LP
  BFLY_CHECK_LAUNCH("bfly_token_logprobs");
  return BFLY_OK;
}
