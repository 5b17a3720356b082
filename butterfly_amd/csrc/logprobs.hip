// Log probabilities of given tokens, entropy and the top alternatives, from rows of logits
// (bfly_token_logprobs, include/butterfly_amd_decoder.h).
//
//   m = max x, l = sum exp(x - m), s = sum exp(x - m) (x - m):
//   log p(token) = (x_token - m) - log l,   H = log l - s / l,   in one pass with a running m, l and s.
//
// A workgroup takes a row, or (few rows) one of up to 32 parts of a row, in rounds of 32 elements a thread; a second
// launch joins the parts.  Every thread keeps a running maximum and sums of its own until the end.
//
// The top k ride along as 64-bit keys (value's order, then the lower index; argmax_key), which are unique.  In the first
// round k threads' largest keys bound the k-th largest from below: the elements from there on (in k threads, so
// at most 32 k) go to a list in LDS.  Later rounds look at each thread's maximum only, and add what is above the bound; a
// list that would overflow is cut to its k largest first, which raises the bound.
#include "argmax.h"

#include "../../include/butterfly_amd_decoder.h"

namespace bfly {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

constexpr int kLpThreads = 256, kLpEach = 32;       // threads, elements of a thread in a round
constexpr int kLpTop = 64;                          // top at most
constexpr int kLpParts = 32;                        // parts of a row at most
constexpr int kLpList = kLpTop + kLpTop * kLpEach;  // the list: k kept and a first round's candidates
constexpr int kLpFew = kLpTop * ((kLpList + kLpThreads - 1) / kLpThreads);
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpFar = -1e30f;                    // below every difference that counts, and finite

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
};

struct Sums {
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

struct LpShared {
  uint64_t list[kLpList], few[kLpFew], most[kLpThreads], bound;
  f32x4 sums[kLpThreads / 64];
  int count, kept;
};

// The k-th largest of the threads' keys, 0 where fewer than k are above 0 (which are unique).
__device__ __forceinline__ uint64_t kth_of_threads(LpShared& sh, uint64_t mine, int k) {
  const int t = threadIdx.x;
  __syncthreads();
  sh.most[t] = mine;
  if (t == 0) sh.bound = 0;
  __syncthreads();
  int above = 0;
#pragma unroll 8
  for (int j = 0; j < kLpThreads; ++j) above += sh.most[j] > mine;
  if (mine != 0 && above == k - 1) sh.bound = mine;
  __syncthreads();
  return sh.bound;
}

// The list's n keys to its k largest in order (0 behind the last).
__device__ __forceinline__ void cut_list(LpShared& sh, int n, int k) {
  const int t = threadIdx.x;
  uint64_t from = 1;
  if (n > kLpThreads) {
    uint64_t mine = 0;
    for (int i = t; i < n; i += kLpThreads) mine = sh.list[i] > mine ? sh.list[i] : mine;
    from = kth_of_threads(sh, mine, k);             // (at least k threads have keys)
  }
  __syncthreads();
  if (t == 0) sh.kept = 0;
  __syncthreads();
  for (int i = t; i < n; i += kLpThreads) {
    const uint64_t x = sh.list[i];
    if (x >= from && x != 0) sh.few[atomicAdd(&sh.kept, 1)] = x;   // k threads' at most: kLpFew
  }
  __syncthreads();
  const int kept = sh.kept;
  for (int i = t; i < k; i += kLpThreads)
    if (i >= kept) sh.list[i] = 0;
  for (int i = t; i < kept; i += kLpThreads) {
    const uint64_t x = sh.few[i];
    int above = 0;
    for (int j = 0; j < kept; ++j) above += sh.few[j] > x;
    if (above < k) sh.list[above] = x;
  }
  if (t == 0) sh.count = kept < k ? kept : k;
  __syncthreads();
}

__device__ __forceinline__ Sums block_sums(LpShared& sh, Sums v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v.add(Sums{__shfl_xor(v.m, o), __shfl_xor(v.l, o), __shfl_xor(v.s, o)});
  if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = f32x4{v.m, v.l, v.s, 0.f};
  __syncthreads();
  v = Sums{sh.sums[0][0], sh.sums[0][1], sh.sums[0][2]};
#pragma unroll
  for (int w = 1; w < kLpThreads / 64; ++w) v.add(Sums{sh.sums[w][0], sh.sums[w][1], sh.sums[w][2]});
  return v;
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  if (u == 0xFFFFFFFFu) return __builtin_nanf("");
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// A row's results from its sums and its list (in order).
template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs& a, const LpShared& sh, int64_t row, const Sums& v) {
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
    const uint64_t key = sh.list[t];
    a.top_logprob[row * a.top + t] = key_value(key) - v.m - log_l;
    a.top_token[row * a.top + t] = argmax_key_index(key);
  }
}

template <typename T, bool kTop>
__global__ void __launch_bounds__(kLpThreads) logprob_kernel(LogprobArgs a) {
  constexpr int VE = 16 / sizeof(T), NV = kLpEach / VE;   // elements of a vector, vectors of a thread in a round
  typedef T vec __attribute__((ext_vector_type(VE)));
  __shared__ LpShared sh;
  const int t = threadIdx.x;
  const int64_t row = (int64_t)(blockIdx.x / (unsigned)a.parts);
  const int part = (int)(blockIdx.x % (unsigned)a.parts);
  const T* x0 = reinterpret_cast<const T*>(a.logits + row * a.stride);
  // vectors lie at whole 16 bytes: `skew` elements of the first one are before the row
  const int skew = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
  const int vectors = (int)(((int64_t)a.vocab + skew + VE - 1) / VE);
  const int v0 = part * a.per < vectors ? part * a.per : vectors, v1 = v0 + a.per < vectors ? v0 + a.per : vectors;
  Sums sum{-INFINITY, 0.f, 0.f};
  uint64_t bound = 0;                               // keys above it count; its value as a float (0: all count)
  float bound_v = 0.f;
  if (kTop && t == 0) sh.count = 0;
  for (int base = v0; base < v1; base += kLpThreads * NV) {
    float x[kLpEach];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = base + t + kLpThreads * i;
      const int64_t at = (int64_t)v * VE - skew;    // its first element
      if (v < v1 && at >= 0 && at + VE <= a.vocab) {
        const vec y = __builtin_nontemporal_load(reinterpret_cast<const vec*>(x0 + at));
#pragma unroll
        for (int e = 0; e < VE; ++e) x[VE * i + e] = to_f32(y[e]);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          x[VE * i + e] = v < v1 && at + e >= 0 && at + e < a.vocab ? to_f32(x0[at + e]) : -INFINITY;
      }
    }
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < kLpEach; ++i) mx = fmaxf(mx, x[i]);
    if (mx > sum.m) sum.to(mx);
    const float ref = sum.m == -INFINITY ? 0.f : sum.m;
    float l[2] = {0.f, 0.f}, s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kLpEach; ++i) {
      const float d = x[i] - ref, e = __builtin_amdgcn_exp2f(d * kLpLog2e);
      l[i & 1] += e;
      s[i & 1] = fmaf(e, fmaxf(d, kLpFar), s[i & 1]);
    }
    sum.l += l[0] + l[1];
    sum.s += s[0] + s[1];
    if constexpr (kTop) {
      // (indices grow from round to round: an element of the bound's value is behind it)
      const bool first = base == v0;
      if (!__syncthreads_or(bound == 0 || mx > bound_v || sum.l != sum.l)) continue;
      const auto each = [&](auto&& f) __attribute__((always_inline)) {   // this thread's keys above the bound
        static_for<kLpEach>([&](auto ic) __attribute__((always_inline)) {
          constexpr int i = decltype(ic)::value;
          const int v = base + t + kLpThreads * (i / VE), at = v * VE - skew + i % VE;   // (below 2^30 + 2^14)
          if (v < v1 && at >= 0 && at < a.vocab) {
            const uint64_t key = argmax_key(x[i], (uint32_t)at);
            if (key > bound) f(key);
          }
        });
      };
      const auto push = [&]() __attribute__((always_inline)) {
        each([&](uint64_t key) __attribute__((always_inline)) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kLpList) sh.list[at] = key;
        });
        __syncthreads();
      };
      const int before = sh.count;
      __syncthreads();
      bool over = first;
      if (!first) {
        push();
        over = sh.count > kLpList;
      }
      if (over) {
        __syncthreads();
        if (before > a.top) {
          cut_list(sh, before, a.top);
          bound = sh.list[a.top - 1];
        } else if (t == 0) {
          sh.count = before;
        }
        uint64_t mine = 0;
        each([&](uint64_t key) __attribute__((always_inline)) { mine = key > mine ? key : mine; });
        const uint64_t kth = kth_of_threads(sh, mine, a.top);
        if (kth != 0) bound = kth - 1;
        push();                                     // 32 keys of at most k threads
        bound_v = key_value(bound);
      }
    }
  }
  if constexpr (kTop) {
    __syncthreads();
    cut_list(sh, sh.count, a.top);
  }
  sum = block_sums(sh, sum);
  if (a.parts == 1) {
    write_row<T>(a, sh, row, sum);
    return;
  }
  const int64_t at = row * a.parts + part;
  if (t == 0) a.sums[at] = f32x4{sum.m, sum.l, sum.s, 0.f};
  if (kTop && t < a.top) a.keys[at * a.top + t] = sh.list[t];
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprob_join_kernel(LogprobArgs a) {
  __shared__ LpShared sh;
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  Sums sum{-INFINITY, 0.f, 0.f};
  if (t < a.parts) {
    const f32x4 x = a.sums[row * a.parts + t];
    sum = Sums{x[0], x[1], x[2]};
  }
  const int n = a.parts * a.top;
  for (int i = t; i < n; i += kLpThreads) sh.list[i] = a.keys[row * n + i];
  __syncthreads();
  if (a.top > 0) cut_list(sh, n, a.top);
  sum = block_sums(sh, sum);
  write_row<T>(a, sh, row, sum);
}
static_assert(kLpParts * kLpTop <= kLpList && kLpParts <= 64, "");

// Parts of a row: enough workgroups for the card, at least 4096 elements each.
static int parts_for(int64_t rows, int64_t vocab) {
  int64_t parts = 1024 / rows;
  const int64_t most = (vocab + 4095) / 4096;
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
  const int64_t ve = 16 / es, vectors = (vocab + 2 * ve - 2) / ve;   // of a row, wherever its first element lies
  a.per = (int)((vectors + a.parts - 1) / a.parts);
  const dim3 grid((unsigned)(rows * a.parts)), block(kLpThreads);
#define BFLY_LP(T)                                                                           \
  do {                                                                                       \
    if (top > 0) hipLaunchKernelGGL((logprob_kernel<T, true>), grid, block, 0, stream, a);   \
    else hipLaunchKernelGGL((logprob_kernel<T, false>), grid, block, 0, stream, a);          \
    if (a.parts > 1) hipLaunchKernelGGL((logprob_join_kernel<T>), dim3((unsigned)rows), block, 0, stream, a); \
  } while (0)
  if (dtype == BFLY_DTYPE_BF16) BFLY_LP(__bf16);
  else BFLY_LP(float);
#undef BFLY_LP
  BFLY_CHECK_LAUNCH("bfly_token_logprobs");
  return BFLY_OK;
}
