// Rows into and out of the 4-bit paged cache on gfx950: the contracts are include/butterfly_amd_paged_q4.h's.
//
//   bias = bf16(min x), scale = bf16(max((max x - min x) / 15, 1e-8)), code = round((x - bias) / scale) in 0..15
//
// for each group of 32 or 64 elements of a row.  D / 8 lanes hold a head's row, 8 elements each; a group's
// extremes meet over its 4 or 8 lanes on DPP.  The arithmetic is 64 bits wide, at the same rate here as 32: next to a
// border between two codes 32 bits would give other codes for another order of a sum.
//
// Bound by HBM and the 64-bit arithmetic for prompts (rows read once, codes and scales written once), by latency for a step's
// rows.  16411 rows of 16 and 4 heads of 256 with norm and RoPE: q 51 us (5.3 TB/s), k and v 48; 4099 rows of 4 heads of 128
// as they lie 5.6 us, 32 rows of 16 and 4 heads with norm and RoPE 3.5; 32768 tokens of 4 heads of 128 out again 20 us (4.3 TB/s).
#include "paged_q4.h"

namespace bfly {

// --------------------------------------------------------------------------- one row's codes
// DPP within 16 lanes: the neighbour in a pair, the other pair of four, the other four of eight and the other eight
// (mirrored: every lane of a four or eight holds the same by then).
constexpr int kPair = 0xB1, kQuad = 0x4E, kEight = 0x141, kRow = 0x140;
template <int kCtrl>
__device__ __forceinline__ int dpp(int x) { return __builtin_amdgcn_update_dpp(0, x, kCtrl, 0xf, 0xf, false); }
template <int kCtrl>
__device__ __forceinline__ float dpp(float x) { return __int_as_float(dpp<kCtrl>(__float_as_int(x))); }
template <int kCtrl>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __double_as_longlong(x);
  return __longlong_as_double((int64_t)(((uint64_t)(uint32_t)dpp<kCtrl>((int)(u >> 32)) << 32) | (uint32_t)dpp<kCtrl>((int)(uint32_t)u)));
}
// over the 8 to 32 lanes of a row, in each of them
template <int kLanes, typename F>
__device__ __forceinline__ F row_sum(F x) {
  x += dpp<kPair>(x);
  x += dpp<kQuad>(x);
  x += dpp<kEight>(x);
  if constexpr (kLanes > 8) x += dpp<kRow>(x);
  if constexpr (kLanes > 16) x += __shfl_xor(x, 16);
  return x;
}
__device__ __forceinline__ float least(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double least(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }

// (opaque: from fp64 through fp32 to bf16 are two roundings by definition, which the compiler would contract into one)
__device__ __forceinline__ uint32_t bf16_bits(float x) {
  asm("" : "+v"(x));
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// a / b rounded as a division is, inv = 1 / b rounded so too: a first quotient, the rest of it, and the rest's part.
// (A 15th as the product alone is a step off where the quotient lies next to a border between two fp32 numbers that is also
// one between two bf16 numbers.)
__device__ __forceinline__ double quotient(double a, double b, double inv) {
  const double t = a * inv;
  return fma(fma(-t, b, a), inv, t);
}

// 8 elements y of a row in each of D / 8 lanes (gl: which): the row's codes, a dword a lane, and the scale and bias
// of a group in its first lane.  F: what the elements are exact in (a row as it lies: fp32).
template <int D, int G, typename F>
__device__ __forceinline__ void q4_store(const F (&y)[8], int gl, char* codes, char* scales) {
  constexpr int LG = G / 8;                         // lanes of a group
  F lo = y[0], hi = y[0], nan = y[0] - y[0];        // (0, or NaN where there is an infinity or NaN)
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = least(lo, y[e]);
    hi = most(hi, y[e]);
    nan += y[e] - y[e];
  }
  int bad = nan == 0 ? 0 : 1;
  lo = least(lo, dpp<kPair>(lo)), hi = most(hi, dpp<kPair>(hi)), bad |= dpp<kPair>(bad);
  lo = least(lo, dpp<kQuad>(lo)), hi = most(hi, dpp<kQuad>(hi)), bad |= dpp<kQuad>(bad);
  if constexpr (LG == 8) lo = least(lo, dpp<kEight>(lo)), hi = most(hi, dpp<kEight>(hi)), bad |= dpp<kEight>(bad);
  uint32_t sb = bf16_bits((float)fmax(quotient((double)hi - (double)lo, 15.0, 1.0 / 15.0), 1e-8)), bb = bf16_bits((float)lo);
  bad |= (sb & 0x7f80u) == 0x7f80u || (bb & 0x7f80u) == 0x7f80u;
  if (bad) sb = bb = 0x7fc0u;
  const double s = __uint_as_float(sb << 16), b = __uint_as_float(bb << 16), inv = 1.0 / s;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    w |= (uint32_t)(int)fmin(fmax(rint(quotient((double)y[e] - b, s, inv)), 0.0), 15.0) << (4 * e);   // (NaN: 0)
  }
  if (bad) w = 0;
  // dword gl of the row: half-words hw = c * H + h, c the piece (of 16) and h the pair of groups (G = 32) or the group
  constexpr int H = D / 64;
  const int lane = threadIdx.x & 63, base = lane - gl;
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int hw = 2 * gl + i, c = hw / H, h = hw % H;
    uint32_t x;
    if constexpr (G == 64) {
      x = __shfl(w, base + 8 * h + (c >> 1)) >> (16 * (c & 1)) & 0xffffu;
    } else {
      const int at = 8 * (c & 3);
      x = (__shfl(w, base + 8 * h + (c >> 2)) >> at & 0xffu) | (__shfl(w, base + 8 * h + 4 + (c >> 2)) >> at & 0xffu) << 8;
    }
    out |= x << (16 * i);
  }
  *reinterpret_cast<uint32_t*>(codes + 4 * gl) = out;
  if (gl % LG == 0) *reinterpret_cast<uint32_t*>(scales + 4 * (gl / LG)) = sb | bb << 16;
}

template <typename T>
struct Row8;                                        // 8 elements as they lie
template <>
struct Row8<__bf16> {
  bf16x8 x;
  template <bool kStream = false>
  __device__ __forceinline__ void load(const char* p) {
    const bf16x8* q = reinterpret_cast<const bf16x8*>(p);
    x = kStream ? __builtin_nontemporal_load(q) : *q;
  }
  __device__ __forceinline__ float get(int e) const { return (float)x[e]; }
  __device__ __forceinline__ Row8 from(int lane) const {
    typedef __attribute__((ext_vector_type(4))) int i32x4;
    const i32x4 v = __builtin_bit_cast(i32x4, x);
    i32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __shfl(v[i], lane);
    return Row8{__builtin_bit_cast(bf16x8, y)};
  }
  template <bool kStream = false>
  static __device__ __forceinline__ void store(char* p, const float (&y)[8]) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (__bf16)y[e];
    if (kStream) __builtin_nontemporal_store(o, reinterpret_cast<bf16x8*>(p));
    else *reinterpret_cast<bf16x8*>(p) = o;
  }
};
template <>
struct Row8<float> {
  f32x4 x[2];
  template <bool kStream = false>
  __device__ __forceinline__ void load(const char* p) {
    const f32x4* q = reinterpret_cast<const f32x4*>(p);
    x[0] = kStream ? __builtin_nontemporal_load(q) : q[0];
    x[1] = kStream ? __builtin_nontemporal_load(q + 1) : q[1];
  }
  __device__ __forceinline__ float get(int e) const { return x[e >> 2][e & 3]; }
  __device__ __forceinline__ Row8 from(int lane) const {
    Row8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.x[i >> 2][i & 3] = __shfl(x[i >> 2][i & 3], lane);
    return y;
  }
  template <bool kStream = false>
  static __device__ __forceinline__ void store(char* p, const float (&y)[8]) {
    f32x4* q = reinterpret_cast<f32x4*>(p);
    const f32x4 a = {y[0], y[1], y[2], y[3]}, b = {y[4], y[5], y[6], y[7]};
    if (kStream) {
      __builtin_nontemporal_store(a, q);
      __builtin_nontemporal_store(b, q + 1);
    } else {
      q[0] = a;
      q[1] = b;
    }
  }
};

// --------------------------------------------------------------------------- rows into pages
struct Q4AppendArgs {
  const char* k;
  const char* v;
  const int64_t* slots;
  Q4Ptr pages;
  int64_t k_row, k_head, v_row, v_head;   // bytes
  int64_t limit;                          // num_pages * page_size
  unsigned items;                         // rows x heads, below 2^31
  unsigned hkv;
  int shift;
};

template <typename T, int D, int G>
__global__ void __launch_bounds__(256) q4_append_kernel(Q4AppendArgs a) {
  constexpr int LPR = D / 8;
  const int gl = threadIdx.x % LPR;
  const unsigned item = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;
  if (item >= a.items) return;                      // whole groups of lanes, here and below
  const unsigned r = item / a.hkv, h = item - r * a.hkv;
  const int64_t slot = a.slots[r];
  if (slot < 0 || slot >= a.limit) return;
  const bool is_v = blockIdx.y != 0;
  const char* from = is_v ? a.v : a.k;
  const int64_t row = is_v ? a.v_row : a.k_row, head = is_v ? a.v_head : a.k_head;
  Row8<T> x;
  x.load(from + r * row + h * head + 8 * sizeof(T) * gl);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = x.get(e);
  const int64_t id = slot >> a.shift;
  const int at = (int)(slot & ((1 << a.shift) - 1));
  const PagePtr codes = is_v ? a.pages.vc : a.pages.kc, scales = is_v ? a.pages.vs : a.pages.ks;
  q4_store<D, G>(y, gl, codes.row(id, h, at), scales.row(id, h, at));
}

// --------------------------------------------------------------------------- norm, RoPE, rows into pages
// q: y = x rsqrt(mean x^2 + eps) w, z = y cos + rotate_half(y) sin in fp32, one rounding.  k: the same in 64 bits, then
// its codes.  v: its codes.  The other half of a rotation comes as x from the lane that holds it, with its weight.
struct Q4RopeArgs {
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
  Q4Ptr pages;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // bytes
  int64_t limit, table_rows;
  unsigned rows, q_blocks, k_blocks;      // workgroups of q heads, of k heads; the others are v's
  int hq, hkv, shift, rot;
  double eps;
};

// cos and sin of a lane's 8 elements (1 and 0 beyond the rotation; si: with the sign of the other half's part).
struct Turn {
  float c[8], si[8];
  int step;                                         // lanes to the other half
  bool inside;
  __device__ __forceinline__ void load(const Q4RopeArgs& a, int gl, int64_t pos) {
    const int half = a.rot / 2 / 8;
    step = gl < half ? half : gl < 2 * half ? -half : 0;
    inside = pos >= 0 && pos < a.table_rows;
    const int64_t at = step != 0 ? (inside ? pos : 0) * a.rot + 8 * gl : 0;
#pragma unroll
    for (int e4 = 0; e4 < 8; e4 += 4) {
      const f32x4 cv = *reinterpret_cast<const f32x4*>(a.cos + at + e4), sv = *reinterpret_cast<const f32x4*>(a.sin + at + e4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e4 + e] = step != 0 ? cv[e] : 1.f;
        si[e4 + e] = step > 0 ? -sv[e] : sv[e];
      }
    }
  }
};

// A head's row after norm and rotation, in F.
template <int D, typename T, typename F>
__device__ __forceinline__ void rope_row(const Q4RopeArgs& a, const Row8<T>& x, const T* w, int gl, const Turn& turn, F (&z)[8]) {
  constexpr int LPR = D / 8;
  const Row8<T> o = x.from((threadIdx.x & 63) + turn.step);   // (every lane of the row takes part)
  F y[8], t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = x.get(e);
    t[e] = o.get(e);
  }
  if (w != nullptr) {
    F ss = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = y[e] * y[e] + ss;
    ss = row_sum<LPR>(ss);
    F r;
    if constexpr (sizeof(F) == 8) r = 1.0 / sqrt(ss * (1.0 / D) + a.eps);
    else r = rsqrtf(ss * (1.f / D) + (float)a.eps);
    Row8<T> wv, wo;
    wv.load(reinterpret_cast<const char*>(w + 8 * gl));
    wo.load(reinterpret_cast<const char*>(w + 8 * (gl + turn.step)));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = y[e] * r * (F)wv.get(e);
      t[e] = t[e] * r * (F)wo.get(e);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const F v = y[e] * (F)turn.c[e] + t[e] * (F)turn.si[e];
    z[e] = !turn.inside ? (F)__builtin_nanf("") : turn.step != 0 ? v : y[e];
  }
}

// A group of D / 8 lanes takes kHeads heads of a token, all of q, of k or of v.  kHeads = 1: a decode step's few rows, spread as
// wide as they go; what they write stays in the caches for the attention that follows.  kHeads = 4, from kManyHeads heads'
// rows on: four loads are under way over one position's cos and sin, and q moves past the caches.  Measured (with the pages read
// back), us, 1 / 4: 350 rows of 16 and 4 heads of 128 6.8 / 12.7, 1400 11.5 / 14.9, 2800 19.3 / 20.4, 5600 (2^17 heads' rows) 31.7 / 31.7,
// 16411 of 256 176 / 132.
constexpr int64_t kManyHeads = 1 << 17;

// Then q has a launch of its own as well (kPart 1, k and v: 2, all: 0): without k's fp64 its lanes need half the registers
// (132 -> 125 us).
template <typename T, int D, int G, int kHeads, int kPart>
__global__ void __launch_bounds__(256) q4_rope_append_kernel(Q4RopeArgs a) {
  constexpr int LPR = D / 8, kGroups = 256 / LPR;
  const int gl = threadIdx.x % LPR;
  const unsigned q_blocks = kPart == 0 ? a.q_blocks : 0;
  const bool is_q = kPart == 0 ? blockIdx.x < q_blocks : kPart == 1, is_k = !is_q && blockIdx.x < q_blocks + a.k_blocks;
  const unsigned block = blockIdx.x - (is_q ? 0 : is_k ? q_blocks : q_blocks + a.k_blocks);
  const unsigned heads = is_q ? a.hq : a.hkv, chunks = (heads + kHeads - 1) / kHeads;
  const unsigned item = block * kGroups + threadIdx.x / LPR, r = item / chunks;
  if (r >= a.rows) return;                          // whole groups of lanes, here and below
  const unsigned head0 = (item - r * chunks) * kHeads;
  const char* from = is_q ? a.q : is_k ? a.k : a.v;
  const int64_t row = is_q ? a.q_row : is_k ? a.k_row : a.v_row, head = is_q ? a.q_head : is_k ? a.k_head : a.v_head;
  const int64_t slot = a.slots[r];
  if (!is_q && (slot < 0 || slot >= a.limit)) return;
  Row8<T> x[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (kHeads == 1 || head0 + i < heads) x[i].template load<(kHeads > 1)>(from + r * row + (head0 + i) * head + 8 * sizeof(T) * gl);
  Turn turn;
  if (is_q || is_k) turn.load(a, gl, a.positions[r]);
  const int64_t id = slot >> a.shift;
  const int at = (int)(slot & ((1 << a.shift) - 1));
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = (int)head0 + i;
    if (kHeads > 1 && h >= (int)heads) break;
    if (is_q) {
      float z[8];
      rope_row<D>(a, x[i], static_cast<const T*>(a.qw), gl, turn, z);
      Row8<T>::template store<(kHeads > 1)>(a.q_out + (((int64_t)r * a.hq + h) * D + 8 * gl) * (int64_t)sizeof(T), z);
    } else if (is_k) {
      double z[8];
      rope_row<D>(a, x[i], static_cast<const T*>(a.kw), gl, turn, z);
      q4_store<D, G>(z, gl, a.pages.kc.row(id, h, at), a.pages.ks.row(id, h, at));
    } else {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = x[i].get(e);
      q4_store<D, G>(z, gl, a.pages.vc.row(id, h, at), a.pages.vs.row(id, h, at));
    }
  }
}

// --------------------------------------------------------------------------- rows out of pages
struct Q4ReadArgs {
  const int32_t* table;
  char* k;
  char* v;
  Q4Ptr pages;
  int64_t table_stride, items;            // items: rows of k (and of v)
  int tokens, hkv, shift, num_pages;
};

template <typename T, int D, int G>
__global__ void __launch_bounds__(256) q4_read_kernel(Q4ReadArgs a) {
  constexpr int LPR = D / 8, H = D / 64;
  const int gl = threadIdx.x % LPR, lane = threadIdx.x & 63, base = lane - gl;
  const int64_t item = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (item >= a.items) return;                      // whole groups of lanes
  const bool is_v = blockIdx.y != 0;
  const unsigned tokens = a.tokens, hkv = a.hkv;
  const unsigned bh = (unsigned)(item / tokens), t = (unsigned)(item - (int64_t)bh * tokens);
  const unsigned b = bh / hkv, h = bh - b * hkv;
  const int id = a.table[b * a.table_stride + (t >> a.shift)];
  const bool there = (unsigned)id < (unsigned)a.num_pages;
  const int at = (int)(t & ((1u << a.shift) - 1));
  const PagePtr &codes = is_v ? a.pages.vc : a.pages.kc, &scales = is_v ? a.pages.vs : a.pages.ks;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(codes.row(there ? id : 0, h, at) + 4 * gl);
  const uint32_t sb = *reinterpret_cast<const uint32_t*>(scales.row(there ? id : 0, h, at) + 4 * (gl / (G / 8)));
  // elements 8 gl and on: half-word c * H + h of the row for each piece c that holds some of them
  uint32_t x = 0;
  if constexpr (G == 64) {
    const int c = 2 * (gl & 7), g = gl >> 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int hw = (c + i) * H + g;
      x |= (__shfl(w, base + (hw >> 1)) >> (16 * (hw & 1)) & 0xffffu) << (16 * i);
    }
  } else {
    const int c = 4 * (gl & 3), g = gl >> 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int hw = (c + i) * H + (g >> 1);
      x |= (__shfl(w, base + (hw >> 1)) >> (16 * (hw & 1) + 8 * (g & 1)) & 0xffu) << (8 * i);
    }
  }
  const float s = there ? __uint_as_float(sb << 16) : __builtin_nanf(""), bias = __uint_as_float(sb & 0xffff0000u);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = fmaf((float)(x >> (4 * e) & 15u), s, bias);
  Row8<T>::store((is_v ? a.v : a.k) + (item * D + 8 * gl) * (int64_t)sizeof(T), y);
}

// --------------------------------------------------------------------------- host
int q4_check_pages(const char* what, const bfly_q4_pages_t& p, int64_t head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("%s: head_dim=%lld unsupported (64, 128, 256)", what, (long long)head_dim);
    return BFLY_ERR_UNSUPPORTED;
  }
  BFLY_CHECK_ARG(p.group == 32 || p.group == 64, "%s: group %lld must be 32 or 64", what, (long long)p.group);
  BFLY_CHECK_ARG(p.page_size >= 16 && p.page_size <= 1024 && (p.page_size & (p.page_size - 1)) == 0,
                 "%s: page_size %lld must be a power of two from 16 to 1024", what, (long long)p.page_size);
  BFLY_CHECK_ARG(p.num_pages > 0 && p.num_pages <= INT32_MAX, "%s: bad num_pages", what);
  for (const int64_t s : {p.k_codes_page, p.k_codes_head, p.k_codes_row, p.v_codes_page, p.v_codes_head, p.v_codes_row})
    BFLY_CHECK_ARG(s >= 0 && s < ((int64_t)1 << 48) && s % 16 == 0, "%s: strides of the codes must be multiples of 16 bytes",
                   what);
  const int64_t row = 4 * head_dim / p.group, unit = row < 16 ? row : 16;
  for (const int64_t s : {p.k_scales_page, p.k_scales_head, p.k_scales_row, p.v_scales_page, p.v_scales_head, p.v_scales_row})
    BFLY_CHECK_ARG(s >= 0 && s < ((int64_t)1 << 48) && s % unit == 0,
                   "%s: strides of the scales must be multiples of %lld bytes", what, (long long)unit);
  // offsets inside a page and head are kept in 32 bits
  for (const int64_t s : {p.k_codes_row, p.v_codes_row, p.k_scales_row, p.v_scales_row})
    BFLY_CHECK_ARG(s * p.page_size <= INT32_MAX, "%s: row stride too large", what);
  return BFLY_OK;
}

static bool strides16(std::initializer_list<int64_t> st, int64_t esize) {
  for (int64_t s : st)
    if (s < 0 || s >= ((int64_t)1 << 48) || (s * esize) % 16 != 0) return false;
  return true;
}

}  // namespace bfly

using namespace bfly;

// KERNEL<T, D, G> by type, head_dim and group (checked before).
#define BFLY_Q4_GROUP(KERNEL, T, D, grid, a)                                                         \
  do {                                                                                               \
    if (x.pages.group == 32) hipLaunchKernelGGL((KERNEL<T, D, 32>), grid, dim3(256), 0, stream, a);  \
    else hipLaunchKernelGGL((KERNEL<T, D, 64>), grid, dim3(256), 0, stream, a);                      \
  } while (0)
#define BFLY_Q4_DIM(KERNEL, T, grid, a)                              \
  do {                                                               \
    if (x.head_dim == 64) BFLY_Q4_GROUP(KERNEL, T, 64, grid, a);     \
    else if (x.head_dim == 128) BFLY_Q4_GROUP(KERNEL, T, 128, grid, a); \
    else BFLY_Q4_GROUP(KERNEL, T, 256, grid, a);                     \
  } while (0)
#define BFLY_Q4_LAUNCH(KERNEL, grid, a)                               \
  do {                                                                \
    if (x.dtype == BFLY_DTYPE_BF16) BFLY_Q4_DIM(KERNEL, __bf16, grid, a); \
    else BFLY_Q4_DIM(KERNEL, float, grid, a);                         \
  } while (0)

extern "C" int bfly_paged_q4_append(const bfly_paged_q4_append_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_q4_append_args_t& x = *args;
  BFLY_CHECK_ARG(x.dtype == BFLY_DTYPE_F32 || x.dtype == BFLY_DTYPE_BF16, "unsupported dtype %lld", (long long)x.dtype);
  const int64_t es = x.dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(x.rows >= 0 && x.rows <= INT32_MAX && x.hkv > 0 && x.hkv <= 65535, "bad shape");
  const int rc = q4_check_pages("bfly_paged_q4_append", x.pages, x.head_dim);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(strides16({x.k_row_stride, x.k_head_stride, x.v_row_stride, x.v_head_stride}, es),
                 "row and head strides must be multiples of 16 bytes");
  if (x.rows == 0) return BFLY_OK;
  BFLY_CHECK_ARG(x.k && x.v && x.slots && q4_given(x.pages), "null pointer");
  BFLY_CHECK_ARG(aligned16(x.k) && aligned16(x.v) && q4_aligned(x.pages), "pointers must be 16-byte aligned");
  Q4AppendArgs a{};
  a.k = static_cast<const char*>(x.k); a.v = static_cast<const char*>(x.v); a.slots = x.slots; a.pages = q4_ptr(x.pages);
  a.k_row = x.k_row_stride * es; a.k_head = x.k_head_stride * es; a.v_row = x.v_row_stride * es; a.v_head = x.v_head_stride * es;
  a.limit = x.pages.num_pages * x.pages.page_size; a.hkv = (unsigned)x.hkv;
  a.shift = __builtin_ctzll(x.pages.page_size);
  BFLY_CHECK_ARG(x.rows * x.hkv < ((int64_t)1 << 30), "too many rows");
  a.items = (unsigned)(x.rows * x.hkv);
  const int64_t blocks = (a.items * (x.head_dim / 8) + 255) / 256;
  BFLY_CHECK_ARG(blocks < (1 << 23), "too many rows");        // a grid (of k and v) holds fewer than 2^32 threads
  BFLY_Q4_LAUNCH(q4_append_kernel, dim3((unsigned)blocks, 2), a);
  BFLY_CHECK_LAUNCH("bfly_paged_q4_append");
  return BFLY_OK;
}

extern "C" int bfly_paged_q4_rope_append(const bfly_paged_q4_rope_append_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_q4_rope_append_args_t& x = *args;
  BFLY_CHECK_ARG(x.dtype == BFLY_DTYPE_F32 || x.dtype == BFLY_DTYPE_BF16, "unsupported dtype %lld", (long long)x.dtype);
  const int64_t es = x.dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(x.rows >= 0 && x.rows <= INT32_MAX, "bad shape");
  BFLY_CHECK_ARG(x.hkv > 0 && x.hq > 0 && x.hq <= (1 << 20) && x.hkv <= x.hq && x.hq % x.hkv == 0,
                 "bad head counts hq=%lld hkv=%lld", (long long)x.hq, (long long)x.hkv);
  const int rc = q4_check_pages("bfly_paged_q4_rope_append", x.pages, x.head_dim);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(x.rotary_dim > 0 && x.rotary_dim <= x.head_dim && x.rotary_dim % 16 == 0,
                 "rotary_dim %lld must be a multiple of 16, at most head_dim", (long long)x.rotary_dim);
  BFLY_CHECK_ARG(x.table_rows > 0, "the cos/sin tables must have rows");
  BFLY_CHECK_ARG(strides16({x.q_row_stride, x.q_head_stride, x.k_row_stride, x.k_head_stride, x.v_row_stride,
                            x.v_head_stride}, es),
                 "row and head strides must be multiples of 16 bytes");
  if (x.rows == 0) return BFLY_OK;
  BFLY_CHECK_ARG(x.q && x.k && x.v && x.cos && x.sin && x.positions && x.slots && x.q_out && q4_given(x.pages), "null pointer");
  BFLY_CHECK_ARG((x.q_weight == nullptr) == (x.k_weight == nullptr), "both norm weights or neither");
  BFLY_CHECK_ARG(aligned16(x.q) && aligned16(x.k) && aligned16(x.v) && aligned16(x.cos) && aligned16(x.sin) && aligned16(x.q_out) &&
                     q4_aligned(x.pages) && aligned16(x.q_weight) && aligned16(x.k_weight),
                 "pointers must be 16-byte aligned");
  Q4RopeArgs a{};
  a.q = static_cast<const char*>(x.q); a.k = static_cast<const char*>(x.k); a.v = static_cast<const char*>(x.v);
  a.qw = x.q_weight; a.kw = x.k_weight; a.cos = x.cos; a.sin = x.sin; a.positions = x.positions; a.slots = x.slots;
  a.q_out = static_cast<char*>(x.q_out); a.pages = q4_ptr(x.pages);
  a.q_row = x.q_row_stride * es; a.q_head = x.q_head_stride * es; a.k_row = x.k_row_stride * es;
  a.k_head = x.k_head_stride * es; a.v_row = x.v_row_stride * es; a.v_head = x.v_head_stride * es;
  a.limit = x.pages.num_pages * x.pages.page_size; a.table_rows = x.table_rows; a.hq = (int)x.hq; a.hkv = (int)x.hkv;
  a.shift = __builtin_ctzll(x.pages.page_size); a.rot = (int)x.rotary_dim; a.eps = x.eps;
  const int64_t heads = x.hq + 2 * x.hkv;
  BFLY_CHECK_ARG(x.rows * heads < ((int64_t)1 << 31) - 256, "too many rows");
  const int64_t each = x.rows * heads >= kManyHeads ? 4 : 1, groups = 256 / (x.head_dim / 8);
  const auto blocks = [&](int64_t h) { return (x.rows * ((h + each - 1) / each) + groups - 1) / groups; };
  BFLY_CHECK_ARG(blocks(x.hq) + 2 * blocks(x.hkv) < (1 << 24), "too many rows");   // a grid holds fewer than 2^32 threads
  a.rows = (unsigned)x.rows; a.q_blocks = (unsigned)blocks(x.hq); a.k_blocks = (unsigned)blocks(x.hkv);
#define BFLY_Q4_ROPE(T, D, G)                                                                                    \
  do {                                                                                                           \
    if (each == 1) {                                                                                             \
      hipLaunchKernelGGL((q4_rope_append_kernel<T, D, G, 1, 0>), dim3(a.q_blocks + 2 * a.k_blocks), dim3(256), 0, stream, a); \
    } else {                                                                                                     \
      hipLaunchKernelGGL((q4_rope_append_kernel<T, D, 64, 4, 1>), dim3(a.q_blocks), dim3(256), 0, stream, a);     \
      hipLaunchKernelGGL((q4_rope_append_kernel<T, D, G, 4, 2>), dim3(2 * a.k_blocks), dim3(256), 0, stream, a); \
    }                                                                                                            \
  } while (0)
#define BFLY_Q4_ROPE_G(T, D)                        \
  do {                                              \
    if (x.pages.group == 32) BFLY_Q4_ROPE(T, D, 32); \
    else BFLY_Q4_ROPE(T, D, 64);                    \
  } while (0)
#define BFLY_Q4_ROPE_D(T)                            \
  do {                                               \
    if (x.head_dim == 64) BFLY_Q4_ROPE_G(T, 64);     \
    else if (x.head_dim == 128) BFLY_Q4_ROPE_G(T, 128); \
    else BFLY_Q4_ROPE_G(T, 256);                     \
  } while (0)
  if (x.dtype == BFLY_DTYPE_BF16) BFLY_Q4_ROPE_D(__bf16);
  else BFLY_Q4_ROPE_D(float);
#undef BFLY_Q4_ROPE_D
#undef BFLY_Q4_ROPE_G
#undef BFLY_Q4_ROPE
  BFLY_CHECK_LAUNCH("bfly_paged_q4_rope_append");
  return BFLY_OK;
}

extern "C" int bfly_paged_q4_read(const bfly_paged_q4_read_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_q4_read_args_t& x = *args;
  BFLY_CHECK_ARG(x.dtype == BFLY_DTYPE_F32 || x.dtype == BFLY_DTYPE_BF16, "unsupported dtype %lld", (long long)x.dtype);
  BFLY_CHECK_ARG(x.requests >= 0 && x.requests <= (1 << 24) && x.hkv > 0 && x.hkv <= 65535, "bad shape");
  const int rc = q4_check_pages("bfly_paged_q4_read", x.pages, x.head_dim);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(x.table_width >= 0 && x.table_width <= INT32_MAX && (x.requests <= 1 || x.table_stride >= 0),
                 "bad block table shape");
  BFLY_CHECK_ARG(x.tokens >= 0 && x.tokens <= INT32_MAX && x.tokens <= x.table_width * x.pages.page_size,
                 "tokens beyond the block table");
  if (x.requests == 0 || x.tokens == 0) return BFLY_OK;
  BFLY_CHECK_ARG(x.block_table && x.k && x.v && q4_given(x.pages), "null pointer");
  BFLY_CHECK_ARG(aligned16(x.k) && aligned16(x.v) && q4_aligned(x.pages), "pointers must be 16-byte aligned");
  Q4ReadArgs a{};
  a.table = x.block_table; a.k = static_cast<char*>(x.k); a.v = static_cast<char*>(x.v); a.pages = q4_ptr(x.pages);
  a.table_stride = x.table_stride; a.tokens = (int)x.tokens; a.hkv = (int)x.hkv;
  a.shift = __builtin_ctzll(x.pages.page_size); a.num_pages = (int)x.pages.num_pages;
  const int64_t heads = x.requests * x.hkv;                   // (below 2^40: no overflow against tokens below 2^31 in the test)
  BFLY_CHECK_ARG(heads < ((int64_t)1 << 31) && heads <= ((int64_t)1 << 31) / x.tokens, "too many rows");
  a.items = heads * x.tokens;
  const int64_t blocks = (a.items * (x.head_dim / 8) + 255) / 256;
  BFLY_CHECK_ARG(blocks < (1 << 23), "too many rows");        // a grid (of k and v) holds fewer than 2^32 threads
  BFLY_Q4_LAUNCH(q4_read_kernel, dim3((unsigned)blocks, 2), a);
  BFLY_CHECK_LAUNCH("bfly_paged_q4_read");
  return BFLY_OK;
}
