// One new token of every request over its 4-bit pages (include/butterfly_amd_paged_q4.h).
//
//   k_t = c_t s_t + b_t for each group of elements (codes c, scale s, bias b), v_t likewise;
//   s_t = scale q . k_t = scale sum_groups (s_t (q . c_t) + b_t sum q),   m = max s_t, l = sum exp(s_t - m),
//   o = (sum exp(s_t - m) v_t) / l,  v's scales and biases on the weights: sum (p_t s_t) c_t + sum p_t b_t.
//
// The schedule, runs and joins are those of paged_attn.hip (paged_runs.h); a workgroup's four waves take every fourth tile of
// 32 or 64 keys.  Both products run over the codes themselves: a code is exact in bf16 as c 2^-130, a number below the smallest
// exponent (a shift and an and for two codes), so nothing is rounded on the way from the cache to the sums but the weights, which
// enter as two bf16 parts (2^-17 of them is left; fp32: three, and q as three).  Three for bf16 brought its outputs no nearer to
// 64 bits and made the step of 32 requests below 82 us for 74.  Codes as 16 + c would do too, and need no care for the
// exponents, but the 16 q has to go again: scores were off by three times as much and fp32 outputs by 2^-20, and that step took 1 to
// 2 us more.  (Codes and q as 8-bit floats: as fast, but that instruction sums 8 products short of fp32, which puts scores 2^-16
// of their size off.)
// Layout: a row's 16 pieces hold a sixteenth of every group each.  S^T = K Q^T: lane (n, g) takes four pieces of key n (a
// quarter of every group), so each product is over one group.  O^T += V^T P^T: lane n takes piece n of a lane's keys, so the 16
// rows of each product are of one group, and P carries that group's scale.  Scales are read as lane (n, g) needs them, for keys
// 4 (n & 3) + g, and reach the other lanes of a four by DPP.
//
// Bound: the cache is read once, 72 + 72 bytes a key and head of 128 in groups of 64 against 512 in bf16.  Four query heads a kv
// head, bf16, d 128, 32 requests of 131072 tokens and less (385 MB): 73 us, 5.3 TB/s with the join (that of bf16 pages reads
// at 6.6, a copy runs at 5.8); there the vector instructions between the loads and the products (codes, scales, weights) take
// two thirds of the time, which is why they are counted: columns in blocks (below) took 101 us to 76.  One request of 32768
// tokens (19 MB): 14 us, mostly the two launches and two rounds of latency.
#include "paged_runs.h"
#include "paged_q4.h"

namespace bfly {

// Rounds (four tiles) of a request that one workgroup takes alone: the more pairs of a request and a kv head the
// more.  Measured, us, 4 for all / this rule / 32 for all: 64 requests of 2048 tokens and 4 kv heads 24.6 / 20.4 / 20.4, 256 of
// 1 to 4096 and 8 heads 99.5 / 83.4 / 83.2; 8 of 8192 and 4 heads 18.0 / 18.0 / 54.1.
constexpr int q4_whole_rounds(int64_t pairs) { return pairs >= 2048 ? 32 : pairs >= 512 ? 16 : pairs >= 128 ? 8 : 4; }

// A column's sums keep their reference until its maximum is more than this many powers of two above it: 16 columns of a
// tile hardly ever rise together, and one that rises would turn all sums over (32 requests of 131072: 77.4 -> 75.9 us, of 2000
// tokens 25.9 -> 25.5).  Weights are at most 2^4 then.
constexpr float kQ4Lag = 4.f;
// v's scales are taken times this, which keeps the weights' products with codes far from fp32's smallest numbers.
constexpr float kQ4Up = 0x1p40f;

struct Q4AttnArgs : RunArgs {
  const char* q;
  Q4Ptr p;
  int64_t q_req, q_head;                 // bytes
};

// lane (n & ~3) + R's x
template <int R>
__device__ __forceinline__ float of_four(float x) {
  constexpr int ctrl = R | R << 2 | R << 4 | R << 6;
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), ctrl, 0xf, 0xf, true));
}
// codes number j of both half-words of r as c 2^-130 in bf16, number 0 as c 2^-133: below the smallest exponent a word's bits are
// its number, and nothing is added to a code.  (The matrix instructions take such operands as they are.)
template <int J>
__device__ __forceinline__ uint32_t codes_of(uint32_t r) {
  return J == 0 ? r & 0x000f000fu : r >> (4 * J - 3) & 0x00780078u;
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Rows of one page and head, through a buffer descriptor: the row of a tile is a scalar offset, so a lane's offset is
// the same for every tile.
struct Rows {
  __amdgpu_buffer_rsrc_t page;
  int at;                                           // the tile's first row, in bytes
};
__device__ __forceinline__ Rows page_rows(const PagePtr& p, int64_t id, int h, int row, int page_size, int row_length) {
  return Rows{__builtin_amdgcn_make_buffer_rsrc(p.row(id, h, 0), (short)0, (page_size - 1) * p.row_bytes + row_length, 0x00020000),
              row * p.row_bytes};
}

template <int N>
struct Words {                                      // N dwords as they lie
  uint32_t w[N];
  template <int kPolicy>
  __device__ __forceinline__ void load(const Rows& r, int lane_at, int at) {
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r.page, lane_at + 4 * i, r.at + at, kPolicy));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = x[j];
      }
    } else if constexpr (N == 2) {
      const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r.page, lane_at, r.at + at, kPolicy));
      w[0] = x[0];
      w[1] = x[1];
    } else {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(r.page, lane_at, r.at + at, kPolicy);
    }
  }
  __device__ __forceinline__ void load(uint64_t address) {   // (somewhere else for every lane)
    typedef __attribute__((address_space(1))) const uint32_t* ptr;
    typedef __attribute__((address_space(1))) const u32x2* ptr2;
    typedef __attribute__((address_space(1))) const u32x4* ptr4;
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const u32x4 x = *(ptr4)(address + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = x[j];
      }
    } else if constexpr (N == 2) {
      const u32x2 x = *(ptr2)address;
      w[0] = x[0];
      w[1] = x[1];
    } else {
      w[0] = *(ptr)address;
    }
  }
};

// Columns of a product in J blocks of C = 16 / J: a block's columns are the rows of q for one subtile (16 keys) of J, so a
// lane's four results are of its own block's subtile and every lane of a unit with few query heads has
// weights to work on.  Rows of q are kept J times, each zero outside its block: the chain over J subtiles then ends in
// one accumulator.  Every column keeps a maximum and sums of its own until the end.
template <typename T, int D, int G, int J>
struct Q4Sweep {
  static constexpr int C = 16 / J;                  // rows of q
  static constexpr int U = J > 2 ? J : 2;           // subtiles of a tile
  static constexpr int A = U / J;                   // of them in a block: results 4 a + r of a lane
  static constexpr int KT = 16 * U;
  // Keys pass the caches (2: non-temporal), values and scales do not: a row of values is read by four instructions, rows of
  // scales lie in a line with their neighbours'.  32 requests of 131072 tokens: keys through the caches 85.6 us, values past them
  // too 81.4, so 75.9 (one request of 60000 of d 64: 24.4, 25.9, 25.7).
  static constexpr int kPolicyK = 2, kPolicyV = 0, kPolicyS = 0;
  static constexpr int kCodes = D / 2, kScales = 4 * (D / G);   // bytes of a row
  static constexpr int H = D / 64;                  // half-words of a piece
  static constexpr int NG = D / G;                  // groups of a row
  static constexpr int N = D / 16;                  // second products for 32 keys
  static constexpr int QP = sizeof(T) == 2 ? 1 : 3, PP = sizeof(T) == 2 ? 2 : 3;   // bf16 parts of q, of the weights
  static constexpr int VW = D == 256 ? 2 : 1;       // dwords of a piece (d 64: half of one)
  f32x4 acc[N];                                     // acc[4 h + j][r]: row n of q's columns, element d_of(4 h + j, 4 g + r)
  float accb[NG];                                   // this lane's keys only, as l
  float m, l, most;                                 // most: the largest q . k, unscaled; m: what the sums refer to
  u32x4 q[J][QP][D / 32];
  float qs[NG];                                     // sums of q over a group, in the scores' unit
  float unit;                                       // what a score counts
  struct Tile {                                     // a tile as it lies
    Words<2 * H> k[U];
    Words<NG> ks[A], vs[A];
    Words<VW> v[4 * U];
  };
  uint32_t mine[J];                           // mine[j]: all bits in the lanes of block j

  static __device__ __forceinline__ int group_of(int i) { return G == 64 ? i / 4 : 2 * (i / 4) + (i % 4) / 2; }
  // element of acc[i] at row m of the product
  static __device__ __forceinline__ int d_of(int i, int m) {
    return G == 64 ? 64 * (i / 4) + 4 * m + i % 4 : 32 * group_of(i) + 2 * m + i % 2;
  }
  __device__ __forceinline__ void clear(int n) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NG; ++i) accb[i] = 0.f;
    m = most = -INFINITY;
    l = 0.f;
    unit = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) mine[j] = n / C == j ? ~0u : 0u;
  }
  // A row of q as it lies: a quarter of each group.
  static constexpr int kVec = 16 / sizeof(T);
  typedef T QVec __attribute__((ext_vector_type(kVec)));
  struct QRow {
    QVec x[NG][G / 4 / kVec];
  };
  static __device__ __forceinline__ void fetch_q(QRow& q, const T* row, int g) {
#pragma unroll
    for (int b = 0; b < NG; ++b)
#pragma unroll
      for (int i = 0; i < G / 4 / kVec; ++i) q.x[b][i] = *reinterpret_cast<const QVec*>(row + G * b + G / 4 * g + kVec * i);
  }
  // q times `sign` (nothing where it is not `there`), in the codes' order.  `size`: the scale's size, times log2 e.
  __device__ __forceinline__ void take_q(const QRow& raw, bool there, int n, float sign, float size) {
    constexpr int E = G / 4;
    float x[NG][E], most = 0.f;
#pragma unroll
    for (int b = 0; b < NG; ++b) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        x[b][i] = there ? to_f32(raw.x[b][i / kVec][i % kVec]) * sign : 0.f;
        most = fmaxf(most, fabsf(x[b][i]));
        sum += x[b][i];
      }
      qs[b] = col_sum4(sum);
    }
    // q f against codes c 2^-130, f the power of two that takes the row's largest to [2^110, 2^111) (at most 2^124): sums are of
    // ordinary size.  (An infinity or NaN in q makes the unit, and with it every weight, NaN.  The unit is finite while the
    // largest of |q| times the scale is below 2^107.)
    most = col_max4(most);
    const int e = (int)(__float_as_uint(most) >> 23);
    const float f = __uint_as_float((uint32_t)(e < 113 ? 251 : 364 - e) << 23);
    unit = size * (0x1p65f / f) * 0x1p65f;
#pragma unroll
    for (int b = 0; b < NG; ++b) {
      unit += qs[b] - qs[b];
      qs[b] = qs[b] * f * 0x1p-65f * 0x1p-65f;
#pragma unroll
      for (int i = 0; i < E; ++i)                   // (codes number 0 are an eighth)
        x[b][i] *= (G == 64 ? i % 4 == 0 : (b | i) % 2 == 0) ? 8.f * f : f;
    }
#pragma unroll
    for (int b = 0; b < NG; ++b)
#pragma unroll
      for (int part = 0; part < QP; ++part) {
        uint32_t w[E / 2];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          // G 64: product i / 4, word j = i % 4: elements 8 (i / 4) + j and 4 further;
          // G 32: word i = 2 p + j: elements 4 p + j and 2 further
          const int e = G == 64 ? 8 * (i / 4) + i % 4 : 4 * (i / 2) + i % 2, f = e + (G == 64 ? 4 : 2);
          w[i] = pack_bf16(x[b][e], x[b][f]);
          if (part + 1 < QP) {
            x[b][e] -= lo_f(w[i]);
            x[b][f] -= hi_f(w[i]);
          }
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < E / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) q[j][part][b * (E / 8) + i][e] = w[4 * i + e] & mine[j];
      }
  }
  // subtile of this lane's results a
  static __device__ __forceinline__ int subtile(int a, int n) { return a * J + n / C; }
  // The key of a subtile in row n of the first product: results r of lane g are of keys 4 r + g then, and an instruction
  // takes four rows of v that follow each other.
  static __device__ __forceinline__ int key_of(int n) { return 4 * (n & 3) + (n >> 2); }
  // A tile inside one page.  Codes of k: key_of(n), its pieces 4 g and on; of v: keys 4 r + g, piece n; scales: of the
  // keys 4 (n & 3) + g of this lane's subtiles.
  static __device__ __forceinline__ void load_k(Tile& x, const Q4Ptr& p, const Rows& codes, const Rows& scales, int n, int g) {
#pragma unroll
    for (int u = 0; u < U; ++u) x.k[u].template load<kPolicyK>(codes, key_of(n) * p.kc.row_bytes + (D / 8) * g, 16 * u * p.kc.row_bytes);
#pragma unroll
    for (int a = 0; a < A; ++a)
      x.ks[a].template load<kPolicyS>(scales, (16 * (n / C) + 4 * (n & 3) + g) * p.ks.row_bytes, 16 * a * J * p.ks.row_bytes);
  }
  static __device__ __forceinline__ void load_v(Tile& x, const Q4Ptr& p, const Rows& codes, const Rows& scales, int n, int g) {
#pragma unroll
    for (int i = 0; i < 4 * U; ++i) load_v_row(x.v[i], p, codes, (16 * (i >> 2) + 4 * (i & 3)) * p.vc.row_bytes, n, g);
#pragma unroll
    for (int a = 0; a < A; ++a)
      x.vs[a].template load<kPolicyS>(scales, (16 * (n / C) + 4 * (n & 3) + g) * p.vs.row_bytes, 16 * a * J * p.vs.row_bytes);
  }
  static __device__ __forceinline__ void load_v_row(Words<VW>& v, const Q4Ptr& p, const Rows& codes, int at, int n, int g) {
    const int lane_at = g * p.vc.row_bytes + (D / 32) * n;
    if constexpr (D == 64) v.w[0] = __builtin_amdgcn_raw_buffer_load_b16(codes.page, lane_at, codes.at + at, kPolicyV);
    else v.template load<kPolicyV>(codes, lane_at, at);
  }
  // A tile over several pages: subtile by subtile, and for the scales the address of a lane's block by masks.
  __device__ __forceinline__ void load_k(Tile& x, const RunArgs& a, const Q4Ptr& p, const int (&id)[U], int kvh, int first, int n,
                                         int g) const {
    const int size = 1 << a.shift;
#pragma unroll
    for (int u = 0; u < U; ++u)
      x.k[u].template load<kPolicyK>(page_rows(p.kc, id[u], kvh, (first + 16 * u) & (size - 1), size, D / 2), key_of(n) * p.kc.row_bytes + (D / 8) * g, 0);
    load_scales(x.ks, p.ks, id, kvh, first, size, n, g);
  }
  __device__ __forceinline__ void load_v(Tile& x, const RunArgs& a, const Q4Ptr& p, const int (&id)[U], int kvh, int first, int n,
                                         int g) const {
    const int size = 1 << a.shift;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Rows codes = page_rows(p.vc, id[u], kvh, (first + 16 * u) & (size - 1), size, D / 2);
#pragma unroll
      for (int r = 0; r < 4; ++r) load_v_row(x.v[4 * u + r], p, codes, 4 * r * p.vc.row_bytes, n, g);
    }
    load_scales(x.vs, p.vs, id, kvh, first, size, n, g);
  }
  __device__ __forceinline__ void load_scales(Words<NG> (&s)[A], const PagePtr& p, const int (&id)[U], int kvh, int first, int size,
                                              int n, int g) const {
#pragma unroll
    for (int a = 0; a < A; ++a) {
      uint32_t lo = 0, hi = 0;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint64_t x = reinterpret_cast<uint64_t>(p.row(id[a * J + j], kvh, (first + 16 * (a * J + j)) & (size - 1)));
        lo |= (uint32_t)x & mine[j];
        hi |= (uint32_t)(x >> 32) & mine[j];
      }
      s[a].load(((uint64_t)hi << 32 | lo) + (uint32_t)((4 * (n & 3) + g) * p.row_bytes));
    }
  }
  static __device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b, int h) {   // half-word h of a and of b
    return __builtin_amdgcn_perm(b, a, h & 1 ? 0x07060302u : 0x05040100u);
  }
  // s[4 a + r] = q . k of key 16 subtile(a) + 4 r + g, in the row's unit
  __device__ __forceinline__ void scores(const Tile& in, float (&s)[4 * A]) const {
#pragma unroll
    for (int a = 0; a < A; ++a) {
      f32x4 c[NG];
#pragma unroll
      for (int b = 0; b < NG; ++b) c[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const Words<2 * H>& x = in.k[a * J + j];
#pragma unroll
        for (int h = 0; h < H; ++h) {
          u32x4 y[2];                               // G 64: products of group h; G 32: of groups 2 h and 2 h + 1
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            uint32_t r;                             // half-words h of pieces 4 g + 2 p and the next
            if constexpr (H == 1) r = x.w[p];
            else if constexpr (H == 2) r = halves(x.w[2 * p], x.w[2 * p + 1], h);
            else r = halves(x.w[4 * p + (h >> 1)], x.w[4 * p + 2 + (h >> 1)], h);
            if constexpr (G == 64) {
              y[p] = u32x4{codes_of<0>(r), codes_of<1>(r), codes_of<2>(r), codes_of<3>(r)};
            } else {
              y[0][2 * p] = codes_of<0>(r);
              y[0][2 * p + 1] = codes_of<1>(r);
              y[1][2 * p] = codes_of<2>(r);
              y[1][2 * p + 1] = codes_of<3>(r);
            }
          }
#pragma unroll
          for (int i = QP - 1; i >= 0; --i)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              f32x4& to = c[G == 64 ? h : 2 * h + p];
              to = mfma(y[p], q[j][i][2 * h + p], to);
            }
        }
      }
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < NG; ++b) {
        const float sc = lo_f(in.ks[a].w[b]), bias = hi_f(in.ks[a].w[b]);
        t[0] = fmaf(of_four<0>(sc), c[b][0], fmaf(of_four<0>(bias), qs[b], t[0]));
        t[1] = fmaf(of_four<1>(sc), c[b][1], fmaf(of_four<1>(bias), qs[b], t[1]));
        t[2] = fmaf(of_four<2>(sc), c[b][2], fmaf(of_four<2>(bias), qs[b], t[2]));
        t[3] = fmaf(of_four<3>(sc), c[b][3], fmaf(of_four<3>(bias), qs[b], t[3]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * a + i] = t[i];
    }
  }
  // The sums with the largest score as their reference.
  __device__ __forceinline__ void settle() {
    const float f = most == m ? 1.f : __builtin_amdgcn_exp2f((m - most) * unit);
    l *= f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= f;
#pragma unroll
    for (int i = 0; i < NG; ++i) accb[i] *= f;
    m = most;
  }
  // Leaves out the keys outside [lo, n) of the tile that begins at `first`: scores of -inf, scales of zero.
  static __device__ __forceinline__ void cut(Tile& in, float (&s)[4 * A], unsigned first, unsigned lo, unsigned end, int n, int g) {
#pragma unroll
    for (int a = 0; a < A; ++a) {
      const unsigned at = first + 16 * subtile(a, n) + g;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (at + 4 * r < lo || at + 4 * r >= end) s[4 * a + r] = -INFINITY;
      if (at + 4 * (n & 3) < lo || at + 4 * (n & 3) >= end) {
#pragma unroll
        for (int b = 0; b < NG; ++b) in.vs[a].w[b] = 0;
      }
    }
  }
  __device__ __forceinline__ void add(const Tile& in, const float (&p)[4 * A]) {
#pragma unroll
    for (int b = 0; b < NG; ++b) {
      uint32_t part[PP][2 * A];                     // the weights of this lane's keys for the group
#pragma unroll
      for (int a = 0; a < A; ++a) {
        const float sc = lo_f(in.vs[a].w[b]) * kQ4Up, bias = hi_f(in.vs[a].w[b]);
        float w[4];
        w[0] = p[4 * a + 0] * of_four<0>(sc);
        w[1] = p[4 * a + 1] * of_four<1>(sc);
        w[2] = p[4 * a + 2] * of_four<2>(sc);
        w[3] = p[4 * a + 3] * of_four<3>(sc);
        // (four keys' sum first: the long one is rounded once for them)
        const float some = fmaf(p[4 * a + 3], of_four<3>(bias), fmaf(p[4 * a + 2], of_four<2>(bias),
                                                                     fmaf(p[4 * a + 1], of_four<1>(bias), p[4 * a] * of_four<0>(bias))));
        accb[b] += some;
#pragma unroll
        for (int i = 0; i < PP; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = pack_bf16(w[2 * j], w[2 * j + 1]);
            part[i][2 * a + j] = x;
            if (i + 1 < PP) {
              w[2 * j] -= lo_f(x);
              w[2 * j + 1] -= hi_f(x);
            }
          }
      }
      // G 64: half-word b, its four codes; G 32: two of half-word b / 2
      const int h = G == 64 ? b : b >> 1;
#pragma unroll
      for (int e = 0; e < U / 2; ++e) {             // 32 keys: subtiles 2 e and 2 e + 1
        u32x4 w[PP];
#pragma unroll
        for (int i = 0; i < PP; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int u = 2 * e + (j >> 1);
            w[i][j] = part[i][2 * (u / J) + (j & 1)];
            if constexpr (J > 1) w[i][j] &= mine[u % J];
          }
        uint32_t r[4];                              // half-words h of the keys 2 j and 2 j + 1
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Words<VW>&x = in.v[8 * e + 2 * j], &y = in.v[8 * e + 2 * j + 1];
          if constexpr (D == 64) r[j] = x.w[0] | y.w[0] << 16;
          else r[j] = halves(x.w[h >> 1], y.w[h >> 1], h);
        }
        const auto product = [&](auto jc) __attribute__((always_inline)) {
          constexpr int K = decltype(jc)::value;
          // (fp32: the long sum is rounded once for 32 keys, not at each part)
          f32x4 sum = PP == 3 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[4 * h + K];
          const u32x4 x = {codes_of<K>(r[0]), codes_of<K>(r[1]), codes_of<K>(r[2]), codes_of<K>(r[3])};
#pragma unroll
          for (int i = PP - 1; i >= 0; --i) sum = mfma(x, w[i], sum);
          if constexpr (PP == 3) acc[4 * h + K] += sum;
          else acc[4 * h + K] = sum;
        };
        using std::integral_constant;
        if (G == 64 || !(b & 1)) {
          product(integral_constant<int, 0>{});
          product(integral_constant<int, 1>{});
        }
        if (G == 64 || (b & 1)) {
          product(integral_constant<int, 2>{});
          product(integral_constant<int, 3>{});
        }
      }
    }
  }
};

// Tiles t, t + kWaves, ... below t_end.  Returns whether a page id was outside the pages.  The next tile's keys are requested
// once this one's scores are done and its values at the end, the page ids of the one behind it after them.  (Two tiles in
// registers, the next one requested whole before: level, 73 us for 32 requests of up to 131072 tokens either way.)
template <typename S, typename T>
__device__ __forceinline__ bool q4_sweep(const Q4AttnArgs& a, S& w, const int32_t* row, const Span& s, int kvh, int t, int t_end,
                                         const T* q, bool there, float sign, float unit) {
  constexpr int KT = S::KT, U = S::U;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  w.clear(n);
  if (t >= t_end) return false;
  const int size = 1 << a.shift;
  const bool whole = size >= KT;                    // a tile lies inside one page
  int id[U];
  bool bad = false;
  const auto ids = [&](int first) __attribute__((always_inline)) {
    if (whole) id[0] = row[(unsigned)first >> a.shift];
    else tile_ids<U>(a, row, first, s, id);
  };
  const auto check = [&]() __attribute__((always_inline)) {
    if (whole) {
      if ((unsigned)id[0] >= (unsigned)a.num_pages) {
        bad = true;
        id[0] = 0;
      }
    } else {
      bad |= tile_bad<U>(a, id);
    }
  };
  const auto load_k = [&](typename S::Tile& x, int first) __attribute__((always_inline)) {
    const int at = first & (size - 1);
    if (whole) w.load_k(x, a.p, page_rows(a.p.kc, id[0], kvh, at, size, S::kCodes), page_rows(a.p.ks, id[0], kvh, at, size, S::kScales), n, g);
    else w.load_k(x, a, a.p, id, kvh, first, n, g);
  };
  const auto load_v = [&](typename S::Tile& x, int first) __attribute__((always_inline)) {
    const int at = first & (size - 1);
    if (whole) w.load_v(x, a.p, page_rows(a.p.vc, id[0], kvh, at, size, S::kCodes), page_rows(a.p.vs, id[0], kvh, at, size, S::kScales), n, g);
    else w.load_v(x, a, a.p, id, kvh, first, n, g);
  };
  typename S::Tile x;
  // one tile, the next one's requests; whether there is another
  const auto step = [&]() __attribute__((always_inline)) {
    const int next = t + kWaves;
    const bool more = next < t_end;
    if (more) check();
    float p[4 * S::A];
    w.scores(x, p);
    if (more) load_k(x, next * KT);
    const unsigned first = (unsigned)t * KT, lo = s.lo, end = s.n;
    if (first < lo || first + KT > end) w.cut(x, p, first, lo, end, n, g);
    float mx = p[0];
#pragma unroll
    for (int i = 1; i < 4 * S::A; ++i) mx = fmaxf(mx, p[i]);
    mx = col_max4(mx);
    w.most = fmaxf(w.most, mx);
    // (not `> kQ4Lag`: a unit of NaN, or one of 0 on the first maximum, goes the careful way)
    if (__any(mx > w.m && !((mx - w.m) * w.unit <= kQ4Lag))) {
      const float nm = fmaxf(w.m, mx);
      const float f = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((w.m - nm) * w.unit);
      w.l *= f;
#pragma unroll
      for (int i = 0; i < S::N; ++i) w.acc[i] *= f;
#pragma unroll
      for (int i = 0; i < S::NG; ++i) w.accb[i] *= f;
      w.m = nm;
    }
    const float ref = w.m == -INFINITY ? 0.f : w.m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * S::A; ++i) {
      p[i] = __builtin_amdgcn_exp2f((p[i] - ref) * w.unit);
      sum += p[i];
    }
    w.l += sum;
    w.add(x, p);
    if (more) {
      load_v(x, next * KT);
      if (next + kWaves < t_end) ids((next + kWaves) * KT);
    }
    t = next;
    return more;
  };
  typename S::QRow raw;                             // (before the tile: loads return in order)
  S::fetch_q(raw, q, g);
  ids(t * KT);
  check();
  load_k(x, t * KT);
  load_v(x, t * KT);
  if (t + kWaves < t_end) ids((t + kWaves) * KT);
  w.take_q(raw, there, n, sign, unit);
  while (step()) {
  }
  w.settle();
  return bad;
}

// Waves of a SIMD that the registers are cut for: two need no more than 256 (and no moves to accumulation registers
// and back), but for the widest rows.  (Those in groups of 32 with one block of columns spill all the same: 5 registers in bf16, 3
// in fp32.)
constexpr int q4_waves(int esize, int d, int g, int j) { return d < 256 || (esize == 2 && g == 64 && j == 2) ? 2 : 1; }

template <typename T, int D, int G, int J>
__global__ void __launch_bounds__(64 * kWaves, q4_waves(sizeof(T), D, G, J)) q4_attn_kernel(Q4AttnArgs a) {
  typedef Q4Sweep<T, D, G, J> S;
  constexpr int KT = S::KT, C = S::C, LD = D + 4;
  __shared__ float so[kWaves][16 * LD];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ int sbad;
  const Run run = plan_run<KT, true>(a, blockIdx.x);
  if (run.b < 0) return;
  // (every store comes after the last page id is read, as in paged_attn_kernel)
  const auto leave = [&]() {
    if (blockIdx.x == 0 && threadIdx.x == 0 && !a.direct) *a.joins = run.joins;
  };
  const int b = __builtin_amdgcn_readfirstlane(run.b), splits = __builtin_amdgcn_readfirstlane(run.splits);
  const int sub = __builtin_amdgcn_readfirstlane(run.sub), slot = __builtin_amdgcn_readfirstlane(run.slot) + sub;
  const int unit = sub / splits, split = sub - unit * splits;
  const int kvh = unit / a.row_tiles, part = unit - kvh * a.row_tiles;
  const int rows = a.group - 16 * part < 16 ? a.group - 16 * part : 16;   // (at most C: there are more than C with J = 1 only)
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
  // scores stay q . k up to the exponential; a scale below zero turns q over, one of zero clears it
  const float sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : a.scale, size = a.scale == 0.f ? 1.f : fabsf(a.scale);
  S w;
  const bool there = n % C < rows;                  // (a column without a row of q reads the first one's)
  const T* q = reinterpret_cast<const T*>(a.q + b * a.q_req + (int64_t)(head0 + (there ? n % C : 0)) * a.q_head);
  const bool bad = q4_sweep<S>(a, w, table, s, kvh, t0 + wave, t1, q, there, sign, size * kLog2e);
  const float l = col_sum4(w.l);
  float accb[S::NG];
#pragma unroll
  for (int i = 0; i < S::NG; ++i) accb[i] = col_sum4(w.accb[i]);
  __syncthreads();
  if (n % C < rows) {
#pragma unroll
    for (int i = 0; i < S::N; i += G / 16)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float bias = accb[w.group_of(i)], c0 = 0x1p93f, c = 0x1p90f;   // (2^133 and 2^130 / kQ4Up)
        float* to = &so[wave][n * LD + w.d_of(i, 4 * g + r)];
        if constexpr (G == 64)
          *reinterpret_cast<f32x4*>(to) = f32x4{fmaf(w.acc[i][r], c0, bias), fmaf(w.acc[i + 1][r], c, bias),
                                                fmaf(w.acc[i + 2][r], c, bias), fmaf(w.acc[i + 3][r], c, bias)};
        else
          *reinterpret_cast<f32x2*>(to) = f32x2{fmaf(w.acc[i][r], i % 4 == 0 ? c0 : c, bias), fmaf(w.acc[i + 1][r], c, bias)};
      }
    if (g == 0) {
      sm[wave][n] = w.m == -INFINITY ? w.m : w.m * (w.unit * 0.6931471805599453f);   // (a wave without tiles has no unit)
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
    for (int k = 1; k < kWaves * J; ++k) mm = fmaxf(mm, sm[k / J][k % J * C + r]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    float ll = poison;
#pragma unroll
    for (int k = 0; k < kWaves * J; ++k) {
      const int col = k % J * C + r;
      const float f = __builtin_amdgcn_exp2f((sm[k / J][col] - ref) * kLog2e);
      // a wave without tiles has no part in it (0 * its sums would do, but for a reference of +inf)
      if (t0 + k / J < t1) {
        ll += f * sl[k / J][col];
        y += f * *reinterpret_cast<const f32x4*>(&so[k / J][col * LD + c]);
      }
    }
    if (splits == 1) {
      store4(static_cast<T*>(a.out) + (row0 + r) * D + c, y, 1.f / ll);
      if (c == 0) finish_stats<T>(a, row0 + r, mm, ll);
    } else {
      const int64_t at = (int64_t)slot * a.rows + r;
      *reinterpret_cast<f32x4*>(a.part + at * D + c) = y;
      if (c == 0) reinterpret_cast<f32x2*>(a.part_ml)[at] = f32x2{mm, ll};
    }
  }
}

// Blocks of columns: as many as leave room for a unit's rows of q, and as the copies of q leave registers for; one where
// all requests together have few keys (their tables' widths; a window) and what counts is how soon the first results are there.
// Measured, us, one / two / these: 32 requests of 131072 tokens 101 / 88 / 76, one of 32768 15.8 / 15.3 / 13.9, 16 of 1024 and 4 kv
// heads (2^16 keys) 11.9 / 11.7 / 11.9; one of 8192 (2^15) 10.6 / 10.7 / 11.6, of 1024 10.2 / 10.3 / 11.6.
constexpr int q4_most_blocks(int esize, int head_dim) {
  return esize == 2 ? (head_dim <= 128 ? 4 : 2) : head_dim == 64 ? 4 : head_dim == 128 ? 2 : 1;
}
static int q4_blocks(int esize, int64_t head_dim, int64_t group, int64_t pairs, int64_t tokens, int64_t window) {
  const int most = q4_most_blocks(esize, (int)head_dim), fit = group <= 4 ? 4 : group <= 8 ? 2 : 1;
  if (window > 0 && window < tokens) tokens = window;
  return tokens < (1 << 16) && pairs * tokens < (1 << 16) ? 1 : most < fit ? most : fit;
}
static int q4_tile(int blocks) { return blocks > 2 ? 64 : 32; }
// Runs in all, where requests and heads leave them: as many workgroups of a CU as waves of a SIMD that the registers are cut
// for (bf16 rows of 64 would leave room for four).  Measured, us, half as many / these: 32 requests of up to 131072 tokens
// 90 / 73, one of 262144 of d 256 66 / 62, 8 of 60000 of d 64 29 / 26; twice as many: 90, 80, 24.  Fewer runs
// of two rounds before as many of one: one request of 32768 tokens 15.8 -> 14.0.
static int q4_runs(int esize, int64_t head_dim, int64_t group, int blocks) {
  return 256 * q4_waves(esize, (int)head_dim, (int)group, blocks);
}
static_assert(256 * 2 <= kMaxRuns, "");

template <typename T, int D, int G>
static void launch_q4(const Q4AttnArgs& a, int blocks, int64_t items, hipStream_t stream) {
  const dim3 grid((unsigned)items), block(64 * kWaves);
  if constexpr (q4_most_blocks(sizeof(T), D) >= 4) {
    if (blocks == 4) {
      hipLaunchKernelGGL((q4_attn_kernel<T, D, G, 4>), grid, block, 0, stream, a);
      return;
    }
  }
  if constexpr (q4_most_blocks(sizeof(T), D) >= 2) {
    if (blocks == 2) {
      hipLaunchKernelGGL((q4_attn_kernel<T, D, G, 2>), grid, block, 0, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((q4_attn_kernel<T, D, G, 1>), grid, block, 0, stream, a);
}

}  // namespace bfly

using namespace bfly;

extern "C" int64_t bfly_paged_q4_attention_workspace_bytes(int dtype, int64_t requests, int hq, int hkv, int head_dim,
                                                           int64_t table_width, int page_size, int window) {
  if (requests <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || head_dim <= 0 || table_width <= 0 || page_size <= 0) return 0;
  const int64_t group = hq / hkv, rows = group < 16 ? group : 16;
  const int64_t pairs = requests * hkv * ((group + 15) / 16);
  const int tile = q4_tile(q4_blocks(dtype == BFLY_DTYPE_F32 ? 4 : 2, head_dim, group, pairs, table_width * page_size, window));
  return most_rounds(table_width * page_size, window, tile) <= q4_whole_rounds(pairs) ? 0 : run_workspace_bytes(rows, head_dim);
}

extern "C" int bfly_paged_q4_attention(const bfly_paged_q4_attention_args_t* args, hipStream_t stream) {
  BFLY_CHECK_ARG(args, "null pointer");
  const bfly_paged_q4_attention_args_t& x = *args;
  BFLY_CHECK_ARG(x.dtype == BFLY_DTYPE_F32 || x.dtype == BFLY_DTYPE_BF16, "unsupported dtype %lld", (long long)x.dtype);
  const int64_t es = x.dtype == BFLY_DTYPE_F32 ? 4 : 2;
  BFLY_CHECK_ARG(x.requests >= 0 && x.requests <= 65535, "bad number of requests (at most 65535)");
  BFLY_CHECK_ARG(x.hkv > 0 && x.hq > 0 && x.hq <= (1 << 20) && x.hkv <= x.hq && x.hq % x.hkv == 0,
                 "bad head counts hq=%lld hkv=%lld", (long long)x.hq, (long long)x.hkv);
  const int rc = q4_check_pages("bfly_paged_q4_attention", x.pages, x.head_dim);
  if (rc != BFLY_OK) return rc;
  BFLY_CHECK_ARG(x.window >= 0 && x.window <= INT32_MAX, "bad window");
  BFLY_CHECK_ARG(x.table_width >= 0 && x.table_width <= INT32_MAX && (x.requests <= 1 || x.table_stride >= 0),
                 "bad block table shape");
  BFLY_CHECK_ARG(x.q_request_stride >= 0 && x.q_head_stride >= 0 && x.q_request_stride < ((int64_t)1 << 48) &&
                     x.q_head_stride < ((int64_t)1 << 48) && x.q_request_stride * es % 16 == 0 &&
                     x.q_head_stride * es % 16 == 0,
                 "q strides must be multiples of 16 bytes");
  if (x.requests == 0) return BFLY_OK;
  BFLY_CHECK_ARG(x.q && x.lengths && x.out && q4_given(x.pages), "null pointer");
  BFLY_CHECK_ARG(x.table_width == 0 || x.block_table, "null pointer");
  BFLY_CHECK_ARG((x.l == nullptr) == (x.m == nullptr), "both l and m or neither");
  BFLY_CHECK_ARG(aligned16(x.q) && aligned16(x.out) && q4_aligned(x.pages), "pointers must be 16-byte aligned");
  const int64_t need = bfly_paged_q4_attention_workspace_bytes((int)x.dtype, x.requests, (int)x.hq, (int)x.hkv, (int)x.head_dim,
                                                               x.table_width, (int)x.pages.page_size, (int)x.window);
  BFLY_CHECK_ARG(need == 0 || (x.workspace && x.workspace_bytes >= need && aligned16(x.workspace)), "workspace too small");
  Q4AttnArgs a{};
  a.q = static_cast<const char*>(x.q);
  a.p = q4_ptr(x.pages);
  a.table = x.block_table; a.lengths = x.lengths; a.out = x.out; a.l = x.l; a.m = x.m;
  a.q_req = x.q_request_stride * es; a.q_head = x.q_head_stride * es; a.scale = (float)x.scale;
  BFLY_CHECK_ARG(run_shape(a, x.requests, x.hq, x.hkv, x.pages.page_size, x.pages.num_pages, x.table_width, x.table_stride,
                           x.window),
                 "too many heads");
  run_workspace(a, x.workspace, x.head_dim);
  a.whole = q4_whole_rounds((int64_t)a.requests * a.units);
  const int blocks = q4_blocks((int)es, x.head_dim, a.group, (int64_t)a.requests * a.units, x.table_width * x.pages.page_size, x.window);
  a.runs = q4_runs((int)es, x.head_dim, x.pages.group, blocks);
  const int64_t items = run_items(a, most_rounds(a.capacity, a.window, q4_tile(blocks)));
  BFLY_CHECK_ARG(items < (1 << 24), "too many requests and heads");   // a grid holds fewer than 2^32 threads
#define BFLY_Q4(T, D, G) launch_q4<T, D, G>(a, blocks, items, stream)
#define BFLY_Q4_G(T, D)                       \
  do {                                        \
    if (x.pages.group == 32) BFLY_Q4(T, D, 32); \
    else BFLY_Q4(T, D, 64);                   \
  } while (0)
#define BFLY_Q4_D(T)                         \
  do {                                       \
    if (x.head_dim == 64) BFLY_Q4_G(T, 64);  \
    else if (x.head_dim == 128) BFLY_Q4_G(T, 128); \
    else BFLY_Q4_G(T, 256);                  \
  } while (0)
  if (x.dtype == BFLY_DTYPE_BF16) BFLY_Q4_D(__bf16);
  else BFLY_Q4_D(float);
#undef BFLY_Q4_D
#undef BFLY_Q4_G
#undef BFLY_Q4
  paged_merge(a, (int)x.dtype, (int)x.head_dim, stream);
  BFLY_CHECK_LAUNCH("bfly_paged_q4_attention");
  return BFLY_OK;
}
