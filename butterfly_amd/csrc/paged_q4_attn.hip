// One new token of every request over its 4-bit pages (include/butterfly_amd_paged_q4.h).
//
//   k_t = c_t s_t + b_t for each group of elements (codes c, scale s, bias b), v_t likewise;
//   s_t = scale q . k_t = scale sum_groups (s_t (q . c_t) + b_t sum q),   m = max s_t, l = sum exp(s_t - m),
//   o = (sum exp(s_t - m) v_t) / l,  v's scales and biases on the weights: sum (p_t s_t) c_t + sum p_t b_t.
//
// The schedule, runs and joins are those of paged_attn.hip (paged_runs.h).  Inside a tile of 32 keys the two products
// run over the codes themselves: a code is exact in bf16 (as 16 + c: two operations for two codes, an operand word
// is ((w >> n) & 0x00780078) | 0x41804180), so nothing is rounded on the way from the cache to the sums but the weights, which
// enter as two bf16 parts (three, and q as three, for fp32).
//   * A row's 16 pieces hold a sixteenth of every group each.  S^T = K Q^T: lane (n, g) takes four pieces of key n
//     (a quarter of every group), so each product is over one group.  O^T += V^T P^T: lane n takes piece n of a lane's 8
//     keys, so the 16 rows of each product are of one group, and P carries that group's scale.
//   * Scales are read as lane (n, g) needs them, for keys 4g + (n & 3), and reach the other lanes of a four by DPP.
#include "paged_runs.h"
#include "paged_q4.h"

namespace bfly {

constexpr int kQ4Tile = 32;
constexpr int q4_runs_for(int) { return 512; }   // in all, where requests and heads leave them
static_assert(q4_runs_for(64) <= kMaxRuns, "");
constexpr int q4_whole_rounds(int64_t pairs) { return pairs >= 2048 ? 32 : pairs >= 512 ? 16 : pairs >= 128 ? 8 : 4; }

struct Q4AttnArgs : RunArgs {
  const char* q;
  Q4Ptr p;
  int64_t q_req, q_head;                 // bytes
};

// lane (n & ~3) + R's x
template <int R>
__device__ __forceinline__ float of_four(float x) {
  constexpr int ctrl = R | R << 2 | R << 4 | R << 6;
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xf, 0xf, false));
}
// codes number j of both half-words of r as 16 + c in bf16
template <int J>
__device__ __forceinline__ uint32_t codes_of(uint32_t r) {
  const uint32_t x = J == 0 ? r << 3 : r >> (4 * J - 3);
  return (x & 0x00780078u) | 0x41804180u;
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

template <int N>
struct Words {                                      // N dwords (or a half-word: N = 0) as they lie
  uint32_t w[N];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = x[j];
      }
    } else if constexpr (N == 2) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      w[0] = x[0];
      w[1] = x[1];
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
};

// One wave's sums over its tiles.  acc[4 h + j][r] of lane (n = lane & 15, g = lane >> 4): query row n, element
// d_of(4 h + j, 4 g + r).
template <typename T, int D, int G>
struct Q4Sweep {
  static constexpr int KT = kQ4Tile;
  static constexpr int H = D / 64;                  // half-words of a piece
  static constexpr int NG = D / G;                  // groups of a row
  static constexpr int N = D / 16;                  // second products a tile
  static constexpr int QP = sizeof(T) == 2 ? 1 : 3, PP = sizeof(T) == 2 ? 2 : 3;   // bf16 parts of q, of the weights
  static constexpr int VW = D == 256 ? 2 : 1;       // dwords of a piece (d 64: half of one)
  f32x4 acc[N];
  float accb[NG];                                   // this lane's keys only, as l
  float m, l;                                       // m: the largest q . k, unscaled
  u32x4 q[QP][D / 32];
  float qs[NG];                                     // sums of q over a group
  Words<2 * H> k[2];
  Words<NG> ks[2], vs[2];
  Words<VW> v[8];

  static __device__ __forceinline__ int group_of(int i) { return G == 64 ? i / 4 : 2 * (i / 4) + (i % 4) / 2; }
  // element of acc[i] at row m of the product
  static __device__ __forceinline__ int d_of(int i, int m) {
    return G == 64 ? 64 * (i / 4) + 4 * m + i % 4 : 32 * group_of(i) + 2 * m + i % 2;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NG; ++i) accb[i] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }
  // q times `sign`: a quarter of each group, in the codes' order
  __device__ __forceinline__ void load_q(const T* row, int g, float sign) {
    constexpr int E = G / 4;
#pragma unroll
    for (int b = 0; b < NG; ++b) {
      float x[E], sum = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] = row != nullptr ? to_f32(row[G * b + E * g + e]) * sign : 0.f;
        sum += x[e];
      }
      qs[b] = col_sum4(sum);
#pragma unroll
      for (int part = 0; part < QP; ++part) {
        uint32_t w[E / 2];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          // G 64: product i / 4, word j = i % 4: elements 8 (i / 4) + j and 4 further;
          // G 32: word i = 2 p + j: elements 4 p + j and 2 further
          const int e = G == 64 ? 8 * (i / 4) + i % 4 : 4 * (i / 2) + i % 2, f = e + (G == 64 ? 4 : 2);
          w[i] = pack_bf16(x[e], x[f]);
          x[e] -= lo_f(w[i]);
          x[f] -= hi_f(w[i]);
        }
#pragma unroll
        for (int i = 0; i < E / 8; ++i) q[part][b * (E / 8) + i] = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      }
    }
  }
  __device__ __forceinline__ void load_k(const char* const (&base)[2], const char* const (&sbase)[2], const Q4Ptr& p, int n, int g) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      k[u].load(base[u] + (uint32_t)(n * p.kc.row_bytes + (D / 8) * g));
      ks[u].load(sbase[u] + (uint32_t)((4 * g + (n & 3)) * p.ks.row_bytes));
    }
  }
  __device__ __forceinline__ void load_v(const char* const (&base)[2], const char* const (&sbase)[2], const Q4Ptr& p, int n, int g) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char* at = base[j >> 2] + (uint32_t)((4 * g + (j & 3)) * p.vc.row_bytes + (D / 32) * n);
      if constexpr (D == 64) v[j].w[0] = *reinterpret_cast<const uint16_t*>(at);
      else v[j].load(at);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) vs[u].load(sbase[u] + (uint32_t)((4 * g + (n & 3)) * p.vs.row_bytes));
  }
  static __device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b, int h) {   // half-word h of a and of b
    return __builtin_amdgcn_perm(b, a, h & 1 ? 0x07060302u : 0x05040100u);
  }
  // this lane's keys 16 u + 4 g + r: s[4 u + r] = q . k
  __device__ __forceinline__ void scores(float (&s)[8]) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t r[2][H];                             // r[p][h]: half-words h of pieces 4 g + 2 p and the next
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          if constexpr (H == 1) r[p][h] = k[u].w[p];
          else if constexpr (H == 2) r[p][h] = halves(k[u].w[2 * p], k[u].w[2 * p + 1], h);
          else r[p][h] = halves(k[u].w[4 * p + (h >> 1)], k[u].w[4 * p + 2 + (h >> 1)], h);
        }
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < NG; ++b) {
        f32x4 c = {0.f, 0.f, 0.f, 0.f};
        if constexpr (G == 64) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const u32x4 x = {codes_of<0>(r[p][b]), codes_of<1>(r[p][b]), codes_of<2>(r[p][b]), codes_of<3>(r[p][b])};
#pragma unroll
            for (int i = QP - 1; i >= 0; --i) c = mfma(x, q[i][2 * b + p], c);
          }
        } else {
          const int h = b >> 1;
          const u32x4 x = b & 1 ? u32x4{codes_of<2>(r[0][h]), codes_of<3>(r[0][h]), codes_of<2>(r[1][h]), codes_of<3>(r[1][h])}
                                : u32x4{codes_of<0>(r[0][h]), codes_of<1>(r[0][h]), codes_of<0>(r[1][h]), codes_of<1>(r[1][h])};
#pragma unroll
          for (int i = QP - 1; i >= 0; --i) c = mfma(x, q[i][b], c);
        }
        const float sc = lo_f(ks[u].w[b]), bias = fmaf(-16.f, sc, hi_f(ks[u].w[b]));
        t[0] = fmaf(of_four<0>(sc), c[0], fmaf(of_four<0>(bias), qs[b], t[0]));
        t[1] = fmaf(of_four<1>(sc), c[1], fmaf(of_four<1>(bias), qs[b], t[1]));
        t[2] = fmaf(of_four<2>(sc), c[2], fmaf(of_four<2>(bias), qs[b], t[2]));
        t[3] = fmaf(of_four<3>(sc), c[3], fmaf(of_four<3>(bias), qs[b], t[3]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * u + i] = t[i];
    }
  }
  static __device__ __forceinline__ int key(int i, int g) { return 16 * (i >> 2) + 4 * g + (i & 3); }
  __device__ __forceinline__ void drop_v(int u) {   // the scales that this lane holds for subtile u
#pragma unroll
    for (int b = 0; b < NG; ++b) vs[u].w[b] = 0;
  }
  __device__ __forceinline__ void add(const float (&p)[8]) {
#pragma unroll
    for (int b = 0; b < NG; ++b) {
      float w[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float sc = lo_f(vs[u].w[b]), bias = fmaf(-16.f, sc, hi_f(vs[u].w[b]));
        w[4 * u + 0] = p[4 * u + 0] * of_four<0>(sc);
        w[4 * u + 1] = p[4 * u + 1] * of_four<1>(sc);
        w[4 * u + 2] = p[4 * u + 2] * of_four<2>(sc);
        w[4 * u + 3] = p[4 * u + 3] * of_four<3>(sc);
        accb[b] = fmaf(p[4 * u + 0], of_four<0>(bias), accb[b]);
        accb[b] = fmaf(p[4 * u + 1], of_four<1>(bias), accb[b]);
        accb[b] = fmaf(p[4 * u + 2], of_four<2>(bias), accb[b]);
        accb[b] = fmaf(p[4 * u + 3], of_four<3>(bias), accb[b]);
      }
      u32x4 part[PP];
#pragma unroll
      for (int i = 0; i < PP; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          part[i][j] = pack_bf16(w[2 * j], w[2 * j + 1]);
          if (i + 1 < PP) {
            w[2 * j] -= lo_f(part[i][j]);
            w[2 * j + 1] -= hi_f(part[i][j]);
          }
        }
      // G 64: half-word b, its four codes; G 32: two of half-word b / 2
      const int h = G == 64 ? b : b >> 1;
      uint32_t r[4];                                // half-words h of the keys 2 j and 2 j + 1
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (D == 64) r[j] = v[2 * j].w[0] | v[2 * j + 1].w[0] << 16;
        else r[j] = halves(v[2 * j].w[h >> 1], v[2 * j + 1].w[h >> 1], h);
      }
      const auto product = [&](auto jc) {
        constexpr int J = decltype(jc)::value;
        const u32x4 x = {codes_of<J>(r[0]), codes_of<J>(r[1]), codes_of<J>(r[2]), codes_of<J>(r[3])};
#pragma unroll
        for (int i = PP - 1; i >= 0; --i) acc[4 * h + J] = mfma(x, part[i], acc[4 * h + J]);
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
};

// Tiles t, t + kWaves, ... below t_end.  Returns whether a page id was outside the pages.
template <typename T, int D, int G>
__device__ __forceinline__ bool q4_sweep(const Q4AttnArgs& a, Q4Sweep<T, D, G>& w, const int32_t* row, const Span& s, int kvh,
                                         int t, int t_end, float unit) {
  constexpr int KT = kQ4Tile;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  w.clear();
  if (t >= t_end) return false;
  int id[2];
  const char *base[2], *sbase[2];
  const auto bases = [&](const PagePtr& codes, const PagePtr& scales, int first) {
    tile_base<2>(a, codes, kvh, first, id, base);
    tile_base<2>(a, scales, kvh, first, id, sbase);
  };
  bool bad = tile_pages<2>(a, row, t * KT, s, id);
  bases(a.p.kc, a.p.ks, t * KT);
  w.load_k(base, sbase, a.p, n, g);
  bases(a.p.vc, a.p.vs, t * KT);
  w.load_v(base, sbase, a.p, n, g);
  while (true) {
    const int next = t + kWaves;
    const bool more = next < t_end;
    if (more) bad |= tile_pages<2>(a, row, next * KT, s, id);
    float p[8];
    w.scores(p);
    if (more) {
      bases(a.p.kc, a.p.ks, next * KT);
      w.load_k(base, sbase, a.p, n, g);
    }
    const unsigned first = (unsigned)t * KT, lo = s.lo, end = s.n;
    if (first < lo || first + KT > end) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned at = first + w.key(i, g);
        if (at < lo || at >= end) p[i] = -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned at = first + 16 * u + 4 * g + (n & 3);
        if (at < lo || at >= end) w.drop_v(u);
      }
    }
    float mx = p[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, p[i]);
    mx = col_max4(mx);
    if (__any(mx > w.m)) {
      const float nm = fmaxf(w.m, mx);
      const float f = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((w.m - nm) * unit);
      w.l *= f;
#pragma unroll
      for (int i = 0; i < w.N; ++i) w.acc[i] *= f;
#pragma unroll
      for (int i = 0; i < w.NG; ++i) w.accb[i] *= f;
      w.m = nm;
    }
    const float ref = w.m == -INFINITY ? 0.f : w.m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f((p[i] - ref) * unit);
      sum += p[i];
    }
    w.l += sum;
    w.add(p);
    if (!more) return bad;
    bases(a.p.vc, a.p.vs, next * KT);
    w.load_v(base, sbase, a.p, n, g);
    t = next;
  }
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(64 * kWaves) q4_attn_kernel(Q4AttnArgs a) {
  constexpr int KT = kQ4Tile, LD = D + 4;
  __shared__ float so[kWaves][16 * LD];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ int sbad;
  const Run run = plan_run<KT>(a, blockIdx.x);
  if (run.b < 0) return;
  // (every store comes after the last page id is read, as in paged_attn_kernel)
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
  // scores stay q . k up to the exponential; a scale below zero turns q over, one of zero clears it
  const float sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : a.scale, size = a.scale == 0.f ? 1.f : fabsf(a.scale);
  Q4Sweep<T, D, G> w;
  w.load_q(n < rows ? reinterpret_cast<const T*>(a.q + b * a.q_req + (int64_t)(head0 + n) * a.q_head) : nullptr, g, sign);
  const bool bad = q4_sweep<T, D, G>(a, w, table, s, kvh, t0 + wave, t1, size * kLog2e);
  const float l = col_sum4(w.l);
  float accb[w.NG];
#pragma unroll
  for (int i = 0; i < w.NG; ++i) accb[i] = col_sum4(w.accb[i]);
  __syncthreads();
  if (n < rows) {
#pragma unroll
    for (int i = 0; i < w.N; i += G / 16)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float bias = accb[w.group_of(i)];
        float* to = &so[wave][n * LD + w.d_of(i, 4 * g + r)];
        if constexpr (G == 64)
          *reinterpret_cast<f32x4*>(to) =
              f32x4{w.acc[i][r] + bias, w.acc[i + 1][r] + bias, w.acc[i + 2][r] + bias, w.acc[i + 3][r] + bias};
        else
          *reinterpret_cast<f32x2*>(to) = f32x2{w.acc[i][r] + bias, w.acc[i + 1][r] + bias};
      }
    if (g == 0) {
      sm[wave][n] = w.m * size;
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
      if (c == 0) reinterpret_cast<f32x2*>(a.part_ml)[at] = f32x2{mm, ll};
    }
  }
}

}  // namespace bfly

using namespace bfly;

extern "C" int64_t bfly_paged_q4_attention_workspace_bytes(int64_t requests, int hq, int hkv, int head_dim, int64_t table_width,
                                                           int page_size, int window) {
  if (requests <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || head_dim <= 0 || table_width <= 0 || page_size <= 0) return 0;
  const int64_t group = hq / hkv, rows = group < 16 ? group : 16;
  const int64_t pairs = requests * hkv * ((group + 15) / 16);
  return most_rounds(table_width * page_size, window, kQ4Tile) <= q4_whole_rounds(pairs) ? 0 : run_workspace_bytes(rows, head_dim);
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
  const int64_t need = bfly_paged_q4_attention_workspace_bytes(x.requests, (int)x.hq, (int)x.hkv, (int)x.head_dim, x.table_width,
                                                               (int)x.pages.page_size, (int)x.window);
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
  a.runs = q4_runs_for((int)x.head_dim);
  a.whole = q4_whole_rounds((int64_t)a.requests * a.units);
  const int64_t items = run_items(a, most_rounds(a.capacity, a.window, kQ4Tile));
  BFLY_CHECK_ARG(items < (1 << 24), "too many requests and heads");   // a grid holds fewer than 2^32 threads
#define BFLY_Q4(T, D, G) hipLaunchKernelGGL((q4_attn_kernel<T, D, G>), dim3((unsigned)items), dim3(64 * kWaves), 0, stream, a)
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
