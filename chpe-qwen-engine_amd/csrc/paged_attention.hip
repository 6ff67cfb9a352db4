// paged_attention.hip -- chpe_paged_attention: the attention of one new token per row over the paged
// cache.  s_j = scale q.k_j over the row's slots lo <= j < len, p = softmax(s), out = sum_j p_j v_j, and,
// for a cache that is kept to a budget, each slot's p summed over the query heads of its kv head.
// The slots are split over workgroups: each leaves its maximum, sum of 2^(s - max) and so weighted sum of V
// rows, and a second launch rescales and joins them (and turns the scores into weights).
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace chpe {
namespace {
using namespace dev;

struct PagedAttnArgs {
  Pages c;
  const float* q;
  const int32_t* lens;
  float* out;
  float *part_ml, *part_acc;      // [row][head][split][2], [row][head][split][hd]
  float* scores;                  // [row][head][score_stride] from the range's first slot, or null
  const float* weight_in;
  float* weight_out;
  uint64_t q_stride, out_stride, weight_stride;
  uint32_t rows, H, max_len, window, splits, chunk, score_stride;
  float scale;
};

// the row's slots lo .. len - 1; false for a length outside 0 .. max_len
__device__ __forceinline__ bool row_range(const PagedAttnArgs& a, uint32_t row, uint32_t* lo, uint32_t* len) {
  const uint32_t n = uint32_t(gld(a.lens + row));
  *len = n <= a.max_len ? n : 0u;
  *lo = a.window != 0 && *len > a.window ? *len - a.window : 0u;
  return n <= a.max_len;
}

// ---- the partial sums of one split -----------------------------------------------------------------------
// One workgroup of 4 waves per (row, kv head, group of HT query heads, split); wave w takes the tiles w, w + 4,
// .. of the split.  A tile's scores are S^T = K . Q^T on the matrix cores (rows: slots, columns: query heads),
// its output O^T = V^T . P^T (rows: dims, columns: heads): with the heads as columns of both, a lane (G, n) =
// (lane / 16, lane % 16) keeps the running maximum and sum of column n in scalars of its own, and the result
// layout of the first product (slots 4 G + i of column n) is the operand layout of the second, so the weights
// never leave the registers.  The order of the dims inside the first product and of the slots inside the
// second is free as long as both operands agree, which is what lets every lane load 16 bytes in a row:
// K rows as pieces of 4 x 16 bytes, V rows as 16 lanes x 16 bytes.
// The running maximum is in units of log2 (scores times scale * log2 e).
constexpr int kWaves = 4;
constexpr uint32_t kMaxSplits = 512;
constexpr float kLog2e = 1.4426950408889634f;

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// 16-bit elements with f32 queries and weights: x is taken apart into parts that the products hold exactly,
// part p of head h in column h + p * W of the 16; all columns' results are added at the end (sum_parts), so no
// precision of the f32 queries or weights is lost to the cache's type.  fp16: two parts, 22 bits; x is brought
// near 2^14 by a power of two first, so that the second part does not fall below fp16's range.  bf16: three
// parts, 24 bits; of up to 4 heads they fit the 16 columns, of 8 the third is an operand of its own.
template <class T, int W>
struct Parts;
template <>
struct Parts<_Float16, 8> {
  using Vec = h8_t;
  static constexpr int kOps = 1, kScaleExp = 15;  // (weights <= 1 times 2^15)
  static __device__ void split(const float (&x)[8], int part, Vec (&out)[1]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const _Float16 hi = _Float16(x[e]);
      out[0][e] = part != 0 ? _Float16(x[e] - float(hi)) : hi;
    }
  }
  static __device__ f4_t mfma(Vec a, Vec b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <int W>
struct Parts<Bf16, W> {
  using Vec = b8_t;
  static constexpr int kOps = W == 8 ? 2 : 1, kScaleExp = 0;
  static __device__ void split(const float (&x)[8], int part, Vec (&out)[kOps]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const __bf16 hi = __bf16(x[e]);
      const float r = x[e] - float(hi);
      const __bf16 mid = __bf16(r);
      const __bf16 lo = __bf16(r - float(mid)), zero = __bf16(0.0f);
      out[0][e] = part == 0 ? hi : part == 1 ? mid : part == 2 ? lo : zero;
      if constexpr (W == 8) out[1][e] = part == 0 ? lo : zero;
    }
  }
  static __device__ f4_t mfma(Vec a, Vec b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <int W>
__device__ __forceinline__ float sum_parts(float v) {
  if constexpr (W == 4) v = pair_sum(v, 4);
  return pair_sum(v, 8);
}

// where a workgroup works
struct Place {
  uint32_t row, kvh, h0, nh, begin, end, lo, len, split;  // query heads h0 .. h0 + nh - 1, slots begin .. end - 1
  bool ok;
};
template <int HT>
__device__ __forceinline__ Place place_of(const PagedAttnArgs& a) {
  Place p;
  const uint32_t gq = a.H / a.c.KV, hz = (gq + HT - 1) / HT;
  uint32_t b = blockIdx.x;
  p.split = b % a.splits;
  b /= a.splits;
  const uint32_t z = b % hz;
  b /= hz;
  p.kvh = b % a.c.KV;
  p.row = b / a.c.KV;
  p.h0 = p.kvh * gq + z * HT;
  p.nh = min(uint32_t(HT), gq - z * HT);
  return p;
}
__device__ __forceinline__ void place_slots(const PagedAttnArgs& a, Place* p) {
  p->ok = row_range(a, p->row, &p->lo, &p->len);
  p->begin = p->lo + p->split * a.chunk;
  p->end = min(p->len, p->begin + a.chunk);
}

// The tile's row offsets (bytes from k or v): lane r of the wave finds row r's page and leaves the
// offset in LDS for the lanes that load the row.  `next` requests the table entry ahead of its use; for the
// first tile of a range that starts at slot 0 it does not wait for the row's length (entries behind it may
// hold anything).  Rows behind the split's end are its last row.
template <int ROWS, int ES>
struct TileRows {
  uint64_t (*s)[ROWS];
  uint32_t id = 0, slot = 0;
  bool bad = false;
  __device__ void next(const PagedAttnArgs& a, uint32_t row, uint32_t t, uint32_t last, int lane) {
    slot = min(t + uint32_t(lane % ROWS), last);
    id = uint32_t(gld(a.c.table + size_t(row) * a.c.table_stride + (slot >> a.c.shift)));
  }
  __device__ void put(const PagedAttnArgs& a, const Place& p, int buf, int lane) {
    // a row behind the end, which `next` did not know yet: the last one's, which is in the tile too
    const uint32_t first = __builtin_amdgcn_readfirstlane(slot);
    const uint32_t id_last = uint32_t(__builtin_amdgcn_readlane(int(id), min(p.end - 1 - first, uint32_t(ROWS - 1))));
    if (slot >= p.end) {
      slot = p.end - 1;
      id = id_last;
    }
    const bool in = id < a.c.n_pages;
    bad |= !in;
    if (lane < ROWS) s[buf][lane] = a.c.at(in ? id : 0u, p.kvh, slot) * ES;
    __builtin_amdgcn_wave_barrier();
  }
};

// joins waves 1 .. 3 into wave 0: each lane's maximum, sum and N accumulators, through LDS
template <int N, int LANES>
__device__ __forceinline__ void join_waves(float* s, int wave, int slot, bool mine, float* m, float* l, f4_t* o) {
#pragma unroll
  for (int half = kWaves / 2; half >= 1; half /= 2) {
    __syncthreads();
    if (wave >= half && wave < 2 * half && mine) {
      float* d = s + (wave - half) * (N * 4 + 4) * LANES;
#pragma unroll
      for (int i = 0; i < N; ++i) *reinterpret_cast<f4_t*>(d + (i * LANES + slot) * 4) = o[i];
      d[N * 4 * LANES + slot] = *m;
      d[(N * 4 + 1) * LANES + slot] = *l;
    }
    __syncthreads();
    if (wave < half && mine) {
      const float* d = s + wave * (N * 4 + 4) * LANES;
      const float m2 = d[N * 4 * LANES + slot], l2 = d[(N * 4 + 1) * LANES + slot];
      const float M = fmaxf(*m, m2), base = M == -INFINITY ? 0.0f : M;
      const float f = __builtin_amdgcn_exp2f(*m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = o[i] * f + *reinterpret_cast<const f4_t*>(d + (i * LANES + slot) * 4) * f2;
      *l = *l * f + l2 * f2;
      *m = M;
    }
  }
}

// leaves a column's split for the join, or, where the row has one split at most, the output itself.
// o[j][i] is dim dim_of(j, i) of the column's head.
template <int HD, int N, int E>
__device__ __forceinline__ void leave(const PagedAttnArgs& a, const Place& p, uint32_t head, int G, float m, float l,
                                      const f4_t* o) {
  const size_t item = size_t(p.row) * a.H + head, pt = item * a.splits + p.split;
  float* dst = a.part_acc + pt * HD;
  float f = 1.0f;
  if (a.splits == 1) {
    dst = a.out + p.row * a.out_stride + size_t(head) * HD;
    f = l == 0.0f ? 0.0f : 1.0f / l;
  }
  if (G == 0) {
    a.part_ml[pt * 2] = m;
    a.part_ml[pt * 2 + 1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < N; j += 4)
      *reinterpret_cast<float4*>(dst + (j / E) * 16 * E + (4 * G + i) * E + j % E) =
          make_float4(o[j][i] * f, o[j + 1][i] * f, o[j + 2][i] * f, o[j + 3][i] * f);
}

// a split without slots: nothing for the join (it goes by the row's length); the output of a row of one
// split at most
template <int HD, int HT>
__device__ __forceinline__ void leave_none(const PagedAttnArgs& a, const Place& p) {
  if (a.splits != 1) return;
  const float v = p.ok ? 0.0f : __builtin_nanf("");
  for (uint32_t i = threadIdx.x; i < p.nh * HD; i += kWaves * 64) a.out[p.row * a.out_stride + size_t(p.h0) * HD + i] = v;
}

template <int HD, class T, int W, int NT>
__global__ void __launch_bounds__(kWaves * 64, 2) k_paged_16(PagedAttnArgs a) {
  using P = Parts<T, W>;
  using Vec = typename P::Vec;
  constexpr int HT = W * NT, KS = HD / 32, VD = HD / 16, E = VD < 8 ? 4 : 8, VP = VD / E;
  __shared__ uint64_t s_off[kWaves][2][32];
  __shared__ Vec s_q[NT][KS][P::kOps][64];  // the query operands, the same for every wave
  __shared__ __align__(16) float s_join[2 * (VD * 4 + 4) * 4 * W];
  Place p = place_of<HT>(a);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, G = lane >> 4, n = lane & 15;
  TileRows<32, 2> rows{s_off[wave]};
  if (a.window == 0) rows.next(a, p.row, p.split * a.chunk + 32 * wave, a.c.capacity - 1, lane);
  place_slots(a, &p);
  if (p.begin >= p.end) return leave_none<HD, HT>(a, p);  // (the whole workgroup)
  const int part = n / W, col = n % W;  // the column's part and head

  uint32_t t = p.begin + 32 * wave;
  uint4 kf[2][KS], vf[8][VP];
  auto load_k = [&](int buf) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* src = a.c.k + rows.s[buf][16 * u + n] + G * 16;
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[u][s] = ld_u128(src + 64 * s);
    }
  };
  auto load_v = [&](int buf) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const uint8_t* src = a.c.v + rows.s[buf][(r >> 2) * 16 + 4 * G + (r & 3)] + n * (2 * E);
#pragma unroll
      for (int c = 0; c < VP; ++c) {
        if constexpr (E == 8) {
          vf[r][c] = ld_u128(src + 256 * c);
        } else {
          const uint2 w = ld_u64(src);
          vf[r][c] = make_uint4(w.x, w.y, 0, 0);
        }
      }
    }
  };
  if (a.window != 0) rows.next(a, p.row, t, p.end - 1, lane);

  // the queries of the columns' heads: dims (G + 4 s) * 8 .. + 7 of head n % W of each tile of heads
  float mult[NT], m[NT], l[NT];
  f4_t o[NT][VD];
#pragma unroll
  for (int ht = 0; ht < NT; ++ht) {
    const uint32_t h = ht * W + col;
    const float* src = a.q + p.row * a.q_stride + size_t(p.h0 + (h < p.nh ? h : 0)) * HD + G * 8;
    float x[KS][8], top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float4 u = ld_f4(src + 32 * s), v = ld_f4(src + 32 * s + 4);
      const float w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[s][e] = h < p.nh ? w[e] : 0.0f;
        top = fmaxf(top, fabsf(x[s][e]));
      }
    }
    mult[ht] = a.scale * kLog2e;
    if constexpr (P::kScaleExp != 0) {
      top = pair_max(pair_max(top, 16), 32);
      int ex = 0;
      if (top > 0.0f && top < INFINITY) ex = 14 - __builtin_amdgcn_frexp_expf(top);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] = __builtin_amdgcn_ldexpf(x[s][e], ex);
      mult[ht] = __builtin_amdgcn_ldexpf(mult[ht], -ex);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (s % kWaves != wave) continue;
      Vec q[P::kOps];
      P::split(x[s], part, q);
#pragma unroll
      for (int op = 0; op < P::kOps; ++op) s_q[ht][s][op][lane] = q[op];
    }
    m[ht] = -INFINITY;
    l[ht] = 0.0f;
#pragma unroll
    for (int j = 0; j < VD; ++j) o[ht][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  int buf = 0;
  if (t < p.end) {
    rows.put(a, p, 0, lane);
    load_k(0);
    load_v(0);
    rows.next(a, p.row, t + 32 * kWaves, p.end - 1, lane);
  }
  __syncthreads();  // (the query operands)
  for (; t < p.end; t += 32 * kWaves) {
    const bool more = t + 32 * kWaves < p.end;
    asm volatile("" ::: "memory");  // (the query operands are read from LDS anew: they would fill the registers)
    // scores; the K registers are free after them and take the next tile's rows
    f4_t sc[NT][2];
#pragma unroll
    for (int ht = 0; ht < NT; ++ht)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int op = 0; op < P::kOps; ++op) acc = P::mfma(__builtin_bit_cast(Vec, kf[u][s]), s_q[ht][s][op][lane], acc);
        sc[ht][u] = acc;
      }
    buf ^= 1;
    if (more) {
      rows.put(a, p, buf, lane);
      load_k(buf);
      rows.next(a, p.row, t + 64 * kWaves, p.end - 1, lane);
    }
    Vec pb[NT][P::kOps];
#pragma unroll
    for (int ht = 0; ht < NT; ++ht) {
      float s8[8], mx = m[ht];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t j = t + (e >> 2) * 16 + 4 * G + (e & 3);
        const float s = sum_parts<W>(sc[ht][e >> 2][e & 3]) * mult[ht];
        s8[e] = j < p.end ? s : -INFINITY;
        mx = fmaxf(mx, s8[e]);
      }
      if (a.scores && part == 0 && ht * W + col < p.nh) {
        float* d = a.scores + (size_t(p.row) * a.H + p.h0 + ht * W + col) * a.score_stride + (t - p.lo) + 4 * G;
        *reinterpret_cast<float4*>(d) = make_float4(s8[0], s8[1], s8[2], s8[3]);
        *reinterpret_cast<float4*>(d + 16) = make_float4(s8[4], s8[5], s8[6], s8[7]);
      }
      mx = pair_max(pair_max(mx, 16), 32);
      const float base = mx == -INFINITY ? 0.0f : mx, f = __builtin_amdgcn_exp2f(m[ht] - base);
      if (__ballot(f != 1.0f) != 0) {
        l[ht] *= f;
#pragma unroll
        for (int j = 0; j < VD; ++j) o[ht][j] *= f;
      }
      m[ht] = mx;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s8[e] = __builtin_amdgcn_exp2f(s8[e] - base);
        l[ht] += s8[e];
        s8[e] *= float(1 << P::kScaleExp);
      }
      P::split(s8, part, pb[ht]);
    }
#pragma unroll
    for (int j = 0; j < VD; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint4 x = vf[2 * r][j / E], y = vf[2 * r + 1][j / E];
        const int wi = (j % E) / 2;
        const uint32_t lo = wi == 0 ? x.x : wi == 1 ? x.y : wi == 2 ? x.z : x.w;
        const uint32_t hi = wi == 0 ? y.x : wi == 1 ? y.y : wi == 2 ? y.z : y.w;
        w[r] = __builtin_amdgcn_perm(hi, lo, (j & 1) ? 0x07060302u : 0x05040100u);
      }
      const Vec vv = __builtin_bit_cast(Vec, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int ht = 0; ht < NT; ++ht)
#pragma unroll
        for (int op = 0; op < P::kOps; ++op) o[ht][j] = P::mfma(vv, pb[ht][op], o[ht][j]);
    }
    if (more) load_v(buf);
  }

  const bool bad = __ballot(rows.bad) != 0;
#pragma unroll
  for (int ht = 0; ht < NT; ++ht) {
    l[ht] = pair_sum(pair_sum(l[ht], 16), 32);
    if (bad) l[ht] = __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < VD; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[ht][j][i] = sum_parts<W>(o[ht][j][i]) * (1.0f / float(1 << P::kScaleExp));
    join_waves<VD, 4 * W>(s_join, wave, G * W + col, part == 0, &m[ht], &l[ht], o[ht]);
    if (wave == 0 && part == 0 && ht * W + col < p.nh) leave<HD, VD, E>(a, p, p.h0 + ht * W + col, G, m[ht], l[ht], o[ht]);
  }
}

// The f32 cache: 16 query heads as columns, tiles of 16 slots, v_mfma_f32_16x16x4f32 (exact f32 products).
template <int HD>
__global__ void __launch_bounds__(kWaves * 64, 2) k_paged_32(PagedAttnArgs a) {
  constexpr int KP = HD / 16, VP = HD / 64, VD = HD / 16;
  __shared__ uint64_t s_off[kWaves][2][16];
  __shared__ f4_t s_q[KP][64];
  __shared__ __align__(16) float s_join[2 * (VD * 4 + 4) * 64];
  Place p = place_of<16>(a);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, G = lane >> 4, n = lane & 15;
  TileRows<16, 4> rows{s_off[wave]};
  if (a.window == 0) rows.next(a, p.row, p.split * a.chunk + 16 * wave, a.c.capacity - 1, lane);
  place_slots(a, &p);
  if (p.begin >= p.end) return leave_none<HD, 16>(a, p);  // (the whole workgroup)

  uint32_t t = p.begin + 16 * wave;
  float4 kf[KP], vf[4][VP];
  auto load_k = [&](int buf) {
    const uint8_t* src = a.c.k + rows.s[buf][n] + G * 16;
#pragma unroll
    for (int c = 0; c < KP; ++c) kf[c] = ld_f4(reinterpret_cast<const float*>(src + 64 * c));
  };
  auto load_v = [&](int buf) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint8_t* src = a.c.v + rows.s[buf][4 * G + r] + n * 16;
#pragma unroll
      for (int c = 0; c < VP; ++c) vf[r][c] = ld_f4(reinterpret_cast<const float*>(src + 256 * c));
    }
  };
  if (a.window != 0) rows.next(a, p.row, t, p.end - 1, lane);
  const bool head = uint32_t(n) < p.nh;
#pragma unroll
  for (int c = 0; c < KP; ++c) {  // dims (G + 4 c) * 4 .. + 3 of head n
    if (c % kWaves != wave) continue;
    const float4 q = ld_f4(a.q + p.row * a.q_stride + size_t(p.h0 + (head ? n : 0)) * HD + G * 4 + 16 * c);
    s_q[c][lane] = head ? f4_t{q.x, q.y, q.z, q.w} : f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const float mult = a.scale * kLog2e;
  float m = -INFINITY, l = 0.0f;
  f4_t o[VD];
#pragma unroll
  for (int j = 0; j < VD; ++j) o[j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};

  int buf = 0;
  if (t < p.end) {
    rows.put(a, p, 0, lane);
    load_k(0);
    load_v(0);
    rows.next(a, p.row, t + 16 * kWaves, p.end - 1, lane);
  }
  __syncthreads();  // (the queries)
  for (; t < p.end; t += 16 * kWaves) {
    const bool more = t + 16 * kWaves < p.end;
    asm volatile("" ::: "memory");  // (the queries are read from LDS anew: they would fill the registers)
    f4_t sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < KP; ++c) {
      const f4_t q = s_q[c][lane];
      sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c].x, q[0], sc, 0, 0, 0);
      sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c].y, q[1], sc, 0, 0, 0);
      sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c].z, q[2], sc, 0, 0, 0);
      sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c].w, q[3], sc, 0, 0, 0);
    }
    buf ^= 1;
    if (more) {
      rows.put(a, p, buf, lane);
      load_k(buf);
      rows.next(a, p.row, t + 32 * kWaves, p.end - 1, lane);
    }
    float s4[4], mx = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s4[i] = t + 4 * G + i < p.end ? sc[i] * mult : -INFINITY;
      mx = fmaxf(mx, s4[i]);
    }
    if (a.scores && head)
      *reinterpret_cast<float4*>(a.scores + (size_t(p.row) * a.H + p.h0 + n) * a.score_stride + (t - p.lo) + 4 * G) =
          make_float4(s4[0], s4[1], s4[2], s4[3]);
    mx = pair_max(pair_max(mx, 16), 32);
    const float base = mx == -INFINITY ? 0.0f : mx, f = __builtin_amdgcn_exp2f(m - base);
    if (__ballot(f != 1.0f) != 0) {
      l *= f;
#pragma unroll
      for (int j = 0; j < VD; ++j) o[j] *= f;
    }
    m = mx;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s4[i] = __builtin_amdgcn_exp2f(s4[i] - base);
      l += s4[i];
    }
#pragma unroll
    for (int j = 0; j < VD; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = vf[i][j / 4];
        const float v = j % 4 == 0 ? x.x : j % 4 == 1 ? x.y : j % 4 == 2 ? x.z : x.w;
        o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s4[i], o[j], 0, 0, 0);
      }
    if (more) load_v(buf);
  }
  l = pair_sum(pair_sum(l, 16), 32);
  if (__ballot(rows.bad) != 0) l = __builtin_nanf("");
  join_waves<VD, 64>(s_join, wave, lane, true, &m, &l, o);
  if (wave == 0 && head) leave<HD, VD, 4>(a, p, p.h0 + n, G, m, l, o);
}

// ---- joining the splits, and the slots' weights -------------------------------------------------------------
// the row's splits that hold slots
__device__ __forceinline__ uint32_t splits_of(const PagedAttnArgs& a, uint32_t lo, uint32_t len) {
  return (len - lo + a.chunk - 1) / a.chunk;
}

// maximum and sum over a head's splits, by one wave
__device__ __forceinline__ void join_ml(const PagedAttnArgs& a, uint32_t item, uint32_t ns, int lane, float* M, float* L) {
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + size_t(item) * a.splits;
  const uint32_t mine = min(uint32_t(lane), a.splits - 1);
  float2 x = ml[mine];  // (does not wait for the row's length)
  if (uint32_t(lane) >= ns) x = make_float2(-INFINITY, 0.0f);
  float m = x.x;
  for (uint32_t s = lane + 64; s < ns; s += 64) m = fmaxf(m, ml[s].x);
  m = wave_max(m);
  if (m == -INFINITY) m = 0.0f;  // (no score above -inf)
  float l = x.y * __builtin_amdgcn_exp2f(x.x - m);
  for (uint32_t s = lane + 64; s < ns; s += 64) l += ml[s].y * __builtin_amdgcn_exp2f(ml[s].x - m);
  *M = m;
  *L = wave_sum(l);
}

// blocks 0 .. joins - 1: the output of one (row, head) each, its splits in 256 / (HD / 4) groups;
// the others: the weights of 1024 slots of one (row, kv head)
template <int HD>
__global__ void __launch_bounds__(256) k_paged_join(PagedAttnArgs a, uint32_t joins, uint32_t weight_parts) {
  constexpr int D4 = HD / 4, GR = 256 / D4;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  uint32_t lo, len;
  if (blockIdx.x < joins) {
    const uint32_t item = blockIdx.x, h = item % a.H, row = item / a.H;
    const bool ok = row_range(a, row, &lo, &len);
    __shared__ __align__(16) float s_o[GR][HD];
    __shared__ float s_f[kMaxSplits];
    const float* ml = a.part_ml + size_t(item) * a.splits * 2;
    const float* acc = a.part_acc + size_t(item) * a.splits * HD + (tid % D4) * 4;
    // the first sums of every group of threads are requested before the statistics say what they count for
    constexpr int U = 4;
    f4_t x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t s = tid / D4 + u * GR;
      const float4 v = ld_f4(acc + size_t(min(s, a.splits - 1)) * HD);
      x[u] = f4_t{v.x, v.y, v.z, v.w};
    }
    const uint32_t ns = splits_of(a, lo, len);
    float M, L;
    join_ml(a, item, ns, lane, &M, &L);  // (every wave for itself)
    for (uint32_t s = tid; s < ns; s += 256) s_f[s] = __builtin_amdgcn_exp2f(gld(ml + 2 * s) - M);
    __syncthreads();
    f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (tid / D4 + u * GR < ns) o += x[u] * s_f[tid / D4 + u * GR];
#pragma unroll 4
    for (uint32_t s = tid / D4 + U * GR; s < ns; s += GR) {
      const float4 v = ld_f4(acc + size_t(s) * HD);
      o += f4_t{v.x, v.y, v.z, v.w} * s_f[s];
    }
    *reinterpret_cast<f4_t*>(&s_o[tid / D4][(tid % D4) * 4]) = o;
    __syncthreads();
    if (tid < HD) {
      float v = 0.0f;
#pragma unroll
      for (int g = 0; g < GR; ++g) v += s_o[g][tid];
      a.out[row * a.out_stride + size_t(h) * HD + tid] = !ok ? __builtin_nanf("") : (L == 0.0f ? 0.0f : v / L);
    }
    return;
  }
  const uint32_t b = blockIdx.x - joins, part = b % weight_parts, item = b / weight_parts;
  const uint32_t kvh = item % a.c.KV, row = item / a.c.KV, gq = a.H / a.c.KV;
  row_range(a, row, &lo, &len);
  const uint32_t first = part * 1024, i = first + tid * 4;  // slots lo + i .. + 3
  const size_t base = (size_t(row) * a.c.KV + kvh) * a.weight_stride;
  // slots before the window were given nothing
  for (uint32_t j = first + tid; j < lo; j += weight_parts * 1024)
    for (uint32_t k = 0; k < 1024 && j + k < lo; k += 256) a.weight_out[base + j + k] = a.weight_in ? a.weight_in[base + j + k] : 0.0f;
  if (lo + first >= len) return;
  const uint32_t ns = splits_of(a, lo, len);
  __shared__ float s_ml[64][2];
  f4_t w = {0.0f, 0.0f, 0.0f, 0.0f};
  const bool in = lo + i < len;
  for (uint32_t g0 = 0; g0 < gq; g0 += 64) {  // 64 query heads at a time
    const uint32_t ng = min(64u, gq - g0);
    const float* sc = a.scores + (size_t(row) * a.H + kvh * gq + g0) * a.score_stride + (in ? i : 0u);
    __syncthreads();
    for (uint32_t g = wave; g < ng; g += kWaves) {
      float M, L;
      join_ml(a, row * a.H + kvh * gq + g0 + g, ns, lane, &M, &L);
      if (lane == 0) {
        s_ml[g][0] = M;
        s_ml[g][1] = L == 0.0f ? 0.0f : 1.0f / L;
      }
    }
    __syncthreads();
#pragma unroll 8
    for (uint32_t g = 0; g < ng; ++g) {
      const float4 s = ld_f4(sc + size_t(g) * a.score_stride);
      const float M = s_ml[g][0], f = s_ml[g][1];
      w += f4_t{__builtin_amdgcn_exp2f(s.x - M), __builtin_amdgcn_exp2f(s.y - M), __builtin_amdgcn_exp2f(s.z - M),
                __builtin_amdgcn_exp2f(s.w - M)} * f;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lo + i + k < len) a.weight_out[base + lo + i + k] = (a.weight_in ? a.weight_in[base + lo + i + k] : 0.0f) + w[k];
}

// ---- host -----------------------------------------------------------------------------------------------------
// How the rows are split: a workgroup's slots (`chunk`) are a multiple of its tiles; about 4 workgroups per CU
// where there are few rows, at most 1024 slots a workgroup where there are many (rows of different lengths
// then still spread evenly: the chip takes the next workgroup where one ends), at most 512 splits.
struct AttnPlan {
  uint32_t splits = 1, chunk = 1, score_stride = 0;
  uint64_t groups = 0;  // (row, kv head, group of query heads)
  size_t off_acc = 0, off_scores = 0, bytes = 0;
};

// query heads a workgroup serves: of the 16 columns one holds a head of an f32 cache, two or (bf16, up to 4
// heads) four one of a 16-bit cache; two such tiles of heads where the accumulators of both fit the registers
uint32_t heads_per_group(const chpe_kv_pages* c, uint32_t heads) {
  const uint32_t gq = heads / c->kv_heads;
  if (c->type == 0 || (gq > 8 && c->head_dim <= 128)) return 16;
  return c->type == 2 && gq <= 4 ? 4 : 8;
}

void split_range(uint64_t groups, uint32_t range, uint32_t step, uint32_t* splits, uint32_t* chunk) {
  const uint64_t n = std::max<uint64_t>(1, (uint64_t(range) + step - 1) / step);  // steps in all
  uint64_t want = std::max<uint64_t>((1024 + groups - 1) / groups, (uint64_t(range) + 1023) / 1024);
  want = std::min<uint64_t>(std::min<uint64_t>(want, n), kMaxSplits);
  const uint64_t per = (n + want - 1) / want;
  *chunk = uint32_t(per * step);
  *splits = uint32_t((n + per - 1) / per);
}

AttnPlan attn_plan(const chpe_kv_pages* c, uint32_t heads, uint32_t max_len, uint32_t window, bool weights) {
  AttnPlan p;
  const uint32_t gq = heads / c->kv_heads, ht = heads_per_group(c, heads), step = (c->type == 0 ? 16 : 32) * kWaves;
  p.groups = uint64_t(c->rows) * c->kv_heads * ((gq + ht - 1) / ht);
  const uint64_t groups = std::max<uint64_t>(1, p.groups), items = uint64_t(c->rows) * heads;
  split_range(groups, window != 0 && window < max_len ? window : max_len, step, &p.splits, &p.chunk);
  // the workspace does not depend on the window: room for the most splits of any shorter range, which the
  // wanted number bounds
  const uint64_t n = std::max<uint64_t>(1, (uint64_t(max_len) + step - 1) / step);
  uint64_t room = std::max<uint64_t>((1024 + groups - 1) / groups, (uint64_t(max_len) + 1023) / 1024);
  room = std::min<uint64_t>(std::min<uint64_t>(room, n), kMaxSplits);
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  p.off_acc = up(items * room * 8);
  p.off_scores = p.off_acc + up(items * room * c->head_dim * 4);
  p.score_stride = uint32_t((max_len + 63) / 64 * 64);
  p.bytes = p.off_scores + (weights ? up(items * p.score_stride * 4) : 0);
  return p;
}

template <int HD>
bool launch_partial(const PagedAttnArgs& a, int type, uint32_t ht, uint64_t blocks, hipStream_t st) {
  const uint32_t thr = kWaves * 64;
  if (type == 0) return launch(&k_paged_32<HD>, blocks, thr, st, a);
  if (type == 2 && ht == 4) return launch(&k_paged_16<HD, Bf16, 4, 1>, blocks, thr, st, a);
  if (ht == 8)
    return type == 1 ? launch(&k_paged_16<HD, _Float16, 8, 1>, blocks, thr, st, a)
                     : launch(&k_paged_16<HD, Bf16, 8, 1>, blocks, thr, st, a);
  if constexpr (HD <= 128)
    return type == 1 ? launch(&k_paged_16<HD, _Float16, 8, 2>, blocks, thr, st, a)
                     : launch(&k_paged_16<HD, Bf16, 8, 2>, blocks, thr, st, a);
  return false;
}

bool attn_shape_ok(const chpe_kv_pages* c, uint32_t heads, uint32_t max_len) {
  return heads != 0 && heads % c->kv_heads == 0 && heads <= 65536 &&
         uint64_t(max_len) <= uint64_t(c->pages_per_row) * c->page_size;
}

}  // namespace
}  // namespace chpe

using namespace chpe;

extern "C" size_t chpe_paged_attention_workspace(const chpe_kv_pages* cache, uint32_t heads, uint32_t max_len,
                                                 int weights) {
  Pages p;
  if (!pages_from(cache, &p) || !attn_shape_ok(cache, heads, max_len)) return 0;
  return attn_plan(cache, heads, max_len, 0, weights != 0).bytes;
}

extern "C" int chpe_paged_attention(const chpe_kv_pages* cache, uint32_t heads, const int32_t* lens, uint32_t max_len,
                                    const float* q, uint64_t q_stride, float scale, uint32_t window, float* out,
                                    uint64_t out_stride, const float* weight_in, float* weight_out,
                                    uint64_t weight_stride, void* workspace, size_t workspace_bytes, void* stream) {
  PagedAttnArgs a{};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!pages_from(cache, &a.c) || !stream_here(st) || !attn_shape_ok(cache, heads, max_len)) return -1;
  if (cache->rows == 0) return 0;
  const uint64_t width = uint64_t(heads) * cache->head_dim;
  if (!lens || !q || !out || !workspace || !aligned16(q) || !aligned16(out) || !aligned16(workspace)) return -1;
  if (q_stride % 4 || out_stride % 4 || (cache->rows > 1 && (q_stride < width || out_stride < width))) return -1;
  if ((weight_in && !weight_out) || (weight_out && weight_stride < max_len)) return -1;
  const AttnPlan p = attn_plan(cache, heads, max_len, window, weight_out != nullptr);
  const uint32_t parts = weight_out ? (max_len + 1023) / 1024 : 0, joins = p.splits > 1 ? cache->rows * heads : 0;
  const uint64_t joined = uint64_t(joins) + uint64_t(cache->rows) * cache->kv_heads * parts;
  if (uint64_t(cache->rows) * heads > kMaxBlocks || p.groups * p.splits > kMaxBlocks || joined > kMaxBlocks) return -1;
  if (workspace_bytes < p.bytes) return -2;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.q = q;
  a.lens = lens;
  a.out = out;
  a.part_ml = reinterpret_cast<float*>(ws);
  a.part_acc = reinterpret_cast<float*>(ws + p.off_acc);
  a.scores = weight_out ? reinterpret_cast<float*>(ws + p.off_scores) : nullptr;
  a.weight_in = weight_in;
  a.weight_out = weight_out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.weight_stride = weight_stride;
  a.rows = cache->rows;
  a.H = heads;
  a.max_len = max_len;
  a.window = window;
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.scale = scale;
  a.score_stride = p.score_stride;
  const int type = cache->type;
  const uint32_t hd = cache->head_dim, ht = heads_per_group(cache, heads);
  const uint64_t blocks = p.groups * p.splits;
  bool ok = hd == 64    ? launch_partial<64>(a, type, ht, blocks, st)
            : hd == 128 ? launch_partial<128>(a, type, ht, blocks, st)
                        : launch_partial<256>(a, type, ht, blocks, st);
  if (ok && joined != 0)
    ok = hd == 64    ? launch(&k_paged_join<64>, joined, 256, st, a, joins, parts)
         : hd == 128 ? launch(&k_paged_join<128>, joined, 256, st, a, joins, parts)
                     : launch(&k_paged_join<256>, joined, 256, st, a, joins, parts);
  return ok ? 0 : -3;
}
