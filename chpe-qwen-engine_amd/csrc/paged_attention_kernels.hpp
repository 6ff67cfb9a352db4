// paged_attention_kernels.hpp -- the attention over a part of the slots of a paged cache: what chpe_paged_attention's
// splits and chpe_paged_prefix_attention's have in common.
// Args (a kernel's argument) says where a workgroup's queries, slots and results lie:
//   place_of<HT>(), place_slots(&p)  its place and the slots of it
//   eager(), eager_slot(p)           whether the first slot is known before the rows' lengths, and that slot
//   query<HD>(p, i)                  query i of the workgroup
//   part_of(p, i), whole()           where its sums go; whether they are the output
//   leave_none<HD>(p)                what a place without slots leaves
//   kScores, scores, score_stride    whether the scores are left too, and where
#pragma once
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace chpe {
namespace {
using namespace dev;

constexpr int kWaves = 4;  // of a workgroup

// a workgroup's place: slots begin .. end - 1 in the pages of row `table`, of row `row`'s range lo .. len - 1, for query
// heads h0 .. h0 + nh - 1
struct Place {
  uint32_t row, table, kvh, h0, nh, split, begin, end, lo, len;
  bool ok;
};
// ---- the sums of a split ------------------------------------------------------------------------------------
// 4 waves; wave w takes the tiles w, w + 4, .. of the split.  A tile's scores are S^T = K . Q^T on the matrix
// cores (rows: slots, columns: query heads), its output O^T = V^T . P^T (rows: dims, columns: heads): with the
// heads as columns of both, a lane (G, n) = (lane / 16, lane % 16) keeps the running maximum and sum of column n
// in scalars of its own, and the result layout of the first product (slots 4 G + i of column n) is the operand
// layout of the second, so the weights never leave the registers.  The order of the dims inside the first product
// and of the slots inside the second is free as long as both operands agree, which is what lets every lane load
// 16 bytes in a row: K rows as pieces of 4 x 16 bytes, V rows as 16 lanes x 16 bytes.
// The running maximum is in units of log2 (scores times scale * log2 e).
// Bound by memory: each K and V row is read once for the query heads of a workgroup (4, 8 or 16 of its kv head's,
// heads_per_group; more query heads read it again), the next tile's K rows while the weights are formed, its V rows
// while the scores are.  64 rows of 8320 slots with 8 kv heads of 128 (2.2 GB, fp16 or bf16) take 370 to 384 us with the
// join, 5.7 to 5.9 TB/s, as do 32 such rows in f32; reads of the card reach 6.3, marked as made once (as V's are) 7.1.
// A wave holds at most 128 dims of a tile's rows and of the accumulators (its registers then allow three waves a
// SIMD); at head dim 256 two waves share a tile, half of the dims each, and add their scores through LDS.
constexpr int kWaveDims = 128;
constexpr int dim_shares(int hd) { return hd > kWaveDims ? hd / kWaveDims : 1; }
constexpr int tiles_at_once(int hd) { return kWaves / dim_shares(hd); }
constexpr uint32_t kMaxSplits = 512;
constexpr float kLog2e = 1.4426950408889634f;

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// 16-bit elements with f32 queries and weights: x is taken apart into parts of the cache's type, part p of head h in
// column h + p * W of the 16; all columns' results are added at the end (sum_parts).  bf16: three parts hold all 24
// bits of x; of up to 4 heads they fit the 16 columns, of 8 the third is an operand of its own.  fp16: two parts hold
// 22 bits, so that a query or weight enters the products rounded, off by up to 2^-23 of itself (one unit in the last
// place of f32, which a quarter of all values are off by): as much as two of the roundings that the f32 sums of hd
// products make anyway, and a third part would double the products.  x is brought near 2^14 by a power of two
// first, so that the second part falls below fp16's range only where x is small beside the others: then it is off
// by 2^-38 of the head's largest query, or by 2^-40 of the row's largest weight.
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
      const float r = x[e] - float(__bf16(x[e])), r2 = r - float(__bf16(r));
      out[0][e] = __bf16(part == 0 ? x[e] : part == 1 ? r : part == 2 && W == 4 ? r2 : 0.0f);
      if constexpr (W == 8) out[1][e] = __bf16(part == 0 ? r2 : 0.0f);
    }
  }
  static __device__ f4_t mfma(Vec a, Vec b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <int W>
__device__ __forceinline__ float sum_parts(float v) {
  if constexpr (W == 4) v = pair_sum(v, 4);
  return pair_sum(v, 8);
}

// A weight's exponent is x mult - base, base the largest product x mult so far, rounded: the product again inside the fma, so
// that it is rounded once, as small as the difference is.  The largest one's own exponent is then what its rounding
// lost, which from 2^22 on is 1 / 4 and more, and past 2^25 would take fp16 parts out of their range and soon leave no
// weight at all.  Where the base is that large the rounded product counts, 0 for the largest whatever its size: x
// becomes the exponent itself, to be taken times 1.
constexpr float kFarScore = 4194304.0f;
template <int N>
__device__ __forceinline__ void far_scores(float (&x)[N], float& mult, float& base) {
  if (!(fabsf(base) >= kFarScore)) return;  // (a column's own: its bits do not depend on the others)
#pragma unroll
  for (int e = 0; e < N; ++e) {
    x[e] *= mult;
    asm("" : "+v"(x[e]));  // (not the fma again)
    x[e] -= base;
  }
  mult = 1.0f;
  base = 0.0f;
}

// The tile's row offsets (bytes from k or v): lane r of the wave finds row r's page and leaves the
// offset in LDS for the lanes that load the row.  `next` requests the table entry ahead of its use; for the
// first tile of a range that starts at slot 0 it does not wait for the row's length (entries behind it may
// hold anything).  Rows behind the split's end are its last row.
template <int ROWS, int ES>
struct TileRows {
  uint64_t (*s)[ROWS];
  uint32_t id, slot;
  bool bad;
  template <class Args>
  __device__ void next(const Args& a, uint32_t row, uint32_t t, uint32_t last, int lane) {
    slot = min(t + uint32_t(lane % ROWS), last);
    id = uint32_t(gld(a.c.table + size_t(row) * a.c.table_stride + (slot >> a.c.shift)));
  }
  template <class Args>
  __device__ void put(const Args& a, const Place& p, int buf, int lane) {
    // a row behind the end, which `next` did not know yet: the last one's, which is in the tile too
    const uint32_t first = uniform(slot);
    const uint32_t id_last = lane_of(id, min(p.end - 1 - first, uint32_t(ROWS - 1)));
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

// An infinite V element makes its dim's sum infinite whatever its slot's weight, but the products give NaN where
// they meet it with a 0: a padding row's weight, a part of a weight that has no bits left, a weight that 32 bits
// hold as 0.  So a sum of dims dim .. dim + 3 that came out infinite or NaN is told again from the split's values
// that are not finite themselves: their sum, or v where there are none (a sum past f32's range).  64 rows of up to
// 8320 slots take 0.52 ms with one such element in every row, 1.4 ms where all are, 0.21 ms without.
__device__ __forceinline__ bool all_finite(f4_t v) {
  return fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY && fabsf(v.z) < INFINITY && fabsf(v.w) < INFINITY;
}
template <class T, class Args>
__device__ __forceinline__ f4_t non_finite_sum(const Args& a, const Place& p, uint32_t dim, f4_t v) {
  f4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t j = p.begin; j < p.end; ++j) {
    uint32_t page;
    a.c.page_of(p.table, j, &page);  // (a bad one: the head's sum of weights is NaN and nothing comes here)
    const T* src = reinterpret_cast<const T*>(a.c.v) + a.c.at(page, p.kvh, j) + dim;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = Elem<T>::get(src + e);
      s[e] += fabsf(x) < INFINITY ? 0.0f : x;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = s[e] == 0.0f ? v[e] : s[e];
  return v;
}

// The split's result from the waves' maxima, sums and accumulators: every wave leaves its own in LDS, then all
// threads join them, 4 dims of a head at a time, and write them out, for the join or, where a row has one split
// at most, as the output.  LANES = 4 * columns lanes of a wave hold something, lane
// slot = G * columns + column; o[j][i] is dim (j / E) * 16 E + (4 G + i) E + j % E of the wave's dims.
template <int LANES>
struct WaveSums {
  f4_t o[kWaves][kWaveDims / 16][LANES];
  float2 ml[kWaves][LANES / 4];
};
template <int HD, class T, int E, int LANES, int VD, class Args>
__device__ __forceinline__ void leave(const Args& a, const Place& p, WaveSums<LANES>& s, int tid, int wave, int G,
                                      int col, bool mine, uint32_t head0, float m, float l, const f4_t (&o)[VD]) {
  constexpr int DS = dim_shares(HD), TW = kWaves / DS, COLS = LANES / 4;
  if (mine) {
#pragma unroll
    for (int r = 0; r < VD; ++r) {  // (j / 4) * 4 + i: dims j .. j + 3 of row i
      const int j = r / 4 * 4, i = r % 4;
      s.o[wave][r][G * COLS + col] = f4_t{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]};
    }
    if (G == 0) s.ml[wave][col] = make_float2(m, l);
  }
  __syncthreads();
  const int at = tid % LANES, tG = at / COLS;  // (256 is a multiple of LANES)
  const uint32_t head = head0 + at % COLS;
  if (head >= p.nh) return;
  float M = -INFINITY, L = 0.0f, f[TW];
#pragma unroll
  for (int w = 0; w < TW; ++w) M = fmaxf(M, s.ml[w * DS][at % COLS].x);
  const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
  for (int w = 0; w < TW; ++w) {
    f[w] = __builtin_amdgcn_exp2f(s.ml[w * DS][at % COLS].x - base);
    L += s.ml[w * DS][at % COLS].y * f[w];
  }
  const size_t pt = a.part_of(p, head);
  const bool whole = a.whole();
  float* dst = whole ? a.out + p.row * a.out_stride + size_t(p.h0 + head) * HD : a.part_acc + pt * HD;
  const float g = !whole ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L;
  if (tid < COLS) reinterpret_cast<float2*>(a.part_ml)[pt] = make_float2(M, L);
  constexpr int PIECES = (DS * VD * LANES + 255) / 256;
  // piece k of a thread: 4 dims from this one on
  auto dim_of = [&](int k) {
    const int i0 = k * (256 / LANES) + tid / LANES, r = i0 % VD, j = r / 4 * 4, i = r % 4;
    return i0 / VD * kWaveDims + (j / E) * 16 * E + (4 * tG + i) * E + j % E;
  };
  auto none = [&](int k) { return DS * VD * LANES % 256 != 0 && k * (256 / LANES) + tid / LANES >= DS * VD; };
  bool finite = true;
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    const int i0 = k * (256 / LANES) + tid / LANES, share = i0 / VD, r = i0 % VD;
    if (none(k)) break;
    f4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < TW; ++w) v += s.o[w * DS + share][r][at] * f[w];
    v *= g;
    finite &= all_finite(v);
    *reinterpret_cast<f4_t*>(dst + dim_of(k)) = v;
  }
  if (finite || L != L) return;
#pragma unroll 1
  for (int k = 0; k < PIECES; ++k) {
    if (none(k)) break;
    f4_t* d = reinterpret_cast<f4_t*>(dst + dim_of(k));
    const f4_t v = *d;
    if (!all_finite(v)) *d = non_finite_sum<T>(a, p, dim_of(k), v);
  }
}

template <int HD, class T, int W, int NT, class Args>
__global__ void __launch_bounds__(kWaves * 64, NT == 1 ? (HD == 64 ? 4 : 3) : (HD == 64 ? 3 : 2)) k_paged_16(Args a) {
  using P = Parts<T, W>;
  using Vec = typename P::Vec;
  constexpr int DS = dim_shares(HD), HW = HD / DS, UNIT = 32 * tiles_at_once(HD);
  constexpr int HT = W * NT, KS = HW / 32, VD = HW / 16, E = VD < 8 ? 4 : 8;
  __shared__ uint64_t s_off[kWaves][2][32];
  __shared__ Vec s_q[NT][HD / 32][P::kOps][64];  // the query operands, the same for every wave
  __shared__ float s_mult[HT];
  // a share's scores for the other one; after the tiles the waves' sums
  __shared__ union {
    WaveSums<4 * W> sums;
    f4_t share[DS > 1 ? 2 * kWaves * NT * 2 * 64 : 1];
  } s_u;
  const int wave = uniform(threadIdx.x >> 6), share = wave % DS;
  const int tid = threadIdx.x, lane = tid & 63, G = lane >> 4, n = lane & 15;
  const int part = n / W, col = n % W;  // the column's part and head
  Place p = a.template place_of<HT>();
  TileRows<32, 2> rows{s_off[wave], 0, 0, false};
  if (a.eager()) rows.next(a, p.table, a.eager_slot(p) + 32 * (wave / DS), a.c.capacity - 1, lane);
  a.place_slots(&p);
  if (p.begin >= p.end) return a.template leave_none<HD>(p);  // (the whole workgroup)
  uint32_t t = p.begin + 32 * (wave / DS);
  u32x4_t kf[2][KS], vf[8];
  auto load_k = [&](int buf) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* src = a.c.k + rows.s[buf][16 * u + n] + G * 16 + share * (HW * 2);
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[u][s] = gld(reinterpret_cast<const u32x4_t*>(src + 64 * s));
    }
  };
  auto load_v = [&](int buf) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const uint8_t* src = a.c.v + rows.s[buf][(r >> 2) * 16 + 4 * G + (r & 3)] + n * (2 * E) + share * (HW * 2);
      if constexpr (E == 8) {
        vf[r] = ld_once(reinterpret_cast<const u32x4_t*>(src));
      } else {
        const u32x2_t w = ld_once(reinterpret_cast<const u32x2_t*>(src));
        vf[r] = u32x4_t{w.x, w.y, 0, 0};
      }
    }
  };
  if (!a.eager()) rows.next(a, p.table, t, p.end - 1, lane);
  // the queries: HD / 8 threads a head take 8 dims each (dims (G + 4 s) * 8 .. + 7 are what lanes of group G
  // need in step s); they are taken apart while the first tile's rows are on their way
  constexpr int TH = HD / 8;
  const int qh = tid / TH, qc = tid % TH;
  float x[8];
  if (qh < HT) {
    const float* src = a.template query<HD>(p, qh < int(p.nh) ? qh : 0) + qc * 8;
    const float4 u = ld_f4(src), v = ld_f4(src + 4);
    const float w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = w[e];
  }
  int buf = 0;
  if (t < p.end) {
    rows.put(a, p, 0, lane);
    load_k(0);
    load_v(0);
    rows.next(a, p.table, t + UNIT, p.end - 1, lane);
  }
  if (qh < HT) {  // (whole groups of TH lanes)
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (qh >= int(p.nh)) x[e] = 0.0f;
      top = fmaxf(top, fabsf(x[e]));
    }
    int ex = 0;
    if constexpr (P::kScaleExp != 0) {
#pragma unroll
      for (int o = 1; o < TH; o <<= 1) top = pair_max(top, o);
      if (top > 0.0f && top < INFINITY) ex = 14 - __builtin_amdgcn_frexp_expf(top);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_ldexpf(x[e], ex);
    }
    if (qc == 0) s_mult[qh] = __builtin_amdgcn_ldexpf(a.scale * kLog2e, -ex);
#pragma unroll
    for (int pt = 0; pt < 16 / W; ++pt) {
      Vec q[P::kOps];
      P::split(x, pt, q);
#pragma unroll
      for (int op = 0; op < P::kOps; ++op) s_q[qh / W][qc / 4][op][(qc % 4) * 16 + pt * W + qh % W] = q[op];
    }
  }
  __syncthreads();  // (the query operands)
  float mult[NT], m[NT], l[NT];
  f4_t o[NT][VD];
#pragma unroll
  for (int ht = 0; ht < NT; ++ht) {
    mult[ht] = s_mult[ht * W + col];
    m[ht] = -INFINITY;
    l[ht] = 0.0f;
#pragma unroll
    for (int j = 0; j < VD; ++j) o[ht][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // (where waves share a tile, all waves of the workgroup take the same number of steps)
  for (uint32_t t0 = p.begin; (DS > 1 ? t0 : t) < p.end; t0 += UNIT, t += UNIT) {
    const bool here = DS == 1 || t < p.end, more = t + UNIT < p.end;
    asm volatile("" ::: "memory");  // (the query operands are read from LDS anew: they would fill the registers)
    // scores; the K registers are free after them and take the next tile's rows
    f4_t sc[NT][2];
    if (here) {
#pragma unroll
      for (int ht = 0; ht < NT; ++ht)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int op = 0; op < P::kOps; ++op)
              acc = P::mfma(__builtin_bit_cast(Vec, kf[u][s]), s_q[ht][share * KS + s][op][lane], acc);
          sc[ht][u] = acc;
          if constexpr (DS > 1) s_u.share[(((buf * kWaves + wave) * NT + ht) * 2 + u) * 64 + lane] = acc;
        }
    }
    buf ^= 1;
    if (more) {
      rows.put(a, p, buf, lane);
      load_k(buf);
      rows.next(a, p.table, t + 2 * UNIT, p.end - 1, lane);
    }
    if constexpr (DS > 1) {
      // (written anew two steps later, past the next step's barrier)
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      if (!here) continue;
#pragma unroll
      for (int ht = 0; ht < NT; ++ht)
#pragma unroll
        for (int u = 0; u < 2; ++u) sc[ht][u] += s_u.share[((((buf ^ 1) * kWaves + (wave ^ 1)) * NT + ht) * 2 + u) * 64 + lane];
    }
    Vec pb[NT][P::kOps];
#pragma unroll
    for (int ht = 0; ht < NT; ++ht) {
      float s8[8], top[8], mx = m[ht];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t j = t + (e >> 2) * 16 + 4 * G + (e & 3);
        s8[e] = sum_parts<W>(sc[ht][e >> 2][e & 3]);
        top[e] = j < p.end ? s8[e] * mult[ht] : -INFINITY;
        mx = fmaxf(mx, top[e]);
      }
      if constexpr (Args::kScores) {
        if (a.scores && share == 0 && part == 0 && ht * W + col < p.nh) {
          float* d = a.scores + (size_t(p.row) * a.H + p.h0 + ht * W + col) * a.score_stride + (t - p.lo) + 4 * G;
          *reinterpret_cast<float4*>(d) = make_float4(top[0], top[1], top[2], top[3]);
          *reinterpret_cast<float4*>(d + 16) = make_float4(top[4], top[5], top[6], top[7]);
        }
      }
      mx = pair_max(pair_max(mx, 16), 32);
      float base = mx == -INFINITY ? 0.0f : mx;
      const float f = __builtin_amdgcn_exp2f(m[ht] - base);
      if (__ballot(f != 1.0f) != 0) {
        l[ht] *= f;
#pragma unroll
        for (int j = 0; j < VD; ++j) o[ht][j] *= f;
      }
      m[ht] = mx;
      float mu = mult[ht];
      far_scores(s8, mu, base);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s8[e] = __builtin_amdgcn_exp2f(top[e] > -INFINITY ? fmaf(s8[e], mu, -base) : top[e]);
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
        const u32x4_t x = vf[2 * r], y = vf[2 * r + 1];
        const uint32_t lo = j / 2 == 0 ? x.x : j / 2 == 1 ? x.y : j / 2 == 2 ? x.z : x.w;
        const uint32_t hi = j / 2 == 0 ? y.x : j / 2 == 1 ? y.y : j / 2 == 2 ? y.z : y.w;
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
    if (ht != 0 || DS > 1) __syncthreads();  // (s_u)
    leave<HD, T, E, 4 * W>(a, p, s_u.sums, tid, wave, G, col, part == 0, ht * W, m[ht], l[ht], o[ht]);
  }
}

// The same for the f32 cache: 16 query heads as columns, tiles of 16 slots, v_mfma_f32_16x16x4f32 (exact f32
// products).  The second product takes the four slots of a lane outside and the dims inside, so that products into
// one accumulator are VD apart.
template <int HD, class Args>
__global__ void __launch_bounds__(kWaves * 64, HD == 64 ? 4 : 3) k_paged_32(Args a) {
  constexpr int DS = dim_shares(HD), HW = HD / DS, UNIT = 16 * tiles_at_once(HD);
  constexpr int KP = HW / 16, VP = HW / 64, VD = HW / 16;
  __shared__ uint64_t s_off[kWaves][2][16];
  __shared__ f4_t s_q[HD / 16][64];  // dims (G + 4 c) * 4 .. + 3 of head n
  // a share's scores for the other one; after the tiles the waves' sums
  __shared__ union {
    WaveSums<64> sums;
    f4_t share[DS > 1 ? 2 * kWaves * 64 : 1];
  } s_u;
  const int wave = uniform(threadIdx.x >> 6), share = wave % DS;
  const int tid = threadIdx.x, lane = tid & 63, G = lane >> 4, n = lane & 15;
  Place p = a.template place_of<16>();
  TileRows<16, 4> rows{s_off[wave], 0, 0, false};
  if (a.eager()) rows.next(a, p.table, a.eager_slot(p) + 16 * (wave / DS), a.c.capacity - 1, lane);
  a.place_slots(&p);
  if (p.begin >= p.end) return a.template leave_none<HD>(p);  // (the whole workgroup)
  uint32_t t = p.begin + 16 * (wave / DS);
  f4_t kf[KP], vf[4][VP];
  auto load_k = [&](int buf) {
    const uint8_t* src = a.c.k + rows.s[buf][n] + G * 16 + share * (HW * 4);
#pragma unroll
    for (int c = 0; c < KP; ++c) kf[c] = gld(reinterpret_cast<const f4_t*>(src + 64 * c));
  };
  auto load_v = [&](int buf) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint8_t* src = a.c.v + rows.s[buf][4 * G + r] + n * 16 + share * (HW * 4);
#pragma unroll
      for (int c = 0; c < VP; ++c) vf[r][c] = ld_once(reinterpret_cast<const f4_t*>(src + 256 * c));
    }
  };
  if (!a.eager()) rows.next(a, p.table, t, p.end - 1, lane);
  const bool head = uint32_t(n) < p.nh;
  constexpr int QW = HD / 16 / kWaves;
  f4_t x[QW];  // the wave's share of the queries
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    const float4 q = ld_f4(a.template query<HD>(p, head ? n : 0) + G * 4 + 16 * (i * kWaves + wave));
    x[i] = f4_t{q.x, q.y, q.z, q.w};
  }
  int buf = 0;
  if (t < p.end) {
    rows.put(a, p, 0, lane);
    load_k(0);
    load_v(0);
    rows.next(a, p.table, t + UNIT, p.end - 1, lane);
  }
#pragma unroll
  for (int i = 0; i < QW; ++i) s_q[i * kWaves + wave][lane] = head ? x[i] : f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  __syncthreads();  // (the queries)
  const float mult = a.scale * kLog2e;
  float m = -INFINITY, l = 0.0f;
  f4_t o[VD];
#pragma unroll
  for (int j = 0; j < VD; ++j) o[j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};

  // (where waves share a tile, all waves of the workgroup take the same number of steps)
  for (uint32_t t0 = p.begin; (DS > 1 ? t0 : t) < p.end; t0 += UNIT, t += UNIT) {
    const bool here = DS == 1 || t < p.end, more = t + UNIT < p.end;
    asm volatile("" ::: "memory");  // (the queries are read from LDS anew: they would fill the registers)
    f4_t sc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (here) {
      // four sums, added in pairs: one sum of all dims in turn was off by three times as much
      f4_t part[4] = {sc, sc, sc, sc};
#pragma unroll
      for (int c = 0; c < KP; ++c) {
        const f4_t q = s_q[share * KP + c][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c][e], q[e], part[e], 0, 0, 0);
      }
      sc = (part[0] + part[1]) + (part[2] + part[3]);
      if constexpr (DS > 1) s_u.share[(buf * kWaves + wave) * 64 + lane] = sc;
    }
    buf ^= 1;
    if (more) {
      rows.put(a, p, buf, lane);
      load_k(buf);
      rows.next(a, p.table, t + 2 * UNIT, p.end - 1, lane);
    }
    if constexpr (DS > 1) {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      if (!here) continue;
      sc += s_u.share[((buf ^ 1) * kWaves + (wave ^ 1)) * 64 + lane];
    }
    float s4[4], top[4], mx = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top[i] = t + 4 * G + i < p.end ? sc[i] * mult : -INFINITY;
      mx = fmaxf(mx, top[i]);
    }
    if constexpr (Args::kScores) {
      if (a.scores && share == 0 && head)
        *reinterpret_cast<float4*>(a.scores + (size_t(p.row) * a.H + p.h0 + n) * a.score_stride + (t - p.lo) + 4 * G) =
            make_float4(top[0], top[1], top[2], top[3]);
    }
    mx = pair_max(pair_max(mx, 16), 32);
    float base = mx == -INFINITY ? 0.0f : mx;
    const float f = __builtin_amdgcn_exp2f(m - base);
    if (__ballot(f != 1.0f) != 0) {
      l *= f;
#pragma unroll
      for (int j = 0; j < VD; ++j) o[j] *= f;
    }
    m = mx;
    float mu = mult;
#pragma unroll
    for (int i = 0; i < 4; ++i) s4[i] = sc[i];
    far_scores(s4, mu, base);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s4[i] = __builtin_amdgcn_exp2f(top[i] > -INFINITY ? fmaf(s4[i], mu, -base) : top[i]);
      l += s4[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VD; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[i][j / 4][j % 4], s4[i], o[j], 0, 0, 0);
    if (more) load_v(buf);
  }
  l = pair_sum(pair_sum(l, 16), 32);
  if (__ballot(rows.bad) != 0) l = __builtin_nanf("");
  if (DS > 1) __syncthreads();  // (s_u)
  leave<HD, float, 4, 64>(a, p, s_u.sums, tid, wave, G, n, true, 0, m, l, o);
}

}  // namespace
}  // namespace chpe
