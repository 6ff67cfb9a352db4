// paged_attention.hip -- chpe_paged_attention: the attention of one new token per row over the paged
// cache.  s_j = scale q.k_j over the row's slots lo <= j < len, p = softmax(s), out = sum_j p_j v_j, and,
// for a cache that is kept to a budget, each slot's p summed over the query heads of its kv head.
// A row's slots are split over workgroups: each leaves its maximum, sum of 2^(s - max) and so weighted sum of V
// rows, and a second launch rescales and joins them (and turns the scores into weights).
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace chpe {
namespace {
using namespace dev;

constexpr int kWaves = 4;  // of a workgroup

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
  uint32_t rows, H, max_len, window, score_stride;
  uint32_t hz, splits, chunk;     // groups of HT query heads of a kv head; splits of `chunk` slots
  float scale;
};

// the row's slots lo .. len - 1; false for a length outside 0 .. max_len
__device__ __forceinline__ bool row_range(const PagedAttnArgs& a, uint32_t row, uint32_t* lo, uint32_t* len) {
  const uint32_t n = uint32_t(gld(a.lens + row));
  *len = n <= a.max_len ? n : 0u;
  *lo = a.window != 0 && *len > a.window ? *len - a.window : 0u;
  return n <= a.max_len;
}

// ---- the splits ------------------------------------------------------------------------------------------------
// a workgroup's place: slots begin .. end - 1 of row `row`, whose range is lo .. len - 1, for query heads
// h0 .. h0 + nh - 1
struct Place {
  uint32_t row, kvh, h0, nh, split, begin, end, lo, len;
  bool ok;
};
template <int HT>
__device__ __forceinline__ Place place_of(const PagedAttnArgs& a) {
  Place p;
  const uint32_t gq = a.H / a.c.KV;
  uint32_t b = blockIdx.x;
  // the rows' last splits, which short rows do not have, on other XCDs for other items (workgroup i runs on
  // XCD i % 8: with 8 splits one XCD had all of them, and f32 rows of up to 2304 slots took 47 us instead of 33)
  p.split = (b + b / a.splits) % a.splits;
  b /= a.splits;
  const uint32_t z = b % a.hz;
  b /= a.hz;
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
// a split without slots: nothing for the join (it goes by the row's length); the output of a row of one
// split at most
template <int HD>
__device__ __forceinline__ void leave_none(const PagedAttnArgs& a, const Place& p) {
  if (a.splits != 1) return;
  const float v = p.ok ? 0.0f : __builtin_nanf("");
  for (uint32_t i = threadIdx.x; i < p.nh * HD; i += kWaves * 64) a.out[p.row * a.out_stride + size_t(p.h0) * HD + i] = v;
}

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

// The tile's row offsets (bytes from k or v): lane r of the wave finds row r's page and leaves the
// offset in LDS for the lanes that load the row.  `next` requests the table entry ahead of its use; for the
// first tile of a range that starts at slot 0 it does not wait for the row's length (entries behind it may
// hold anything).  Rows behind the split's end are its last row.
template <int ROWS, int ES>
struct TileRows {
  uint64_t (*s)[ROWS];
  uint32_t id, slot;
  bool bad;
  __device__ void next(const PagedAttnArgs& a, uint32_t row, uint32_t t, uint32_t last, int lane) {
    slot = min(t + uint32_t(lane % ROWS), last);
    id = uint32_t(gld(a.c.table + size_t(row) * a.c.table_stride + (slot >> a.c.shift)));
  }
  __device__ void put(const PagedAttnArgs& a, const Place& p, int buf, int lane) {
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
template <class T>
__device__ __forceinline__ f4_t non_finite_sum(const PagedAttnArgs& a, const Place& p, uint32_t dim, f4_t v) {
  f4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t j = p.begin; j < p.end; ++j) {
    uint32_t page;
    a.c.page_of(p.row, j, &page);  // (a bad one: the head's sum of weights is NaN and nothing comes here)
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
template <int HD, class T, int E, int LANES, int VD>
__device__ __forceinline__ void leave(const PagedAttnArgs& a, const Place& p, WaveSums<LANES>& s, int tid, int wave, int G,
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
  const size_t pt = (size_t(p.row) * a.H + p.h0 + head) * a.splits + p.split;
  const bool whole = a.splits == 1;
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

template <int HD, class T, int W, int NT>
__global__ void __launch_bounds__(kWaves * 64, NT == 1 ? (HD == 64 ? 4 : 3) : (HD == 64 ? 3 : 2)) k_paged_16(PagedAttnArgs a) {
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
  Place p = place_of<HT>(a);
  TileRows<32, 2> rows{s_off[wave], 0, 0, false};
  if (a.window == 0) rows.next(a, p.row, p.split * a.chunk + 32 * (wave / DS), a.c.capacity - 1, lane);
  place_slots(a, &p);
  if (p.begin >= p.end) return leave_none<HD>(a, p);  // (the whole workgroup)
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
  if (a.window != 0) rows.next(a, p.row, t, p.end - 1, lane);
  // the queries: HD / 8 threads a head take 8 dims each (dims (G + 4 s) * 8 .. + 7 are what lanes of group G
  // need in step s); they are taken apart while the first tile's rows are on their way
  constexpr int TH = HD / 8;
  const int qh = tid / TH, qc = tid % TH;
  float x[8];
  if (qh < HT) {
    const float* src = a.q + p.row * a.q_stride + size_t(p.h0 + (qh < int(p.nh) ? qh : 0)) * HD + qc * 8;
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
    rows.next(a, p.row, t + UNIT, p.end - 1, lane);
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
      rows.next(a, p.row, t + 2 * UNIT, p.end - 1, lane);
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
      if (a.scores && share == 0 && part == 0 && ht * W + col < p.nh) {
        float* d = a.scores + (size_t(p.row) * a.H + p.h0 + ht * W + col) * a.score_stride + (t - p.lo) + 4 * G;
        *reinterpret_cast<float4*>(d) = make_float4(top[0], top[1], top[2], top[3]);
        *reinterpret_cast<float4*>(d + 16) = make_float4(top[4], top[5], top[6], top[7]);
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
        // (the product again inside the fma: rounded once, as small as the difference is)
        s8[e] = __builtin_amdgcn_exp2f(top[e] > -INFINITY ? fmaf(s8[e], mult[ht], -base) : top[e]);
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
template <int HD>
__global__ void __launch_bounds__(kWaves * 64, HD == 64 ? 4 : 3) k_paged_32(PagedAttnArgs a) {
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
  Place p = place_of<16>(a);
  TileRows<16, 4> rows{s_off[wave], 0, 0, false};
  if (a.window == 0) rows.next(a, p.row, p.split * a.chunk + 16 * (wave / DS), a.c.capacity - 1, lane);
  place_slots(a, &p);
  if (p.begin >= p.end) return leave_none<HD>(a, p);  // (the whole workgroup)
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
  if (a.window != 0) rows.next(a, p.row, t, p.end - 1, lane);
  const bool head = uint32_t(n) < p.nh;
  constexpr int QW = HD / 16 / kWaves;
  f4_t x[QW];  // the wave's share of the queries
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    const float4 q = ld_f4(a.q + p.row * a.q_stride + size_t(p.h0 + (head ? n : 0)) * HD + G * 4 + 16 * (i * kWaves + wave));
    x[i] = f4_t{q.x, q.y, q.z, q.w};
  }
  int buf = 0;
  if (t < p.end) {
    rows.put(a, p, 0, lane);
    load_k(0);
    load_v(0);
    rows.next(a, p.row, t + UNIT, p.end - 1, lane);
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
      rows.next(a, p.row, t + 2 * UNIT, p.end - 1, lane);
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
    if (a.scores && share == 0 && head)
      *reinterpret_cast<float4*>(a.scores + (size_t(p.row) * a.H + p.h0 + n) * a.score_stride + (t - p.lo) + 4 * G) =
          make_float4(top[0], top[1], top[2], top[3]);
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
      s4[i] = __builtin_amdgcn_exp2f(top[i] > -INFINITY ? fmaf(sc[i], mult, -base) : top[i]);
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

// ---- joining the splits, and the slots' weights -------------------------------------------------------------
// the row's splits that hold slots
__device__ __forceinline__ uint32_t splits_of(const PagedAttnArgs& a, uint32_t lo, uint32_t len) {
  return (len - lo + a.chunk - 1) / a.chunk;
}

// maximum and sum over a head's splits, by one wave
__device__ __forceinline__ void join_ml(const PagedAttnArgs& a, uint32_t item, uint32_t ns, int lane, float* M, float* L) {
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + size_t(item) * a.splits;
  float2 x = ml[min(uint32_t(lane), a.splits - 1)];  // (does not wait for the row's length)
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

// Bound by latency: the lengths, the statistics and the sums, one after the other (64 heads of 86 splits 4.8 us,
// 4096 heads of 9 splits 9.6 us; with the weights of 24 rows of up to 4097 slots 9.4 us).
// blocks 0 .. joins - 1: the output of one (row, query head) each, 256 / (HD / 4) splits at a time;
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
      const float4 v = ld_f4(acc + size_t(min(uint32_t(tid / D4 + u * GR), a.splits - 1)) * HD);
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
      v = !ok ? __builtin_nanf("") : (L == 0.0f ? 0.0f : v / L);
      if (!(fabsf(v) < INFINITY) && ok && L == L) {
        // an infinite sum counts whatever its split's factor, which may be 0
        float inf = 0.0f;
        for (uint32_t s = 0; s < ns; ++s) {
          const float x = gld(a.part_acc + (size_t(item) * a.splits + s) * HD + tid);
          inf += fabsf(x) < INFINITY ? 0.0f : x;
        }
        if (inf != 0.0f) v = inf;
      }
      a.out[row * a.out_stride + size_t(h) * HD + tid] = v;
    }
    return;
  }
  const uint32_t b = blockIdx.x - joins, part = b % weight_parts, kv = b / weight_parts;
  const uint32_t kvh = kv % a.c.KV, row = kv / a.c.KV, gq = a.H / a.c.KV;
  row_range(a, row, &lo, &len);
  const uint32_t first = part * 1024, i = first + tid * 4;  // slots lo + i .. + 3
  const size_t base = (size_t(row) * a.c.KV + kvh) * a.weight_stride;
  // slots before the window were given nothing
  for (uint32_t j = first + tid; j < min(first + 1024, lo); j += 256) a.weight_out[base + j] = a.weight_in ? a.weight_in[base + j] : 0.0f;
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
// query heads a workgroup serves: of the 16 columns one holds a head of an f32 cache, two or (bf16, up to 4
// heads) four one of a 16-bit cache; two such tiles of heads where the accumulators of both fit the registers
uint32_t heads_per_group(const chpe_kv_pages* c, uint32_t heads) {
  const uint32_t gq = heads / c->kv_heads;
  if (c->type == 0 || (gq > 8 && c->head_dim <= kWaveDims)) return 16;
  return c->type == 2 && gq <= 4 ? 4 : 8;
}

struct AttnPlan {
  bool ok = false;  // the launches fit
  uint32_t ht = 0, hz = 0, splits = 1, chunk = 1, score_stride = 0, joins = 0, weight_parts = 0;
  uint64_t blocks = 0, joined = 0;
  size_t off_acc = 0, off_scores = 0, bytes = 0;
};

// How the rows are split: into about 1024 workgroups where the rows are few (4 a CU: a long row alone takes
// 28.6 us over 32771 slots of 4 KB; with 1536 workgroups 30.8), and into splits of at most 512 KB where they
// are many, so that rows of different lengths keep the chip busy to the end (64 rows of up to 8320 slots: 207 us
// with 512 KB, 204 to 211 with 768 KB, 238 with 256 KB).  Between 512 and 768 KB neither wins everywhere: over twelve
// batches of 24 to 200 rows of all types 768 took 0.82 to 1.17 of the time, 0.98 in the mean, by how the number of
// splits meets that of the workgroups that the chip holds.  A row's split depends on max_len and the number of rows,
// not on the other rows' lengths.  (Dealing all rows' tiles out in equal runs over the workgroups that the chip
// holds took as long on f32 and 5 to 25 % longer on 16-bit caches: finding the place costs 2 us and the slowest
// run ends the launch.)
AttnPlan attn_plan(const chpe_kv_pages* c, uint32_t heads, uint32_t max_len, uint32_t window, bool weights) {
  AttnPlan p;
  const uint32_t gq = heads / c->kv_heads, step = (c->type == 0 ? 16 : 32) * tiles_at_once(c->head_dim);
  p.ht = heads_per_group(c, heads);
  p.hz = (gq + p.ht - 1) / p.ht;
  const uint64_t items = uint64_t(c->rows) * c->kv_heads * p.hz, some = std::max<uint64_t>(1, items);
  const uint64_t large = (512 << 10) / (2 * c->head_dim * (c->type == 0 ? 4 : 2));  // slots
  auto most = [&](uint32_t range) {
    const uint64_t steps = std::max<uint64_t>(1, (uint64_t(range) + step - 1) / step);
    const uint64_t want = std::max<uint64_t>((1024 + some - 1) / some, (uint64_t(range) + large - 1) / large);
    return std::min<uint64_t>(std::min<uint64_t>(want, steps), kMaxSplits);
  };
  // (items <= heads_in_all)
  const uint64_t heads_in_all = uint64_t(c->rows) * heads;
  p.weight_parts = weights ? (max_len + 1023) / 1024 : 0;
  const uint64_t weight_blocks = uint64_t(c->rows) * c->kv_heads * p.weight_parts;
  if (heads_in_all > kMaxBlocks || weight_blocks > kMaxBlocks) return p;
  const uint32_t range = window != 0 && window < max_len ? window : max_len;
  const uint64_t steps = std::max<uint64_t>(1, (uint64_t(range) + step - 1) / step), fit = kMaxBlocks / some;
  uint64_t per = (steps + most(range) - 1) / most(range);
  if ((steps + per - 1) / per > fit) per = (steps + fit - 1) / fit;  // (more than a launch holds: longer splits)
  p.chunk = uint32_t(per * step);
  p.splits = uint32_t((steps + per - 1) / per);
  p.blocks = items * p.splits;
  p.joins = p.splits > 1 ? uint32_t(heads_in_all) : 0;
  p.joined = p.joins + weight_blocks;
  p.ok = p.joined <= kMaxItems / 256;
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  // the workspace does not depend on the window: `most` grows with the range
  const size_t places = size_t(c->rows) * heads * most(max_len);
  p.off_acc = up(places * 8);
  p.off_scores = p.off_acc + up(places * c->head_dim * 4);
  p.score_stride = uint32_t((max_len + 63) / 64 * 64);
  p.bytes = p.off_scores + (weights ? up(size_t(c->rows) * heads * p.score_stride * 4) : 0);
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
  const AttnPlan plan = attn_plan(cache, heads, max_len, 0, weights != 0);
  return plan.ok ? plan.bytes : 0;
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
  if (!p.ok) return -1;
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
  a.hz = p.hz;
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.scale = scale;
  a.score_stride = p.score_stride;
  const int type = cache->type;
  const uint32_t hd = cache->head_dim;
  bool ok = hd == 64    ? launch_partial<64>(a, type, p.ht, p.blocks, st)
            : hd == 128 ? launch_partial<128>(a, type, p.ht, p.blocks, st)
                        : launch_partial<256>(a, type, p.ht, p.blocks, st);
  if (ok && p.joined != 0)
    ok = hd == 64    ? launch(&k_paged_join<64>, p.joined, 256, st, a, p.joins, p.weight_parts)
         : hd == 128 ? launch(&k_paged_join<128>, p.joined, 256, st, a, p.joins, p.weight_parts)
                     : launch(&k_paged_join<256>, p.joined, 256, st, a, p.joins, p.weight_parts);
  return ok ? 0 : -3;
}
