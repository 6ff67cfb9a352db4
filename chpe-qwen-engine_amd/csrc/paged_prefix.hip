// paged_prefix.hip -- chpe_paged_prefix_attention: the attention of one new token per row where groups of rows share
// the first slots of their cache.  The softmax over a row's slots is joined from parts, so a group's prefix is read
// once for the queries of all its rows (as if they were query heads of one row), the rest of a row for its own, both in one
// launch, and a second one joins them: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the parts s of a row.
#include "paged_attention_kernels.hpp"

namespace chpe {
namespace {
using namespace dev;

struct PrefixArgs {
  Pages c;
  const float* q;
  const int32_t *lens, *group_rows, *prefix_lens;
  float *out, *part_ml, *part_acc;  // parts: [row][head][prefix splits, rest splits]
  uint64_t q_stride, out_stride;
  uint32_t rows, H, groups, max_prefix, max_rest;
  uint32_t prefix_splits, prefix_chunk, prefix_blocks, rest_splits, rest_chunk, step, hz;
  float scale;

  static constexpr bool kScores = false;
  __device__ bool eager() const { return false; }
  __device__ uint32_t eager_slot(const Place&) const { return 0; }
  __device__ bool whole() const { return false; }
  template <int HD>
  __device__ void leave_none(const Place&) const {}  // (the join goes by the lengths)

  // group g's rows r0 .. r1 - 1 and prefix; false where they do not lie in the rows, or in max_prefix
  __device__ bool group(uint32_t g, uint32_t* r0, uint32_t* r1, uint32_t* prefix) const {
    *r0 = uint32_t(gld(group_rows + g));
    *r1 = uint32_t(gld(group_rows + g + 1));
    *prefix = uint32_t(gld(prefix_lens + g));
    return *r0 <= *r1 && *r1 <= rows && *prefix <= max_prefix;
  }
  // the last group of which `first`(its first row, its number) <= x, 64 candidates a step; -1: none
  template <class F>
  __device__ int last_group(uint32_t x, F first) const {
    if (groups == 0) return -1;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t at = 0, n = groups;
    do {
      const uint32_t step = (n + 63) / 64, g = at + min(lane * step, n - 1);
      const uint64_t in = __ballot(lane * step < n && first(uint32_t(max(gld(group_rows + g), 0)), g) <= x);
      if (in == 0) return -1;
      const uint32_t last = 63u - uint32_t(__builtin_clzll(in));
      at += last * step;
      n = min(step, n - last * step);
    } while (n > 1);
    return int(at);
  }
  // What is joined of a row: `shared` splits of its group's prefix, then slots lo .. len - 1 in splits of `chunk`, in the
  // pages of row `table`: its own slots in its own, or, for a row shorter than its prefix, what it sees of that (the
  // prefix's sums hold slots that are not the row's, and an infinity there could not be taken out again).  false for a
  // length or a group that is not valid.
  struct Row {
    uint32_t shared, lo, len, chunk, table;
  };
  __device__ bool row_parts(uint32_t row, Row* r) const {
    const int g = last_group(row, [](uint32_t r, uint32_t) { return r; });
    uint32_t r0 = row, r1 = 0, prefix = 0;
    bool ok = true;
    if (g >= 0) {
      ok = group(g, &r0, &r1, &prefix);
      if (int(r0) <= int(r1) && int(r1) <= int(row)) {  // (behind the group, whatever else it holds: in none)
        ok = true;
        prefix = 0;
      }
    }
    const uint32_t len = uint32_t(gld(lens + row));
    *r = Row{(prefix + prefix_chunk - 1) / prefix_chunk, prefix, len, rest_chunk, row};
    if (len < prefix) {
      const uint32_t steps = (len + step - 1) / step;
      *r = Row{0, 0, len, max(1u, (steps + rest_splits - 1) / rest_splits) * step, r0};
    }
    return ok && len <= 0x7fffffffu && (len <= prefix || len - prefix <= max_rest);
  }
};

// The parts.  A workgroup's queries are HT of the query heads of one kv head, row by row: of all rows of a group for a split
// of its prefix (blocks up to prefix_blocks), of one row for a split of its own slots.  A launch does not know the
// groups' sizes: group g's tiles of queries have the numbers from (its first row) * gq / HT + g on (a first row behind the rows
// counts as the one behind the last: its number lies above those of all rows, and none passes 32 bits).
struct PartArgs : PrefixArgs {
  __device__ void at(const Place& p, uint32_t i, uint32_t* row, uint32_t* head) const {
    const uint32_t gq = H / c.KV, x = p.h0 + min(i, p.nh - 1);
    *row = p.row + x / gq;
    *head = p.kvh * gq + x % gq;
  }
  template <int HD>
  __device__ const float* query(const Place& p, uint32_t i) const {
    uint32_t row, head;
    at(p, i, &row, &head);
    return q + row * q_stride + size_t(head) * HD;
  }
  __device__ size_t part_of(const Place& p, uint32_t i) const {
    uint32_t row, head;
    at(p, i, &row, &head);
    return (size_t(row) * H + head) * (prefix_splits + rest_splits) + p.split;
  }
  template <int HT>
  __device__ Place place_of() const {
    Place p;
    const uint32_t gq = H / c.KV;
    uint32_t b = blockIdx.x;
    p.lo = 0;
    p.ok = b < prefix_blocks;
    if (p.ok) {
      p.split = b % prefix_splits;
      b /= prefix_splits;
      p.kvh = b % c.KV;
      b /= c.KV;
      auto first = [&](uint32_t r, uint32_t g) { return uint32_t(uint64_t(min(r, rows)) * gq / HT) + g; };
      const int g = last_group(b, first);
      uint32_t r0 = 0, r1 = 0, prefix = 0;
      const bool there = g >= 0 && group(g, &r0, &r1, &prefix);
      const uint32_t n = there ? (r1 - r0) * gq : 0u, h0 = there ? (b - first(r0, g)) * HT : 0u;
      p.row = p.table = h0 < n ? r0 : 0u;
      p.h0 = h0 < n ? h0 : 0u;
      p.nh = h0 < n ? min(uint32_t(HT), n - h0) : 1u;
      p.len = h0 < n ? prefix : 0u;
      return p;
    }
    b -= prefix_blocks;
    p.split = (b + b / rest_splits) % rest_splits;  // (the last ones not all on one XCD)
    b /= rest_splits;
    const uint32_t z = b % hz;
    b /= hz;
    p.kvh = b % c.KV;
    p.row = b / c.KV;
    p.h0 = z * HT;
    p.nh = min(uint32_t(HT), gq - z * HT);
    return p;
  }
  __device__ void place_slots(Place* p) const {
    if (p->ok) {
      p->begin = p->split * prefix_chunk;
      p->end = min(p->len, p->begin + prefix_chunk);
      return;
    }
    Row r;
    const bool ok = row_parts(p->row, &r);
    p->table = r.table;
    p->lo = r.lo;
    p->begin = r.lo + p->split * r.chunk;
    p->end = ok ? min(r.len, p->begin + r.chunk) : 0u;
    p->split += prefix_splits;
  }
};

// ---- many queries ---------------------------------------------------------------------------------------------------
// Where a group has more queries than a few: a wave keeps 16 QT of them as columns (QT = 2, at head dim 256 1), with
// their parts as operands in registers, and the four waves of a workgroup share every 32 slots' K and V in LDS, the next
// 32 on the way.  S^T = K . Q^T and O^T = V^T . P^T as in k_paged_16: a lane's column is a query in both, the scores' layout is
// the weights'; V's rows become operands with slots inside by the transposing reads of LDS.
// k_paged_16 reads each K and V row once per 16 queries, and every lane pair forms a score's weight twice: 64 rows of 8
// query heads behind 8192 fp16 slots took 116 us there (1.1 GB through the CUs' caches at 27 bytes a cycle each, 65 us, and
// 50 us of vector instructions).
// Now 57 to 59 us, 0.6 PFLOP/s with the queries' and weights' two parts (bf16, three: 74).  Two workgroups a CU; for 32 slots of one a SIMD's matrix cores
// are busy 1024 cycles and its vector ALU about 1000 (softmax, parts, addresses), which the two overlap in part: 1800 cycles.
// A workgroup's own start (group, page numbers, K, V and queries behind each other) and end are 8 us.
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));
template <class T>
struct ManyParts;
template <>
struct ManyParts<_Float16> {
  static constexpr int N = 2, kScaleExp = 15;  // (22 bits, x brought near 2^14: Parts<_Float16, 8>)
  static __device__ void split(const float (&x)[8], u32x4_t (&out)[N]) {
    h8_t hi, lo;
    float one = -1.0f;
    asm("" : "+v"(one));  // (a product with it takes the 16 bits as they are: without it they are widened first)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const h2_t h = __builtin_convertvector((f2_t{x[e], x[e + 1]}), h2_t);
      const f2_t r = {fmaf(float(h.x), one, x[e]), fmaf(float(h.y), one, x[e + 1])};
      const h2_t l = __builtin_convertvector(r, h2_t);
      hi[e] = h.x, hi[e + 1] = h.y;
      lo[e] = l.x, lo[e + 1] = l.y;
    }
    out[0] = __builtin_bit_cast(u32x4_t, hi);
    out[1] = __builtin_bit_cast(u32x4_t, lo);
  }
  static __device__ f4_t mfma(u32x4_t a, u32x4_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
  }
};
template <>
struct ManyParts<Bf16> {
  static constexpr int N = 3, kScaleExp = 0;  // (all 24 bits)
  static __device__ void split(const float (&x)[8], u32x4_t (&out)[N]) {
    b8_t a, b, c;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = __bf16(x[e]);
      const float r = x[e] - float(a[e]);
      b[e] = __bf16(r);
      c[e] = __bf16(r - float(b[e]));
    }
    out[0] = __builtin_bit_cast(u32x4_t, a);
    out[1] = __builtin_bit_cast(u32x4_t, b);
    out[2] = __builtin_bit_cast(u32x4_t, c);
  }
  static __device__ f4_t mfma(u32x4_t a, u32x4_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
  }
};
constexpr int many_tiles(int hd) { return hd == 256 ? 1 : 2; }
constexpr int many_queries(int hd) { return 64 * many_tiles(hd); }

template <int HD, class T>
__global__ void __launch_bounds__(256, 2) k_prefix_many(PartArgs a) {
  using P = ManyParts<T>;
  constexpr int NP = P::N, QT = many_tiles(HD), KS = HD / 32, VD = HD / 16;
  constexpr int CPR = HD / 8, RPP = 256 / CPR, PASS = 32 / RPP;  // 16-byte pieces of a row; rows a pass of the workgroup loads
  constexpr int KROW = CPR + 1, VROW = CPR + 2;                  // (room so that neither side's reads meet in a few banks)
  __shared__ u32x4_t s_k[2][32][KROW], s_v[2][32][VROW];
  __shared__ int s_bad;
  const int wave = uniform(threadIdx.x >> 6), tid = threadIdx.x, lane = tid & 63, G = lane >> 4, n = lane & 15;
  Place p = a.template place_of<many_queries(HD)>();
  a.place_slots(&p);
  if (p.begin >= p.end) return;  // (the whole workgroup)
  if (tid == 0) s_bad = 0;
  // the thread's pieces of a tile's rows
  const int piece = tid % CPR, row0 = tid / CPR;
  uint32_t id[PASS];
  bool bad = false;
  u32x4_t kr[PASS], vr[PASS];
  auto ids = [&](uint32_t t) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const uint32_t slot = min(t + uint32_t(row0 + RPP * i), p.end - 1);
      id[i] = uint32_t(gld(a.c.table + size_t(p.table) * a.c.table_stride + (slot >> a.c.shift)));
    }
  };
  auto load = [&](uint32_t t) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const uint32_t slot = min(t + uint32_t(row0 + RPP * i), p.end - 1);
      const bool in = id[i] < a.c.n_pages;
      bad |= !in;
      const size_t at = a.c.at(in ? id[i] : 0u, p.kvh, slot) * 2 + piece * 16;
      kr[i] = gld(reinterpret_cast<const u32x4_t*>(a.c.k + at));
      vr[i] = gld(reinterpret_cast<const u32x4_t*>(a.c.v + at));
    }
  };
  auto leave = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      s_k[buf][row0 + RPP * i][piece] = kr[i];
      s_v[buf][row0 + RPP * i][piece] = vr[i];
    }
  };
  uint32_t t = p.begin;
  ids(t);
  load(t);
  if (t + 32 < p.end) ids(t + 32);
  // the queries: lane (G, n) has dims 32 s + 8 G .. of query n
  const uint32_t q0 = wave * 16 * QT;
  const bool idle = q0 >= p.nh;  // (a wave without queries loads and waits with the others)
  u32x4_t qf[QT][KS][NP];
  float mult[QT], m[QT], l[QT];
  f4_t o[QT][VD];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const uint32_t i = q0 + 16 * qt + n;
    const float* src = a.template query<HD>(p, i) + 8 * G;  // (behind the last query: that one again, not used)
    float x[KS][8], top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float4 u = ld_f4(src + 32 * s), v = ld_f4(src + 32 * s + 4);
      const float w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[s][e] = w[e];
        top = fmaxf(top, fabsf(w[e]));
      }
    }
    int ex = 0;
    if constexpr (P::kScaleExp != 0) {
      top = pair_max(pair_max(top, 16), 32);
      if (top > 0.0f && top < INFINITY) ex = 14 - __builtin_amdgcn_frexp_expf(top);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[s][e] = __builtin_amdgcn_ldexpf(a.scale < 0.0f ? -x[s][e] : x[s][e], ex);
      P::split(x[s], qf[qt][s]);
    }
    mult[qt] = __builtin_amdgcn_ldexpf(fabsf(a.scale) * kLog2e, -ex);
    if (mult[qt] == 0.0f) mult[qt] = 1e-38f;  // (what scores come to stays 0; -inf behind the end stays -inf)
    m[qt] = -INFINITY;
    l[qt] = 0.0f;
#pragma unroll
    for (int j = 0; j < VD; ++j) o[qt][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  leave(0);
  if (t + 32 < p.end) {
    load(t + 32);
    if (t + 64 < p.end) ids(t + 64);
  }
  lds_barrier();
  for (int buf = 0; t < p.end; t += 32, buf ^= 1) {
    if (t + 32 < p.end) {
      leave(buf ^ 1);
      if (t + 64 < p.end) {
        load(t + 64);
        if (t + 96 < p.end) ids(t + 96);
      }
    }
    if (!idle) {
      f4_t sc[QT][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4_t kf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[s] = s_k[buf][16 * u + n][4 * s + G];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) sc[qt][u] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) sc[qt][u] = P::mfma(kf[s], qf[qt][s][i], sc[qt][u]);
      }
      u32x4_t pf[QT][NP];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        // weights are 2^(x mult - m + kScaleExp), m the largest x mult so far rounded up: a whole number, so that what older sums
        // are multiplied by is exact, and 1 most of the time
        float x[8], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = sc[qt][e >> 2][e & 3];
        if (t + 32 > p.end) {  // (uniform: the last tile)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = t + (e >> 2) * 16 + 4 * G + (e & 3) < p.end ? x[e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, x[e]);
        mx = fmaxf(m[qt], ceilf(pair_max(pair_max(mx, 16), 32) * mult[qt]));
        if (__ballot(mx != m[qt]) != 0) {
          const float f = m[qt] > -INFINITY ? __builtin_amdgcn_exp2f(m[qt] - mx) : 0.0f;
          l[qt] *= f;
#pragma unroll
          for (int j = 0; j < VD; ++j) o[qt][j] *= f;
        }
        m[qt] = mx;
        float mu = mult[qt], base = mx == -INFINITY ? 0.0f : mx;
        far_scores(x, mu, base);
        const float less = float(P::kScaleExp) - base;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], mu, less));
          l[qt] += x[e];
        }
        P::split(x, pf[qt]);
      }
#pragma unroll
      for (int j = 0; j < VD; ++j) {
        // lane n of a group of 16 names 4 dims of slot n / 4 and gets dim n of the four slots
        const u32x2_t lo = ld_transposed(reinterpret_cast<const u32x2_t*>(&s_v[buf][4 * G + n / 4][2 * j]) + n % 4);
        const u32x2_t hi = ld_transposed(reinterpret_cast<const u32x2_t*>(&s_v[buf][16 + 4 * G + n / 4][2 * j]) + n % 4);
        const u32x4_t vf = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) o[qt][j] = P::mfma(vf, pf[qt][i], o[qt][j]);
      }
    }
    lds_barrier();
  }
  if (__ballot(bad) != 0 && lane == 0) s_bad = 1;
  lds_barrier();
  if (idle) return;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const uint32_t i = q0 + 16 * qt + n;
    float L = pair_sum(pair_sum(l[qt], 16), 32) * (1.0f / float(1 << P::kScaleExp));
    if (s_bad != 0) L = __builtin_nanf("");
    if (i >= p.nh) continue;
    const size_t pt = a.part_of(p, i);
    if (G == 0) reinterpret_cast<float2*>(a.part_ml)[pt] = make_float2(m[qt], L);
    bool finite = true;
#pragma unroll
    for (int j = 0; j < VD; ++j) {
      const f4_t v = o[qt][j] * (1.0f / float(1 << P::kScaleExp));
      finite &= all_finite(v);
      *reinterpret_cast<f4_t*>(a.part_acc + pt * HD + 16 * j + 4 * G) = v;
    }
    if (finite || L != L) continue;
#pragma unroll 1
    for (int j = 0; j < VD; ++j) {
      f4_t* d = reinterpret_cast<f4_t*>(a.part_acc + pt * HD + 16 * j + 4 * G);
      const f4_t v = *d;
      if (!all_finite(v)) *d = non_finite_sum<T>(a, p, 16 * j + 4 * G, v);
    }
  }
}

// ---- the join: a workgroup per (row, query head), 256 / (HD / 4) parts at a time.  Bound by latency for few rows (5 rows
// 3.2 us), by the parts' bytes for many (64 rows of 64 heads of 128, 14 parts each, 30 MB: 9.8 us) ---------------------------------
template <int HD>
__global__ void __launch_bounds__(256) k_prefix_join(PrefixArgs a) {
  constexpr int D4 = HD / 4, GR = 256 / D4;
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t h = blockIdx.x % a.H, row = blockIdx.x / a.H;
  __shared__ __align__(16) float s_o[GR][HD];
  __shared__ float s_f[2 * kMaxSplits];
  PrefixArgs::Row r;
  const bool ok = a.row_parts(row, &r);
  const uint32_t np = ok ? r.shared : 0u, ns = np + (ok && r.len > r.lo ? (r.len - r.lo + r.chunk - 1) / r.chunk : 0u);
  const size_t base = size_t(blockIdx.x) * (a.prefix_splits + a.rest_splits);
  auto place = [&](uint32_t s) { return base + (s < np ? s : a.prefix_splits + (s - np)); };
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  float M = -INFINITY, L = 0.0f;  // (every wave for itself)
  for (uint32_t s = lane; s < ns; s += 64) M = fmaxf(M, ml[place(s)].x);
  M = wave_max(M);
  if (M == -INFINITY) M = 0.0f;  // (no score above -inf)
  for (uint32_t s = lane; s < ns; s += 64) {
    const float2 x = ml[place(s)];
    const float f = __builtin_amdgcn_exp2f(x.x - M);
    L += x.y * f;
    if (tid < 64) s_f[s] = f;
  }
  L = wave_sum(L);
  __syncthreads();
  f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t s = tid / D4; s < ns; s += GR) {
    const float4 v = ld_f4(a.part_acc + place(s) * HD + tid % D4 * 4);
    o += f4_t{v.x, v.y, v.z, v.w} * s_f[s];
  }
  *reinterpret_cast<f4_t*>(&s_o[tid / D4][tid % D4 * 4]) = o;
  __syncthreads();
  if (tid >= HD) return;
  float v = 0.0f;
#pragma unroll
  for (int g = 0; g < GR; ++g) v += s_o[g][tid];
  v = !ok ? __builtin_nanf("") : (L == 0.0f ? 0.0f : v / L);
  if (!(fabsf(v) < INFINITY) && ok && L == L) {
    // an infinite sum counts whatever its part's factor, which may be 0
    float inf = 0.0f;
    for (uint32_t s = 0; s < ns; ++s) {
      const float x = gld(a.part_acc + place(s) * HD + tid);
      inf += fabsf(x) < INFINITY ? 0.0f : x;
    }
    if (inf != 0.0f) v = inf;
  }
  a.out[row * a.out_stride + size_t(h) * HD + tid] = v;
}

// ---- host -----------------------------------------------------------------------------------------------------
struct PrefixPlan {
  bool ok = false;
  uint32_t prefix_splits = 1, prefix_chunk = 1, rest_splits = 1, rest_chunk = 1, ht = 0, hz = 0, step = 0;
  uint64_t prefix_blocks = 0, rest_blocks = 0, joins = 0;
  size_t off_acc = 0, bytes = 0;
};

PrefixPlan prefix_plan(const chpe_kv_pages* c, uint32_t heads, uint32_t groups, uint32_t max_prefix, uint32_t max_rest) {
  PrefixPlan p;
  const uint32_t gq = heads / c->kv_heads, step = (c->type == 0 ? 16 : 32) * tiles_at_once(c->head_dim);
  const uint64_t large = (512 << 10) / (2 * c->head_dim * (c->type == 0 ? 4 : 2));  // slots
  auto split = [&](uint64_t items, uint64_t blocks, uint64_t want, uint32_t range, uint32_t* splits, uint32_t* chunk) {
    const uint64_t steps = std::max<uint64_t>(1, (uint64_t(range) + step - 1) / step), some = std::max<uint64_t>(1, items);
    uint64_t n = std::min<uint64_t>({std::max<uint64_t>((blocks + some - 1) / some, want), steps, kMaxSplits});
    n = std::max<uint64_t>(1, std::min<uint64_t>(n, kMaxBlocks / some));
    const uint64_t per = (steps + n - 1) / n;
    *chunk = uint32_t(per * step);
    *splits = uint32_t((steps + per - 1) / per);
  };
  p.step = step;
  const uint64_t in_all = uint64_t(c->rows) * heads;
  if (in_all > kMaxBlocks) return p;
  // queries of a workgroup: 16 where the registers allow them and the groups have as many
  const bool many = gq > 8 || (max_prefix != 0 && groups != 0 && uint64_t(c->rows) * gq > 8 * uint64_t(groups));
  p.ht = c->type == 0 || (many && c->head_dim <= kWaveDims) ? 16 : 8;
  // ... and k_prefix_many where they have more than a few, the calls are not all latency, and the rows' own slots, for which it
  // has most of its columns idle, do not count: behind 4096 slots with 64 of their own 64 rows of the 72B layout took 53 us
  // there and 74 in k_paged_16, 4 rows 17 and 20; 8 rows of the 9B layout (32 queries) 20 and 18; 64 rows behind 1000 slots
  // with up to 1000 of their own 82 and 69; 8 groups of 6 rows of 6 queries 31 and 21.  (f32 caches: k_paged_32 always, 16
  // queries a workgroup; 64 rows of the 72B layout behind 8192 slots 245 us, 110 of them at the f32 matrix cores' rate.)
  if (c->type != 0 && groups != 0 && uint64_t(c->rows) * gq >= 24 * uint64_t(groups) &&
      uint64_t(c->rows) * heads >= 256 && max_prefix / 2 >= max_rest)
    p.ht = many_queries(c->head_dim);
  p.hz = (gq + p.ht - 1) / p.ht;
  const uint64_t rest = uint64_t(c->rows) * c->kv_heads * p.hz;
  const uint64_t shared = (uint64_t(c->rows) * gq / p.ht + groups) * c->kv_heads;
  if (shared > kMaxBlocks || rest > kMaxBlocks) return p;
  split(rest, p.ht > 16 ? 512 : 1024, (max_rest + large - 1) / large, max_rest, &p.rest_splits, &p.rest_chunk);
  // (two workgroups of k_prefix_many a CU, 512 at once, some of them the rests': `shared` counts a tile a group too many)
  const uint64_t likely = std::max<uint64_t>((uint64_t(c->rows) * gq + p.ht - 1) / p.ht, groups) * c->kv_heads;
  split(p.ht > 16 ? likely : shared, p.ht > 16 ? 448 : 1024, 1, max_prefix, &p.prefix_splits, &p.prefix_chunk);
  p.rest_blocks = rest * p.rest_splits;
  p.prefix_blocks = max_prefix == 0 || groups == 0 ? 0 : shared * p.prefix_splits;
  if (p.rest_blocks + p.prefix_blocks > kMaxItems / 256) return p;
  p.joins = in_all;
  const uint64_t places = in_all * (p.prefix_splits + p.rest_splits);
  p.off_acc = (places * 8 + 255) / 256 * 256;
  p.bytes = p.off_acc + places * c->head_dim * 4;
  p.ok = true;
  return p;
}

template <int HD>
bool launch_prefix(const PrefixArgs& x, const PrefixPlan& p, int type, hipStream_t st) {
  const uint32_t thr = kWaves * 64;
  const uint64_t blocks = p.prefix_blocks + p.rest_blocks;
  const PartArgs a{x};
  bool ok = false;
  if (type == 0) {
    ok = launch(&k_paged_32<HD, PartArgs>, blocks, thr, st, a);
  } else if (p.ht > 16) {
    ok = type == 1 ? launch(&k_prefix_many<HD, _Float16>, blocks, thr, st, a) : launch(&k_prefix_many<HD, Bf16>, blocks, thr, st, a);
  } else if (p.ht == 8) {
    ok = type == 1 ? launch(&k_paged_16<HD, _Float16, 8, 1, PartArgs>, blocks, thr, st, a)
                   : launch(&k_paged_16<HD, Bf16, 8, 1, PartArgs>, blocks, thr, st, a);
  } else if constexpr (HD <= kWaveDims) {
    ok = type == 1 ? launch(&k_paged_16<HD, _Float16, 8, 2, PartArgs>, blocks, thr, st, a)
                   : launch(&k_paged_16<HD, Bf16, 8, 2, PartArgs>, blocks, thr, st, a);
  }
  return ok && launch(&k_prefix_join<HD>, p.joins, 256, st, x);
}

bool prefix_shape_ok(const chpe_kv_pages* c, uint32_t heads, uint32_t groups, uint32_t max_prefix, uint32_t max_rest) {
  return heads != 0 && heads % c->kv_heads == 0 && heads <= 65536 && groups <= 0x7ffffffeu &&
         uint64_t(max_prefix) + max_rest <= uint64_t(c->pages_per_row) * c->page_size;
}

}  // namespace
}  // namespace chpe

using namespace chpe;

extern "C" size_t chpe_paged_prefix_workspace(const chpe_kv_pages* cache, uint32_t heads, uint32_t groups,
                                              uint32_t max_prefix, uint32_t max_rest) {
  Pages c;
  if (!pages_from(cache, &c) || !prefix_shape_ok(cache, heads, groups, max_prefix, max_rest)) return 0;
  const PrefixPlan p = prefix_plan(cache, heads, groups, max_prefix, max_rest);
  return p.ok ? p.bytes : 0;
}

extern "C" int chpe_paged_prefix_attention(const chpe_kv_pages* cache, uint32_t heads, const int32_t* lens,
                                           uint32_t groups, const int32_t* group_rows, const int32_t* prefix_lens,
                                           uint32_t max_prefix, uint32_t max_rest, const float* q, uint64_t q_stride,
                                           float scale, float* out, uint64_t out_stride, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  PrefixArgs a{};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!pages_from(cache, &a.c) || !stream_here(st) || !prefix_shape_ok(cache, heads, groups, max_prefix, max_rest)) return -1;
  if (cache->rows == 0) return 0;
  const uint64_t width = uint64_t(heads) * cache->head_dim;
  if (!lens || !q || !out || !workspace || !aligned16(q) || !aligned16(out) || !aligned16(workspace)) return -1;
  if (groups != 0 && (!group_rows || !prefix_lens)) return -1;
  if (q_stride % 4 || out_stride % 4 || (cache->rows > 1 && (q_stride < width || out_stride < width))) return -1;
  if (cache->rows > 1 && (q_stride > (uint64_t(1) << 60) / cache->rows || out_stride > (uint64_t(1) << 60) / cache->rows)) return -1;
  const PrefixPlan p = prefix_plan(cache, heads, groups, max_prefix, max_rest);
  if (!p.ok) return -1;
  if (workspace_bytes < p.bytes) return -2;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.q = q;
  a.lens = lens;
  a.group_rows = group_rows;
  a.prefix_lens = prefix_lens;
  a.out = out;
  a.part_ml = reinterpret_cast<float*>(ws);
  a.part_acc = reinterpret_cast<float*>(ws + p.off_acc);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.rows = cache->rows;
  a.H = heads;
  a.groups = groups;
  a.max_prefix = max_prefix;
  a.max_rest = max_rest;
  a.prefix_splits = p.prefix_splits;
  a.prefix_chunk = p.prefix_chunk;
  a.prefix_blocks = uint32_t(p.prefix_blocks);
  a.rest_splits = p.rest_splits;
  a.rest_chunk = p.rest_chunk;
  a.step = p.step;
  a.hz = p.hz;
  a.scale = scale;
  const bool ok = cache->head_dim == 64    ? launch_prefix<64>(a, p, cache->type, st)
                  : cache->head_dim == 128 ? launch_prefix<128>(a, p, cache->type, st)
                                           : launch_prefix<256>(a, p, cache->type, st);
  return ok ? 0 : -3;
}
