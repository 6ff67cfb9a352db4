// paged_attention.hip -- chpe_paged_attention: the attention of one new token per row over the paged
// cache.  s_j = scale q.k_j over the row's slots lo <= j < len, p = softmax(s), out = sum_j p_j v_j, and,
// for a cache that is kept to a budget, each slot's p summed over the query heads of its kv head.
// A row's slots are split over workgroups: each leaves its maximum, sum of 2^(s - max) and so weighted sum of V
// rows, and a second launch rescales and joins them (and turns the scores into weights).
#include "paged_attention_kernels.hpp"

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
  uint32_t rows, H, max_len, window, score_stride;
  uint32_t hz, splits, chunk;     // groups of HT query heads of a kv head; splits of `chunk` slots
  float scale;

  static constexpr bool kScores = true;
  __device__ bool eager() const { return window == 0; }
  __device__ uint32_t eager_slot(const Place& p) const { return p.split * chunk; }
  __device__ bool whole() const { return splits == 1; }
  template <int HD>
  __device__ const float* query(const Place& p, uint32_t i) const {
    return q + p.row * q_stride + size_t(p.h0 + i) * HD;
  }
  __device__ size_t part_of(const Place& p, uint32_t i) const { return (size_t(p.row) * H + p.h0 + i) * splits + p.split; }
  template <int HT>
  __device__ Place place_of() const;
  __device__ void place_slots(Place* p) const;
  template <int HD>
  __device__ void leave_none(const Place& p) const;
};

// the row's slots lo .. len - 1; false for a length outside 0 .. max_len
__device__ __forceinline__ bool row_range(const PagedAttnArgs& a, uint32_t row, uint32_t* lo, uint32_t* len) {
  const uint32_t n = uint32_t(gld(a.lens + row));
  *len = n <= a.max_len ? n : 0u;
  *lo = a.window != 0 && *len > a.window ? *len - a.window : 0u;
  return n <= a.max_len;
}

// ---- the splits ------------------------------------------------------------------------------------------------
// (Args: paged_attention_kernels.hpp)
template <int HT>
__device__ __forceinline__ Place PagedAttnArgs::place_of() const {
  const PagedAttnArgs& a = *this;
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
  p.row = p.table = b / a.c.KV;
  p.h0 = p.kvh * gq + z * HT;
  p.nh = min(uint32_t(HT), gq - z * HT);
  return p;
}
__device__ __forceinline__ void PagedAttnArgs::place_slots(Place* p) const {
  const PagedAttnArgs& a = *this;
  p->ok = row_range(a, p->row, &p->lo, &p->len);
  p->begin = p->lo + p->split * a.chunk;
  p->end = min(p->len, p->begin + a.chunk);
}
// a split without slots: nothing for the join (it goes by the row's length); the output of a row of one
// split at most
template <int HD>
__device__ __forceinline__ void PagedAttnArgs::leave_none(const Place& p) const {
  const PagedAttnArgs& a = *this;
  if (a.splits != 1) return;
  const float v = p.ok ? 0.0f : __builtin_nanf("");
  for (uint32_t i = threadIdx.x; i < p.nh * HD; i += kWaves * 64) a.out[p.row * a.out_stride + size_t(p.h0) * HD + i] = v;
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
  if (type == 0) return launch(&k_paged_32<HD, PagedAttnArgs>, blocks, thr, st, a);
  if (type == 2 && ht == 4) return launch(&k_paged_16<HD, Bf16, 4, 1, PagedAttnArgs>, blocks, thr, st, a);
  if (ht == 8)
    return type == 1 ? launch(&k_paged_16<HD, _Float16, 8, 1, PagedAttnArgs>, blocks, thr, st, a)
                     : launch(&k_paged_16<HD, Bf16, 8, 1, PagedAttnArgs>, blocks, thr, st, a);
  if constexpr (HD <= 128)
    return type == 1 ? launch(&k_paged_16<HD, _Float16, 8, 2, PagedAttnArgs>, blocks, thr, st, a)
                     : launch(&k_paged_16<HD, Bf16, 8, 2, PagedAttnArgs>, blocks, thr, st, a);
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
