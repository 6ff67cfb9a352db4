// paged_attention.hip -- chpe_paged_attention: the attention of one new token per row over the paged
// cache.  s_j = scale q.k_j over the row's slots lo <= j < len, p = softmax(s), out = sum_j p_j v_j, and,
// for a cache that is kept to a budget, each slot's p summed over the query heads of its kv head.
// The slots are split over workgroups: each leaves its maximum, sum of exp(s - max) and exp-weighted sum
// of V rows, and a second launch rescales and joins them (and turns the scores into weights).
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
  float* scores;                  // [row][head][max_len], or null
  const float* weight_in;
  float* weight_out;
  uint64_t q_stride, out_stride, weight_stride;
  uint32_t rows, H, max_len, window, splits, chunk;
  float scale;
};

// the row's slots lo .. len - 1; false for a length outside 0 .. max_len
__device__ __forceinline__ bool row_range(const PagedAttnArgs& a, uint32_t row, uint32_t* lo, uint32_t* len) {
  const uint32_t n = uint32_t(gld(a.lens + row));
  *len = n <= a.max_len ? n : 0u;
  *lo = a.window != 0 && *len > a.window ? *len - a.window : 0u;
  return n <= a.max_len;
}

// one wave per (row, query head, split): slot after slot, lane l holds dims l, l + 64, ..
template <int HD, class T>
__global__ void __launch_bounds__(64) k_paged_partial(PagedAttnArgs a) {
  constexpr int N = HD / 64;
  const uint32_t split = blockIdx.x % a.splits, item = blockIdx.x / a.splits, h = item % a.H, row = item / a.H;
  const int lane = threadIdx.x;
  uint32_t lo, len;
  row_range(a, row, &lo, &len);
  const uint32_t b = lo + split * a.chunk, e = min(len, b + a.chunk);
  const uint32_t kvh = h / (a.H / a.c.KV);
  float q[N], acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = a.q[row * a.q_stride + h * HD + lane + 64 * i];
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (uint32_t j = b; j < e; ++j) {
    uint32_t page;
    const bool ok = a.c.page_of(row, j, &page);
    const size_t at = a.c.at(page, kvh, j);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], Elem<T>::get(reinterpret_cast<const T*>(a.c.k) + at + lane + 64 * i), s);
    s = ok ? wave_sum(s) * a.scale : __builtin_nanf("");
    if (a.scores && lane == 0) a.scores[(size_t(row) * a.H + h) * a.max_len + j] = s;
    const float m2 = fmaxf(m, s), base = m2 == -INFINITY ? 0.0f : m2;
    const float f = expf(m - base), p = expf(s - base);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < N; ++i)
      acc[i] = acc[i] * f + p * Elem<T>::get(reinterpret_cast<const T*>(a.c.v) + at + lane + 64 * i);
    m = m2;
  }
  const size_t pt = size_t(item) * a.splits + split;
#pragma unroll
  for (int i = 0; i < N; ++i) a.part_acc[pt * HD + lane + 64 * i] = acc[i];
  if (lane == 0) {
    a.part_ml[pt * 2] = m;
    a.part_ml[pt * 2 + 1] = l;
  }
}

// maximum and sum over an item's splits
__device__ __forceinline__ void join_ml(const PagedAttnArgs& a, uint32_t item, float* M, float* L) {
  float m = -INFINITY, l = 0.0f;
  for (uint32_t s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[(size_t(item) * a.splits + s) * 2]);
  const float base = m == -INFINITY ? 0.0f : m;
  for (uint32_t s = 0; s < a.splits; ++s) {
    const size_t pt = (size_t(item) * a.splits + s) * 2;
    l += a.part_ml[pt + 1] * expf(a.part_ml[pt] - base);
  }
  *M = base;
  *L = l;
}

template <int HD>
__global__ void __launch_bounds__(HD) k_paged_join(PagedAttnArgs a) {
  const uint32_t item = blockIdx.x, h = item % a.H, row = item / a.H, d = threadIdx.x;
  uint32_t lo, len;
  const bool ok = row_range(a, row, &lo, &len);
  float M, L, o = 0.0f;
  join_ml(a, item, &M, &L);
  for (uint32_t s = 0; s < a.splits; ++s) {
    const size_t pt = size_t(item) * a.splits + s;
    if (a.part_ml[pt * 2 + 1] != 0.0f) o += a.part_acc[pt * HD + d] * expf(a.part_ml[pt * 2] - M);
  }
  a.out[row * a.out_stride + h * HD + d] = !ok ? __builtin_nanf("") : (L == 0.0f ? 0.0f : o / L);
}

__global__ void __launch_bounds__(256) k_paged_weights(PagedAttnArgs a, uint32_t blocks_per_row) {
  const uint32_t part = blockIdx.x % blocks_per_row, item = blockIdx.x / blocks_per_row;
  const uint32_t kvh = item % a.c.KV, row = item / a.c.KV, gq = a.H / a.c.KV, j = part * 256 + threadIdx.x;
  uint32_t lo, len;
  if (!row_range(a, row, &lo, &len) || j >= len) return;
  float w = 0.0f;
  for (uint32_t g = 0; j >= lo && g < gq; ++g) {
    const uint32_t hh = row * a.H + kvh * gq + g;
    float M, L;
    join_ml(a, hh, &M, &L);
    if (L != 0.0f) w += expf(a.scores[size_t(hh) * a.max_len + j] - M) / L;
  }
  const size_t at = (size_t(row) * a.c.KV + kvh) * a.weight_stride + j;
  a.weight_out[at] = (a.weight_in ? a.weight_in[at] : 0.0f) + w;
}

struct AttnPlan {
  uint32_t splits = 1, chunk = 1;
  size_t off_acc = 0, off_scores = 0, bytes = 0;
};

// at most this many splits of a range of slots (it grows with the range)
uint32_t most_splits(uint64_t items, uint32_t range) {
  const uint64_t want = (8192 + items - 1) / items, most = (uint64_t(range) + 31) / 32;
  return uint32_t(std::max<uint64_t>(1, std::min(want, most)));
}

AttnPlan attn_plan(const chpe_kv_pages* c, uint32_t heads, uint32_t max_len, uint32_t window, bool weights) {
  AttnPlan p;
  const uint32_t range = window != 0 && window < max_len ? window : max_len;
  const uint64_t items = std::max<uint64_t>(1, uint64_t(c->rows) * heads);
  p.chunk = std::max(1u, (range + most_splits(items, range) - 1) / most_splits(items, range));
  p.splits = range ? (range + p.chunk - 1) / p.chunk : 1;
  // the workspace does not depend on the window
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const uint32_t room = most_splits(items, max_len);
  p.off_acc = up(items * room * 8);
  p.off_scores = p.off_acc + up(items * room * c->head_dim * 4);
  p.bytes = p.off_scores + (weights ? up(items * max_len * 4) : 0);
  return p;
}

template <class T>
bool launch_attn(const PagedAttnArgs& a, uint32_t hd, hipStream_t st) {
  const uint64_t items = uint64_t(a.rows) * a.H, blocks = items * a.splits;
  bool ok;
  if (hd == 64) ok = launch(&k_paged_partial<64, T>, blocks, 64, st, a) && launch(&k_paged_join<64>, items, 64, st, a);
  else if (hd == 128) ok = launch(&k_paged_partial<128, T>, blocks, 64, st, a) && launch(&k_paged_join<128>, items, 128, st, a);
  else ok = launch(&k_paged_partial<256, T>, blocks, 64, st, a) && launch(&k_paged_join<256>, items, 256, st, a);
  if (ok && a.weight_out && a.max_len) {
    const uint32_t per = (a.max_len + 255) / 256;
    ok = launch(&k_paged_weights, uint64_t(a.rows) * a.c.KV * per, 256, st, a, per);
  }
  return ok;
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
  if (uint64_t(cache->rows) * heads * p.splits > kMaxBlocks) return -1;
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
  const bool ok = cache->type == 0 ? launch_attn<float>(a, cache->head_dim, st)
                                   : cache->type == 1 ? launch_attn<_Float16>(a, cache->head_dim, st)
                                                      : launch_attn<Bf16>(a, cache->head_dim, st);
  return ok ? 0 : -3;
}
