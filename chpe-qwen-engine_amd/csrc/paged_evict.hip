// paged_evict.hip -- chpe_paged_evict: a row's cache cut to a budget of n slots per kv head.  The newest
// positions and the first ones stay; of the others those with the largest accumulated weights (equal
// weights: the lower slot; NaN last).  The kept slots at n and above move into the holes below n, both in
// ascending order: the softmax does not ask for an order, so no other row moves, and no slot is both read
// and written.
#include <utility>

#include "paged.hpp"

namespace chpe {
namespace {
using namespace dev;

struct EvictArgs {
  Pages c;
  const int32_t* lens;
  const float* weight;
  const int32_t* pos;
  int32_t* lens_out;
  float* weight_out;
  int32_t *pos_out, *slot_src;
  uint32_t *moves, *n_moves;  // [row][kv head][half][2] (to, from), [row][kv head]
  uint64_t stride;
  uint32_t rows, max_len, budget, recent, sinks, half;
};

constexpr int kSelect = 256;  // threads of the selection

// the order of the weights as unsigned integers: NaN 0, then -inf .. +inf (-0 as +0)
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t block_sum(uint32_t v, uint32_t* s) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < kSelect / 64; ++w) v += s[w];
  return v;
}

// exclusive prefix count of `f` over the workgroup's threads; *total: the count
__device__ __forceinline__ uint32_t block_rank(bool f, uint32_t* s, uint32_t* total) {
  const uint64_t b = __ballot(f);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[wave] = __popcll(b);
  __syncthreads();
  uint32_t before = __popcll(b & ((uint64_t(1) << (threadIdx.x & 63)) - 1)), all = 0;
  for (int w = 0; w < kSelect / 64; ++w) {
    if (w < wave) before += s[w];
    all += s[w];
  }
  *total = all;
  return before;
}

// one workgroup per (row, kv head)
__global__ void __launch_bounds__(kSelect) k_evict_select(EvictArgs a) {
  __shared__ uint32_t s_red[kSelect / 64];
  const uint32_t item = blockIdx.x, row = item / a.c.KV, tid = threadIdx.x;
  const uint32_t raw = uint32_t(gld(a.lens + row));
  const bool bad = raw > a.max_len;
  const uint32_t len = bad ? 0u : raw, keep = min(len, a.budget);
  if (tid == 0 && item % a.c.KV == 0) a.lens_out[row] = bad ? int32_t(raw) : int32_t(keep);
  const size_t base = size_t(item) * a.stride;
  const float* weight = a.weight + base;
  const int32_t* pos = a.pos + base;

  int32_t newest = INT32_MIN;
  for (uint32_t j = tid; j < len; j += kSelect) newest = max(newest, pos[j]);
  for (int o = 32; o > 0; o >>= 1) newest = max(newest, __shfl_xor(newest, o));
  if ((tid & 63) == 0) s_red[tid >> 6] = uint32_t(newest);
  __syncthreads();
  for (int w = 0; w < kSelect / 64; ++w) newest = max(newest, int32_t(s_red[w]));
  auto key = [&](uint32_t j) {
    const int64_t p = pos[j];
    return p > int64_t(newest) - a.recent || p < int64_t(a.sinks) ? 0xffffffffu : weight_key(weight[j]);
  };

  // the largest threshold that `keep` keys reach, bit by bit
  uint32_t T = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = T | (1u << bit);
    uint32_t n = 0;
    for (uint32_t j = tid; j < len; j += kSelect) n += key(j) >= cand ? 1u : 0u;
    if (block_sum(n, s_red) >= keep) T = cand;
  }
  uint32_t above = 0;
  for (uint32_t j = tid; j < len; j += kSelect) above += key(j) > T ? 1u : 0u;
  above = block_sum(above, s_red);
  const uint32_t ties = keep - min(above, keep);  // of the keys equal to T, the first `ties` slots stay

  uint32_t *to = a.moves + size_t(item) * a.half * 2, *from = to + a.half;
  uint32_t seen = 0, holes = 0, movers = 0;
  for (uint32_t j0 = 0; j0 < len; j0 += kSelect) {
    const uint32_t j = j0 + tid;
    const uint32_t k = j < len ? key(j) : 0u;
    uint32_t all;
    const uint32_t r = seen + block_rank(j < len && k == T, s_red, &all);
    seen += all;
    const bool kept = j < len && (k > T || (k == T && r < ties));
    const bool hole = j < keep && !kept, mover = j >= keep && kept;
    const uint32_t rh = holes + block_rank(hole, s_red, &all);
    holes += all;
    const uint32_t rm = movers + block_rank(mover, s_red, &all);
    movers += all;
    if (hole) to[rh] = j;
    if (mover) from[rm] = j;
    if (j < keep && kept) {
      a.weight_out[base + j] = weight[j];
      a.pos_out[base + j] = pos[j];
      if (a.slot_src) a.slot_src[base + j] = int32_t(j);
    }
  }
  if (tid == 0) a.n_moves[item] = holes;
  __syncthreads();
  for (uint32_t i = tid; i < holes; i += kSelect) {
    const uint32_t d = to[i], s = from[i];
    a.weight_out[base + d] = weight[s];
    a.pos_out[base + d] = pos[s];
    if (a.slot_src) a.slot_src[base + d] = int32_t(s);
  }
}

// the K and V rows of the moves, 16 bytes a lane
template <int ROW16>
__global__ void __launch_bounds__(256) k_evict_move(EvictArgs a, uint32_t parts, uint32_t elem) {
  constexpr int PER = 256 / ROW16;
  const uint32_t item = blockIdx.x / parts, part = blockIdx.x % parts, row = item / a.c.KV, h = item % a.c.KV;
  const uint32_t n = a.n_moves[item], lane = threadIdx.x % ROW16;
  const uint32_t *to = a.moves + size_t(item) * a.half * 2, *from = to + a.half;
  for (uint32_t i = part * PER + threadIdx.x / ROW16; i < n; i += parts * PER) {
    const uint32_t d = to[i], s = from[i];
    uint32_t pd, ps;
    if (!a.c.page_of(row, d, &pd) || !a.c.page_of(row, s, &ps)) continue;
    const size_t od = a.c.at(pd, h, d) * elem + lane * 16, os = a.c.at(ps, h, s) * elem + lane * 16;
    const uint4 kk = ld_u128(a.c.k + os), vv = ld_u128(a.c.v + os);
    *reinterpret_cast<uint4*>(a.c.k + od) = kk;
    *reinterpret_cast<uint4*>(a.c.v + od) = vv;
  }
}

size_t evict_bytes(const chpe_kv_pages* c, uint32_t max_len, size_t* off) {
  const size_t items = size_t(c->rows) * c->kv_heads, half = max_len / 2 + 1;
  *off = (items * 4 + 255) / 256 * 256;
  return *off + items * half * 8;
}

bool evict_shape_ok(const chpe_kv_pages* c, uint32_t max_len) {
  return uint64_t(max_len) <= uint64_t(c->pages_per_row) * c->page_size && uint64_t(c->rows) * c->kv_heads <= kMaxBlocks;
}

}  // namespace
}  // namespace chpe

using namespace chpe;

extern "C" size_t chpe_paged_evict_workspace(const chpe_kv_pages* cache, uint32_t max_len) {
  Pages p;
  size_t off;
  return pages_from(cache, &p) && evict_shape_ok(cache, max_len) ? evict_bytes(cache, max_len, &off) : 0;
}

extern "C" int chpe_paged_evict(const chpe_kv_pages* cache, const int32_t* lens, uint32_t max_len, uint32_t budget,
                                uint32_t recent, uint32_t sinks, const float* weight, const int32_t* slot_pos,
                                uint64_t stride, int32_t* lens_out, float* weight_out, int32_t* pos_out,
                                int32_t* slot_src, void* workspace, size_t workspace_bytes, void* stream) {
  EvictArgs a{};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!pages_from(cache, &a.c) || !stream_here(st) || !evict_shape_ok(cache, max_len)) return -1;
  if (cache->rows == 0) return 0;
  if (!lens || !weight || !slot_pos || !lens_out || !weight_out || !pos_out || !workspace || !aligned16(workspace) ||
      stride < max_len || uint64_t(recent) + sinks > budget)
    return -1;
  size_t off;
  if (workspace_bytes < evict_bytes(cache, max_len, &off)) return -2;
  a.lens = lens;
  a.weight = weight;
  a.pos = slot_pos;
  a.lens_out = lens_out;
  a.weight_out = weight_out;
  a.pos_out = pos_out;
  a.slot_src = slot_src;
  a.n_moves = static_cast<uint32_t*>(workspace);
  a.moves = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + off);
  a.stride = stride;
  a.rows = cache->rows;
  a.max_len = max_len;
  a.budget = budget;
  a.recent = recent;
  a.sinks = sinks;
  a.half = max_len / 2 + 1;
  const uint64_t items = uint64_t(cache->rows) * cache->kv_heads;
  if (!launch(&k_evict_select, items, kSelect, st, a)) return -3;
  const uint32_t elem = cache->type == 0 ? 4 : 2, row16 = cache->head_dim * elem / 16, parts = 8;
  if (items * parts > kMaxBlocks) return -1;
  const bool ok = row16 == 8    ? launch(&k_evict_move<8>, items * parts, 256, st, a, parts, elem)
                  : row16 == 16 ? launch(&k_evict_move<16>, items * parts, 256, st, a, parts, elem)
                  : row16 == 32 ? launch(&k_evict_move<32>, items * parts, 256, st, a, parts, elem)
                                : launch(&k_evict_move<64>, items * parts, 256, st, a, parts, elem);
  return ok ? 0 : -3;
}
