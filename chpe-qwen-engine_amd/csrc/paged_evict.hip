// paged_evict.hip -- chpe_paged_evict: a row's cache cut to a budget of n slots per kv head.  The newest
// positions and the first ones stay; of the others those with the largest accumulated weights (equal
// weights: the lower slot; NaN last).  The kept slots at n and above move into the holes below n, both in
// ascending order: the softmax does not ask for an order, so no other row moves, and no slot is both read
// and written.
#include <algorithm>

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
  uint32_t rows, max_len, budget, recent, sinks, half, fused;
  uint32_t elem, row16;  // bytes of an element; 16-byte pieces of a row
};

constexpr int kSelect = 1024, kSelWaves = kSelect / 64;  // threads of the selection
constexpr uint32_t kFusedMoves = 64;                     // at most this many moves: made by the selection itself

// the order of the weights as unsigned integers: NaN 0, then -inf .. +inf (-0 as +0)
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// a slot's place in the order: the protected ones above all weights
__device__ __forceinline__ uint32_t slot_key(const EvictArgs& a, float w, int32_t pos, int32_t newest) {
  return int64_t(pos) > int64_t(newest) - a.recent || int64_t(pos) < int64_t(a.sinks) ? 0xffffffffu : weight_key(w);
}

__device__ __forceinline__ int32_t block_max(int32_t v, int32_t* s) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, int32_t(pair_u(uint32_t(v), o)));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < kSelWaves; ++w) v = max(v, s[w]);
  return v;
}

// The threshold T that `keep` of len keys reach, and how many of the keys equal to it stay.  Two bits of T a
// step, from the top: how many keys reach T + 1, 2, 3 of the step's size says which of the four intervals
// holds the keep-th largest key.  A step ends the search where an interval's lower end is reached by exactly
// `keep` keys.  count(cand, n): adds this wave's number of keys >= cand[i] to n[i] (uniform in the wave).
struct Threshold {
  uint32_t T, ties;
  bool all;  // every key equal to T stays
};
template <class Count>
__device__ __forceinline__ Threshold find_threshold(uint32_t len, uint32_t keep, uint32_t (*s)[4], Count count) {
  if (keep == len) return {0u, len, true};
  uint32_t T = 0, reach = len, above = 0;  // keys >= T; keys >= T + the last step's size
  int buf = 0;
  for (int bit = 30; bit >= 0 && reach != keep; bit -= 2, buf = buf == 2 ? 0 : buf + 1) {
    const uint32_t cand[3] = {T + (1u << bit), T + (2u << bit), T + (3u << bit)};
    uint32_t n[3] = {0, 0, 0};
    count(cand, n);
    // three buffers: this step's was cleared in the step before, when the step before that had been read
    if (threadIdx.x < 3) s[buf == 2 ? 0 : buf + 1][threadIdx.x] = 0;
    if ((threadIdx.x & 63) < 3) atomicAdd(&s[buf][threadIdx.x & 63], (threadIdx.x & 63) == 0 ? n[0] : (threadIdx.x & 63) == 1 ? n[1] : n[2]);
    __syncthreads();
    const uint32_t c1 = s[buf][0], c2 = s[buf][1], c3 = s[buf][2];
    if (c3 >= keep) T = cand[2], reach = c3;
    else if (c2 >= keep) T = cand[1], reach = c2, above = c3;
    else if (c1 >= keep) T = cand[0], reach = c1, above = c2;
    else above = c1;
  }
  return {T, reach == keep ? keep : keep - above, reach == keep};
}

// exclusive prefix sums of n <= kSelect values in LDS; returns the total
__device__ __forceinline__ uint32_t block_scan(uint32_t* tab, uint32_t n, uint32_t* s) {
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __syncthreads();
  const uint32_t v = tid < n ? tab[tid] : 0u;
  uint32_t x = v;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= uint32_t(o)) x += y;
  }
  if (lane == 63) s[wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t w = 0; w < kSelWaves; ++w) {
    if (w < wave) before += s[w];
    all += s[w];
  }
  if (tid < n) tab[tid] = before + x - v;
  __syncthreads();
  return all;
}

__device__ __forceinline__ uint32_t below(uint64_t ballot, int lane) {
  return __popcll(ballot & ((uint64_t(1) << lane) - 1));
}

// the K and V rows of `n` moves, 16 bytes a lane, `lanes` lanes a row
__device__ __forceinline__ void move_rows(const EvictArgs& a, uint32_t row, uint32_t h, const uint32_t* to,
                                          const uint32_t* from, uint32_t n, uint32_t first, uint32_t step, uint32_t lane) {
  for (uint32_t i = first; i < n; i += step) {
    const uint32_t d = to[i], s = from[i];
    uint32_t pd, ps;
    if (!a.c.page_of(row, d, &pd) || !a.c.page_of(row, s, &ps)) continue;
    const size_t od = a.c.at(pd, h, d) * a.elem + lane * 16, os = a.c.at(ps, h, s) * a.elem + lane * 16;
    const uint4 kk = ld_u128(a.c.k + os), vv = ld_u128(a.c.v + os);
    *reinterpret_cast<uint4*>(a.c.k + od) = kk;
    *reinterpret_cast<uint4*>(a.c.v + od) = vv;
  }
}

// One workgroup per (row, kv head): the slots' keys in registers (thread tid holds slots tid, tid + 1024, ..,
// KPT of them), read once; the threshold by counting with ballots; then the ranks of the holes and of the
// movers among the slots, from one table of counts per (1024 slots, wave).
template <int KPT>
__global__ void __launch_bounds__(kSelect) k_evict_select(EvictArgs a) {
  __shared__ uint32_t s_tab[KPT * kSelWaves], s_red[kSelWaves], s_cnt[3][4], s_moves[2 * kFusedMoves];
  const uint32_t item = blockIdx.x, row = item / a.c.KV, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const uint32_t raw = uint32_t(gld(a.lens + row));
  const bool bad = raw > a.max_len;
  const uint32_t len = bad ? 0u : raw, keep = min(len, a.budget);
  if (tid == 0 && item % a.c.KV == 0) a.lens_out[row] = bad ? int32_t(raw) : int32_t(keep);
  if (len == 0) {
    if (tid == 0) a.n_moves[item] = 0;
    return;
  }
  const size_t base = size_t(item) * a.stride;
  const float* weight = a.weight + base;
  const int32_t* pos = a.pos + base;

  // up to 16 slots a thread their weights and positions stay in registers too, for the slots that keep their
  // place; more are read again (from the L2)
  constexpr bool kHold = KPT <= 16;
  constexpr int HOLD = kHold ? KPT : 1;
  float w[HOLD];
  int32_t p[HOLD], newest = INT32_MIN;
  uint32_t key[KPT];
  auto slot_of = [&](int k) { return min(k * kSelect + tid, len - 1); };
  if constexpr (kHold) {
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
      p[k] = gld(pos + slot_of(k));
      w[k] = gld(weight + slot_of(k));
    }
  }
#pragma unroll
  for (int k = 0; k < KPT; ++k) newest = max(newest, kHold ? p[k % HOLD] : gld(pos + slot_of(k)));
  if (tid < 12) s_cnt[tid / 4][tid % 4] = 0;
  newest = block_max(newest, reinterpret_cast<int32_t*>(s_red));
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const float wk = kHold ? w[k % HOLD] : gld(weight + slot_of(k));
    const int32_t pk = kHold ? p[k % HOLD] : gld(pos + slot_of(k));
    key[k] = k * kSelect + tid < len ? slot_key(a, wk, pk, newest) : 0u;
  }

  const Threshold th = find_threshold(len, keep, s_cnt, [&](const uint32_t (&cand)[3], uint32_t (&n)[3]) {
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
      if (uint32_t(k) * kSelect >= len) break;
#pragma unroll
      for (int i = 0; i < 3; ++i) n[i] += __popcll(__ballot(key[k] >= cand[i]));
    }
  });

  // of the keys equal to the threshold the first `ties` slots stay
  uint64_t kept[KPT];
#pragma unroll
  for (int k = 0; k < KPT; ++k) kept[k] = __ballot(k * kSelect + tid < len && key[k] >= th.T);
  if (!th.all) {
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
      const uint64_t eq = __ballot(k * kSelect + tid < len && key[k] == th.T);
      if (lane == 0) s_tab[k * kSelWaves + wave] = __popcll(eq);
    }
    block_scan(s_tab, KPT * kSelWaves, s_red);
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
      const bool eq = k * kSelect + tid < len && key[k] == th.T;
      const uint32_t rank = s_tab[k * kSelWaves + wave] + below(__ballot(eq), lane);
      kept[k] &= ~__ballot(eq && rank >= th.ties);
    }
    __syncthreads();
  }
  // holes in the lower, movers in the upper half of a count (either is at most half of 65536 slots)
  const uint64_t bit = uint64_t(1) << lane;
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const uint32_t j = k * kSelect + tid;
    const uint64_t in = __ballot(j < keep);
    const uint32_t holes = __popcll(in & ~kept[k]), movers = __popcll(kept[k] & ~in);
    if (lane == 0) s_tab[k * kSelWaves + wave] = holes | movers << 16;
  }
  const uint32_t moves = block_scan(s_tab, KPT * kSelWaves, s_red) & 0xffffu;
  const bool fused = a.fused != 0;
  uint32_t *to = fused ? s_moves : a.moves + size_t(item) * a.half * 2, *from = to + (fused ? kFusedMoves : a.half);
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const uint32_t j = k * kSelect + tid;
    const uint64_t in = __ballot(j < keep);
    const uint32_t at = s_tab[k * kSelWaves + wave];
    if (j < keep && !(kept[k] & bit)) to[(at & 0xffffu) + below(in & ~kept[k], lane)] = j;
    if (j >= keep && (kept[k] & bit)) from[(at >> 16) + below(kept[k] & ~in, lane)] = j;
    if (j < keep && (kept[k] & bit)) {
      a.weight_out[base + j] = kHold ? w[k % HOLD] : gld(weight + j);
      a.pos_out[base + j] = kHold ? p[k % HOLD] : gld(pos + j);
      if (a.slot_src) a.slot_src[base + j] = int32_t(j);
    }
  }
  if (tid == 0) a.n_moves[item] = moves;
  __syncthreads();
  for (uint32_t i = tid; i < moves; i += kSelect) {
    const uint32_t d = to[i], s = from[i];
    a.weight_out[base + d] = weight[s];
    a.pos_out[base + d] = pos[s];
    if (a.slot_src) a.slot_src[base + d] = int32_t(s);
  }
  if (fused) move_rows(a, row, item % a.c.KV, to, from, moves, tid / a.row16, kSelect / a.row16, tid % a.row16);
}

// The same for rows past kLongest slots: the keys are read again for every step, the ranks counted in one walk.
constexpr uint32_t kLongest = 64 * kSelect;
__device__ __forceinline__ uint32_t block_rank(bool f, uint32_t* s, uint32_t* total) {
  const uint64_t b = __ballot(f);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[wave] = __popcll(b);
  __syncthreads();
  uint32_t before = below(b, threadIdx.x & 63), all = 0;
  for (int w = 0; w < kSelWaves; ++w) {
    if (w < wave) before += s[w];
    all += s[w];
  }
  *total = all;
  return before;
}

__global__ void __launch_bounds__(kSelect) k_evict_select_long(EvictArgs a) {
  __shared__ uint32_t s_red[kSelWaves], s_cnt[3][4];
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
  if (tid < 12) s_cnt[tid / 4][tid % 4] = 0;
  newest = block_max(newest, reinterpret_cast<int32_t*>(s_red));
  auto key = [&](uint32_t j) { return slot_key(a, gld(weight + j), gld(pos + j), newest); };
  const Threshold th = find_threshold(len, keep, s_cnt, [&](const uint32_t (&cand)[3], uint32_t (&n)[3]) {
    for (uint32_t j0 = 0; j0 < len; j0 += kSelect) {
      const uint32_t k = j0 + tid < len ? key(j0 + tid) : 0u;
      for (int i = 0; i < 3; ++i) n[i] += __popcll(__ballot(k >= cand[i]));
    }
  });
  uint32_t *to = a.moves + size_t(item) * a.half * 2, *from = to + a.half;
  uint32_t seen = 0, holes = 0, movers = 0;
  for (uint32_t j0 = 0; j0 < len; j0 += kSelect) {
    const uint32_t j = j0 + tid;
    const uint32_t k = j < len ? key(j) : 0u;
    uint32_t all;
    const uint32_t r = seen + block_rank(j < len && k == th.T, s_red, &all);
    seen += all;
    const bool kept = j < len && (k > th.T || (k == th.T && (th.all || r < th.ties)));
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

// the moves that the selection left, `parts` workgroups per (row, kv head)
__global__ void __launch_bounds__(256) k_evict_move(EvictArgs a, uint32_t parts) {
  const uint32_t item = blockIdx.x / parts, part = blockIdx.x % parts, per = 256 / a.row16;
  const uint32_t *to = a.moves + size_t(item) * a.half * 2, *from = to + a.half;
  move_rows(a, item / a.c.KV, item % a.c.KV, to, from, gld(a.n_moves + item), part * per + threadIdx.x / a.row16,
            parts * per, threadIdx.x % a.row16);
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
  a.elem = cache->type == 0 ? 4 : 2;
  a.row16 = cache->head_dim * a.elem / 16;
  // a (row, kv head) has at most this many moves
  const uint32_t most = max_len > budget ? std::min(budget, max_len - budget) : 0;
  a.fused = most <= kFusedMoves && max_len <= kLongest ? 1 : 0;
  const uint64_t items = uint64_t(cache->rows) * cache->kv_heads;
  const uint32_t parts = std::max(1u, std::min(8u, most / 64));
  if (items * parts > kMaxBlocks) return -1;
  const bool ok = max_len <= kSelect        ? launch(&k_evict_select<1>, items, kSelect, st, a)
                  : max_len <= 4 * kSelect  ? launch(&k_evict_select<4>, items, kSelect, st, a)
                  : max_len <= 16 * kSelect ? launch(&k_evict_select<16>, items, kSelect, st, a)
                  : max_len <= kLongest     ? launch(&k_evict_select<64>, items, kSelect, st, a)
                                            : launch(&k_evict_select_long, items, kSelect, st, a);
  if (!ok || (most != 0 && !a.fused && !launch(&k_evict_move, items * parts, 256, st, a, parts))) return -3;
  return 0;
}
