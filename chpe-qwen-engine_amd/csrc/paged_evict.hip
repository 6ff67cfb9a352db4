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
  uint32_t in_place;     // lens_out is lens: written after the selection, whose workgroups all read the lengths
};

constexpr int kSelect = 1024, kSelWaves = kSelect / 64;  // threads of the selection
// At most this many moves are made by the selection itself: 16 rows of 4 heads of 256 with 64 moves each 11.7 us a
// call, with a launch for them 17.9.  The two meet at some 256 moves (22.1 us both ways; 512: 30.3 against 24.5).
constexpr uint32_t kFusedMoves = 64;
constexpr uint32_t kFew = 8;                             // at most this many slots to drop: one after the other

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

// the sum over the waves before this one, and over all, of what every wave's last lane holds
__device__ __forceinline__ uint32_t waves_before(uint32_t last, uint32_t* s, uint32_t* all) {
  const uint32_t wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) s[wave] = last;
  __syncthreads();
  uint32_t before = 0, sum = 0;
#pragma unroll
  for (uint32_t w = 0; w < kSelWaves; ++w) {
    const uint32_t x = s[w];
    before += w < wave ? x : 0u;
    sum += x;
  }
  *all = sum;
  return before;
}

// The threshold T that `keep` of len keys reach, and how many of the keys equal to it stay: the digits of T
// from the top, 11, 11 and 10 bits, each from a histogram of the keys that share the digits above it.  The
// search ends where a bin is kept whole.  each(f): calls f(valid, key) for every key of this thread, with all
// lanes of the wave active.
struct Threshold {
  uint32_t T, ties;
  bool all;  // every key that reaches T stays
};
constexpr int kBins = 2048;
template <class Each>
__device__ __forceinline__ Threshold find_threshold(uint32_t len, uint32_t keep, uint32_t* hist, uint32_t* s, uint32_t* found,
                                                    Each each) {
  if (keep == len) return {0u, len, true};
  if (keep == 0) return {0xffffffffu, 0u, false};
  const uint32_t tid = threadIdx.x;
  uint32_t T = 0, need = keep;  // the digits so far; keys still to be found below the larger ones
  for (int shift = 21, bits = 11;; ) {
    hist[tid] = hist[tid + kSelect] = 0;
    __syncthreads();
    const uint32_t above = T >> (shift + bits - 1) >> 1;  // (shift + bits may be 32)
    each([&](bool valid, uint32_t key) {
      const bool in = valid && key >> (shift + bits - 1) >> 1 == above;
      const uint32_t bin = key >> shift & ((1u << bits) - 1);
      // a wave whose keys all fall into one bin (equal weights) counts them at once
      const uint64_t who = __ballot(in);
      if (who == 0) return;
      const uint32_t first = __builtin_amdgcn_readlane(bin, __ffsll((unsigned long long)who) - 1);
      if (__ballot(in && bin == first) == who) {
        if ((tid & 63) == 0) atomicAdd(&hist[first], uint32_t(__popcll(who)));
      } else if (in) {
        atomicAdd(&hist[bin], 1u);
      }
    });
    __syncthreads();
    // from the largest bin down, two bins a thread: the bin that holds the need-th key
    const uint32_t hi = hist[kBins - 1 - 2 * tid], lo = hist[kBins - 2 - 2 * tid], x = wave_scan(hi + lo);
    uint32_t all;
    const uint32_t before = waves_before(x, s, &all) + x - hi - lo;
    if (before < need && need <= before + hi + lo) {
      const bool upper = need <= before + hi;
      found[0] = upper ? kBins - 1 - 2 * tid : kBins - 2 - 2 * tid;
      found[1] = upper ? before : before + hi;
      found[2] = upper ? hi : lo;
    }
    __syncthreads();
    T |= found[0] << shift;
    need -= found[1];
    if (need == found[2] || shift == 0) return {T, need, need == found[2]};
    bits = shift == 21 ? 11 : 10;
    shift = shift == 21 ? 10 : 0;
  }
}

// exclusive prefix sums of n <= kSelect values in LDS; returns the total
__device__ __forceinline__ uint32_t block_scan(uint32_t* tab, uint32_t n, uint32_t* s) {
  const uint32_t tid = threadIdx.x;
  __syncthreads();
  const uint32_t v = tid < n ? tab[tid] : 0u, x = wave_scan(v);
  uint32_t all;
  const uint32_t before = waves_before(x, s, &all);
  if (tid < n) tab[tid] = before + x - v;
  __syncthreads();
  return all;
}

__device__ __forceinline__ uint32_t below(uint64_t ballot, int lane) {
  return __popcll(ballot & ((uint64_t(1) << lane) - 1));
}

// the K and V rows of `n` moves, 16 bytes a lane, row16 lanes a row.  What lay in a page outside the pool is lost:
// its new slot, which good pages may surround, becomes NaN (all bits set, in every type), so that the attention
// over it still says so.
__device__ __forceinline__ void move_rows(const EvictArgs& a, uint32_t row, uint32_t h, const uint32_t* to,
                                          const uint32_t* from, uint32_t n, uint32_t first, uint32_t step, uint32_t lane) {
  bool lost = false;
  for (uint32_t i = first; i < n; i += step) {
    const uint32_t d = to[i], s = from[i];
    uint32_t pd, ps;
    if (!a.c.page_of(row, d, &pd)) continue;
    if (!a.c.page_of(row, s, &ps)) {
      lost = true;
      continue;
    }
    const size_t od = a.c.at(pd, h, d) * a.elem + lane * 16, os = a.c.at(ps, h, s) * a.elem + lane * 16;
    const u32x4_t kk = ld_once(reinterpret_cast<const u32x4_t*>(a.c.k + os));
    const u32x4_t vv = ld_once(reinterpret_cast<const u32x4_t*>(a.c.v + os));
    st_once(reinterpret_cast<u32x4_t*>(a.c.k + od), kk);
    st_once(reinterpret_cast<u32x4_t*>(a.c.v + od), vv);
  }
  if (!lost) return;
  for (uint32_t i = first; i < n; i += step) {
    uint32_t pd, ps;
    if (!a.c.page_of(row, to[i], &pd) || a.c.page_of(row, from[i], &ps)) continue;
    const size_t od = a.c.at(pd, h, to[i]) * a.elem + lane * 16;
    *reinterpret_cast<u32x4_t*>(a.c.k + od) = *reinterpret_cast<u32x4_t*>(a.c.v + od) = u32x4_t{~0u, ~0u, ~0u, ~0u};
  }
}

// One workgroup per (row, kv head): the slots' keys in registers (thread tid holds slots tid, tid + 1024, ..,
// KPT of them), read once; the threshold from histograms of its digits; then the ranks of the holes and of the
// movers among the slots, from one table of counts per (1024 slots, wave).
// Bound by the latency of its steps and by its 16 waves meeting at barriers: 2049 slots to 2048 6.7 us, 1088 to 1024
// 10 us, 128 x 8320 slots to 2080 18 us (256 threads instead of 1024: 14.5 us for 2049 slots).
template <int KPT>
__global__ void __launch_bounds__(kSelect) k_evict_select(EvictArgs a) {
  __shared__ uint32_t s_tab[KPT * kSelWaves], s_red[kSelWaves], s_found[3], s_moves[2 * kFusedMoves], s_hist[kBins];
  __shared__ uint64_t s_least[2][kSelWaves];
  const uint32_t item = blockIdx.x, row = item / a.c.KV, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const uint32_t raw = uint32_t(gld(a.lens + row));
  const bool bad = raw > a.max_len;
  const uint32_t len = bad ? 0u : raw, keep = min(len, a.budget);
  if (tid == 0 && item % a.c.KV == 0 && !a.in_place) a.lens_out[row] = bad ? int32_t(raw) : int32_t(keep);
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
  // (up to max_len, not to the row's length: the loads do not wait for it)
  auto slot_of = [&](int k) { return min(k * kSelect + tid, a.max_len - 1); };
  if constexpr (kHold) {
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
      p[k] = gld(pos + slot_of(k));
      w[k] = gld(weight + slot_of(k));
    }
  }
  if (len == 0) {  // (the whole workgroup)
    if (tid == 0) a.n_moves[item] = 0;
    return;
  }
#pragma unroll
  for (int k = 0; k < KPT; ++k) newest = max(newest, k * kSelect + tid >= len ? INT32_MIN : kHold ? p[k % HOLD] : gld(pos + slot_of(k)));
  newest = block_max(newest, reinterpret_cast<int32_t*>(s_red));
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const float wk = kHold ? w[k % HOLD] : gld(weight + slot_of(k));
    const int32_t pk = kHold ? p[k % HOLD] : gld(pos + slot_of(k));
    key[k] = k * kSelect + tid < len ? slot_key(a, wk, pk, newest) : 0u;
  }

  uint32_t kept = 0;  // bit k: slot k * kSelect + tid
  auto is_kept = [&](int k) { return (kept >> k & 1) != 0; };
  if (len - keep <= kFew) {
    // (the same in all threads.)  A cache that is full drops a slot or a few at every step: one after the other the
    // slot that goes first, 0.35 us each, where the threshold and the ranks of its ties take 4.5 us
#pragma unroll
    for (int k = 0; k < KPT; ++k)
      if (k * kSelect + tid < len) kept |= 1u << k;
    for (uint32_t i = 0; i < len - keep; ++i) {
      uint64_t least = ~uint64_t(0);  // (the key, then the higher slot first)
#pragma unroll
      for (int k = 0; k < KPT; ++k)
        if (is_kept(k)) least = min(least, uint64_t(key[k]) << 32 | ~(k * kSelect + tid));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1)
        least = min(least, uint64_t(pair_u(uint32_t(least >> 32), o)) << 32 | pair_u(uint32_t(least), o));
      if (lane == 0) s_least[i & 1][wave] = least;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kSelWaves; ++w) least = min(least, s_least[i & 1][w]);
      const uint32_t slot = ~uint32_t(least);
      if (slot % kSelect == tid) kept &= ~(1u << slot / kSelect);
    }
  } else {
    const Threshold th = find_threshold(len, keep, s_hist, s_red, s_found, [&](auto f) {
#pragma unroll
      for (int k = 0; k < KPT; ++k) {
        if (uint32_t(k) * kSelect >= len) break;
        f(k * kSelect + tid < len, key[k]);
      }
    });

    // of the keys equal to the threshold the first `ties` slots stay
#pragma unroll
    for (int k = 0; k < KPT; ++k)
      if (k * kSelect + tid < len && key[k] >= th.T) kept |= 1u << k;
    if (!th.all) {
#pragma unroll
      for (int k = 0; k < KPT; ++k) {
        const uint64_t eq = __ballot(is_kept(k) && key[k] == th.T);
        if (lane == 0) s_tab[k * kSelWaves + wave] = __popcll(eq);
      }
      block_scan(s_tab, KPT * kSelWaves, s_red);
#pragma unroll
      for (int k = 0; k < KPT; ++k) {
        const bool eq = is_kept(k) && key[k] == th.T;
        const uint32_t rank = s_tab[k * kSelWaves + wave] + below(__ballot(eq), lane);
        if (eq && rank >= th.ties) kept &= ~(1u << k);
      }
      __syncthreads();
    }
  }
  // holes in the lower, movers in the upper half of a count (either is at most half of kLongest)
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const uint32_t j = k * kSelect + tid;
    const uint32_t holes = __popcll(__ballot(j < keep && !is_kept(k))), movers = __popcll(__ballot(j >= keep && is_kept(k)));
    if (lane == 0) s_tab[k * kSelWaves + wave] = holes | movers << 16;
  }
  const uint32_t moves = block_scan(s_tab, KPT * kSelWaves, s_red) & 0xffffu;
  const bool fused = a.fused != 0;
  uint32_t *to = fused ? s_moves : a.moves + size_t(item) * a.half * 2, *from = to + (fused ? kFusedMoves : a.half);
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const uint32_t j = k * kSelect + tid;
    const bool hole = j < keep && !is_kept(k), mover = j >= keep && is_kept(k);
    const uint32_t at = s_tab[k * kSelWaves + wave];
    const uint32_t rh = (at & 0xffffu) + below(__ballot(hole), lane), rm = (at >> 16) + below(__ballot(mover), lane);
    if (hole) to[rh] = j;
    if (mover) from[rm] = j;
    if (j < keep && is_kept(k)) {
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
constexpr uint32_t kLongest = 32 * kSelect;
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
  __shared__ uint32_t s_red[kSelWaves], s_found[3], s_hist[kBins];
  const uint32_t item = blockIdx.x, row = item / a.c.KV, tid = threadIdx.x;
  const uint32_t raw = uint32_t(gld(a.lens + row));
  const bool bad = raw > a.max_len;
  const uint32_t len = bad ? 0u : raw, keep = min(len, a.budget);
  if (tid == 0 && item % a.c.KV == 0 && !a.in_place) a.lens_out[row] = bad ? int32_t(raw) : int32_t(keep);
  const size_t base = size_t(item) * a.stride;
  const float* weight = a.weight + base;
  const int32_t* pos = a.pos + base;

  int32_t newest = INT32_MIN;
  for (uint32_t j = tid; j < len; j += kSelect) newest = max(newest, pos[j]);
  newest = block_max(newest, reinterpret_cast<int32_t*>(s_red));
  auto key = [&](uint32_t j) { return slot_key(a, gld(weight + j), gld(pos + j), newest); };
  const Threshold th = find_threshold(len, keep, s_hist, s_red, s_found, [&](auto f) {
    for (uint32_t j0 = 0; j0 < len; j0 += kSelect) f(j0 + tid < len, j0 + tid < len ? key(j0 + tid) : 0u);
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

// the moves that the selection left, `parts` workgroups per (row, kv head).  128 x 1560 moves of 256-byte
// rows 48.5 us, 4.2 TB/s read and written: a thread has one row in flight, behind its slots' and pages' numbers.
__global__ void __launch_bounds__(256) k_evict_move(EvictArgs a, uint32_t parts) {
  const uint32_t item = blockIdx.x / parts, part = blockIdx.x % parts, per = 256 / a.row16;
  const uint32_t *to = a.moves + size_t(item) * a.half * 2, *from = to + a.half;
  move_rows(a, item / a.c.KV, item % a.c.KV, to, from, gld(a.n_moves + item), part * per + threadIdx.x / a.row16,
            parts * per, threadIdx.x % a.row16);
}

__global__ void __launch_bounds__(256) k_evict_lens(EvictArgs a) {
  const uint32_t row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  const uint32_t len = uint32_t(a.lens_out[row]);
  if (len <= a.max_len) a.lens_out[row] = int32_t(min(len, a.budget));
}

size_t evict_bytes(const chpe_kv_pages* c, uint32_t max_len, size_t* off) {
  const size_t items = size_t(c->rows) * c->kv_heads, half = max_len / 2 + 1;
  *off = (items * 4 + 255) / 256 * 256;
  return *off + items * half * 8;
}

bool evict_shape_ok(const chpe_kv_pages* c, uint32_t max_len) {
  return uint64_t(max_len) <= uint64_t(c->pages_per_row) * c->page_size &&
         uint64_t(c->rows) * c->kv_heads <= kMaxItems / kSelect;
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
  a.in_place = lens_out == lens ? 1 : 0;
  a.fused = most <= kFusedMoves && max_len <= kLongest ? 1 : 0;
  const uint64_t items = uint64_t(cache->rows) * cache->kv_heads;
  const uint32_t parts = std::max(1u, std::min({8u, most / 64, uint32_t(kMaxBlocks / items)}));
  const bool ok = max_len == 0              ? launch(&k_evict_select_long, items, kSelect, st, a)  // (lens_out)
                  : max_len <= kSelect      ? launch(&k_evict_select<1>, items, kSelect, st, a)
                  : max_len <= 4 * kSelect  ? launch(&k_evict_select<4>, items, kSelect, st, a)
                  : max_len <= 16 * kSelect ? launch(&k_evict_select<16>, items, kSelect, st, a)
                  : max_len <= kLongest     ? launch(&k_evict_select<32>, items, kSelect, st, a)
                                            : launch(&k_evict_select_long, items, kSelect, st, a);
  if (!ok || (most != 0 && !a.fused && !launch(&k_evict_move, items * parts, 256, st, a, parts))) return -3;
  if (a.in_place && max_len > budget && !launch(&k_evict_lens, (cache->rows + 255) / 256, 256, st, a)) return -3;
  return 0;
}
