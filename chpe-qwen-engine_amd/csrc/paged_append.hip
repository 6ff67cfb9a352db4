// paged_append.hip -- chpe_paged_append: what a layer writes into the paged cache, in one pass over the
// projections' outputs.  Per token and head: RMSNorm of the query or key over the head's dims (where
// gains are given), the rotary embedding of its first rot dims, y0 = x0 c - x1 s, y1 = x0 s + x1 c with
// the pair (i, i + rot/2) or (2i, 2i + 1); keys and values are rounded once to the cache's type, queries
// stay f32.  The arithmetic of k_hyb_qk (hybrid.hip) on caller buffers.
#include <algorithm>

#include "paged.hpp"

namespace chpe {
namespace {
using namespace dev;

struct AppendArgs {
  Pages c;
  const float *q, *k, *v, *q_norm, *k_norm, *rope_cos, *rope_sin;
  const int32_t *row, *slot, *pos;
  float* q_out;
  int32_t* slot_pos;
  float* slot_weight;
  uint64_t q_stride, q_head_stride, k_stride, v_stride, track_stride;
  uint32_t tokens, H, rot, rope_rows, rows;
  int interleaved;
  float eps;
};

// HD / 4 lanes hold one head's row, 16 bytes each; a workgroup's 256 / (HD / 4) groups of lanes walk the rows
// of one token: the query heads, the key heads, the value heads.  A lane keeps the same dims in every row, so
// its gains, cosines and sines are read once.  Bound by memory where the tokens are many (8189 tokens of 80 rows
// of 128, fp16: 104 us, 6.2 TB/s read and written), else by two dependent loads (one token 2.8 us).
template <int HD, class T>
__global__ void __launch_bounds__(256) k_paged_append(AppendArgs a, uint32_t parts) {
#pragma clang fp contract(off)
  constexpr int L = HD / 4, GR = 256 / L, U = 4;  // U rows of a group in flight
  const uint32_t t = blockIdx.x / parts, part = blockIdx.x % parts;
  const uint32_t lane = threadIdx.x % L, d = lane * 4, n_rows = a.H + 2 * a.c.KV, half = a.rot / 2;
  const uint32_t step = parts * GR;
  uint32_t r = part * GR + threadIdx.x / L;
  const int32_t pos = gld(a.pos + t), row = gld(a.row + t), slot = gld(a.slot + t);
  const bool turns = a.rot == 0 || (pos >= 0 && uint32_t(pos) < a.rope_rows);
  // (uniform in the workgroup)
  uint32_t page = 0;
  const bool writes = turns && row >= 0 && uint32_t(row) < a.rows && slot >= 0 && uint32_t(slot) < a.c.capacity &&
                      a.c.page_of(row, slot, &page);
  f32x4_t x[U];
  auto load = [&](uint32_t at, f32x4_t& v) {
    v = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (at >= n_rows) return;
    const float* src = at < a.H ? a.q + t * a.q_stride + at * a.q_head_stride
                       : at < a.H + a.c.KV ? a.k + t * a.k_stride + size_t(at - a.H) * HD
                                           : a.v + t * a.v_stride + size_t(at - a.H - a.c.KV) * HD;
    v = ld_once(reinterpret_cast<const f32x4_t*>(src + d));
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(r + u * step, x[u]);
  float4 gq = make_float4(1, 1, 1, 1), gk = gq, cs = gq, sn = make_float4(0, 0, 0, 0);
  if (a.q_norm) gq = ld_f4(a.q_norm + d);
  if (a.k_norm) gk = ld_f4(a.k_norm + d);
  const bool in_rot = d < a.rot && turns;
  if (in_rot) {
    if (a.interleaved) {  // pairs d / 2 and d / 2 + 1
      const float2 c = *reinterpret_cast<const float2*>(a.rope_cos + size_t(pos) * half + d / 2);
      const float2 s = *reinterpret_cast<const float2*>(a.rope_sin + size_t(pos) * half + d / 2);
      cs = make_float4(c.x, c.x, c.y, c.y);
      sn = make_float4(-s.x, s.x, -s.y, s.y);
    } else {
      const uint32_t i = d < half ? d : d - half;
      cs = ld_f4(a.rope_cos + size_t(pos) * half + i);
      sn = ld_f4(a.rope_sin + size_t(pos) * half + i);
      if (d < half) sn = make_float4(-sn.x, -sn.y, -sn.z, -sn.w);
    }
  }
  // the lane of the other half of the pairs
  const int base = int(threadIdx.x & 63) - int(lane);
  const int other = base + (!in_rot ? int(lane) : d < half ? int(lane + half / 4) : int(lane - half / 4));

  while (true) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = r + u * step;
      f32x4_t y = x[u];
      load(at + U * step, x[u]);
      if (at - threadIdx.x / L >= n_rows) return;  // (the whole workgroup)
      const bool is_q = at < a.H, is_v = at >= a.H + a.c.KV;
      if ((is_q ? a.q_norm : a.k_norm) != nullptr && !is_v) {
        float s2 = (y.x * y.x + y.y * y.y) + (y.z * y.z + y.w * y.w);
#pragma unroll
        for (int o = 1; o < L; o <<= 1) s2 += __shfl_xor(s2, o);
        const float inv = 1.0f / sqrtf(s2 / float(HD) + a.eps);
        const float4 g = is_q ? gq : gk;
        y = f32x4_t{y.x * inv * g.x, y.y * inv * g.y, y.z * inv * g.z, y.w * inv * g.w};
      }
      if (a.rot != 0) {
        float4 z;  // the pairs' other halves
        if (a.interleaved) z = make_float4(y.y, y.x, y.w, y.z);
        else z = make_float4(__shfl(y.x, other), __shfl(y.y, other), __shfl(y.z, other), __shfl(y.w, other));
        if (in_rot && !is_v)
          y = f32x4_t{y.x * cs.x + z.x * sn.x, y.y * cs.y + z.y * sn.y, y.z * cs.z + z.z * sn.z, y.w * cs.w + z.w * sn.w};
      }
      if (at >= n_rows) continue;
      if (is_q) {
        if (!turns) y.x = y.y = y.z = y.w = __builtin_nanf("");
        st_once(reinterpret_cast<f32x4_t*>(a.q_out + (size_t(t) * a.H + at) * HD + d), y);
      } else if (writes) {
        const uint32_t h = is_v ? at - a.H - a.c.KV : at - a.H;
        T* dst = reinterpret_cast<T*>(is_v ? a.c.v : a.c.k) + a.c.at(page, h, slot) + d;
        struct alignas(4 * sizeof(T)) Four { T e[4]; };
        *reinterpret_cast<Four*>(dst) = Four{{Elem<T>::put(y.x), Elem<T>::put(y.y), Elem<T>::put(y.z), Elem<T>::put(y.w)}};
        if (!is_v && lane == 0 && uint64_t(slot) < a.track_stride) {
          const size_t i = (size_t(row) * a.c.KV + h) * a.track_stride + slot;
          if (a.slot_pos) a.slot_pos[i] = pos;
          if (a.slot_weight) a.slot_weight[i] = 0.0f;
        }
      }
    }
    r += U * step;
  }
}

// workgroups per token: one where the tokens alone fill the chip (4 workgroups a CU), as many as its rows
// allow where they are few (501 tokens of 24 rows of 256: 3 workgroups a token 8.0 us, 5 9.3 us; one token
// 2.8 us)
uint32_t token_parts(uint32_t tokens, uint32_t n_rows, uint32_t groups) {
  const uint32_t most = (n_rows + groups - 1) / groups, want = (1024 + tokens - 1) / tokens;
  return std::max(1u, std::min(most, want));
}

template <int HD, class T>
bool launch_append_hd(const AppendArgs& a, hipStream_t st) {
  const uint32_t parts = token_parts(a.tokens, a.H + 2 * a.c.KV, 256 / (HD / 4));
  return launch(&k_paged_append<HD, T>, uint64_t(a.tokens) * parts, 256, st, a, parts);
}
template <class T>
bool launch_append(const AppendArgs& a, uint32_t hd, hipStream_t st) {
  return hd == 64 ? launch_append_hd<64, T>(a, st) : hd == 128 ? launch_append_hd<128, T>(a, st) : launch_append_hd<256, T>(a, st);
}

}  // namespace
}  // namespace chpe

using namespace chpe;

extern "C" int chpe_paged_append(const chpe_kv_pages* cache, uint32_t tokens, uint32_t heads, const float* q,
                                 uint64_t q_stride, uint64_t q_head_stride, const float* k, uint64_t k_stride,
                                 const float* v, uint64_t v_stride, const float* q_norm, const float* k_norm, float eps,
                                 const float* rope_cos, const float* rope_sin, uint32_t rot_dim, uint32_t rope_rows,
                                 int interleaved, const int32_t* token_row, const int32_t* token_slot,
                                 const int32_t* token_pos, float* q_out, int32_t* slot_pos, float* slot_weight,
                                 uint64_t track_stride, void* stream) {
  AppendArgs a{};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!pages_from(cache, &a.c) || !stream_here(st)) return -1;
  const uint32_t hd = cache->head_dim;
  if (tokens == 0) return 0;
  if (!k || !v || !token_row || !token_slot || !token_pos || (heads != 0 && (!q || !q_out))) return -1;
  if (k_stride < uint64_t(cache->kv_heads) * hd || v_stride < uint64_t(cache->kv_heads) * hd) return -1;
  if (heads > 1 && q_head_stride > (uint64_t(1) << 60) / heads) return -1;  // (their extent fits 64 bits, as the pool's)
  if (heads != 0 && (q_head_stride < hd || (tokens > 1 && q_stride < (heads - 1) * q_head_stride + hd))) return -1;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(q_norm) || !aligned16(k_norm) ||
      q_stride % 4 || q_head_stride % 4 || k_stride % 4 || v_stride % 4)
    return -1;
  if (rot_dim > hd || rot_dim % 8 != 0 || (rot_dim != 0 && (!rope_cos || !rope_sin || rope_rows == 0))) return -1;
  if (!aligned16(rope_cos) || !aligned16(rope_sin)) return -1;
  if ((slot_pos || slot_weight) && track_stride == 0) return -1;
  if (heads > 65536 || cache->kv_heads > 65536 || uint64_t(tokens) * (heads + 2 * cache->kv_heads) > (uint64_t(1) << 31) ||
      uint64_t(tokens) > kMaxBlocks)
    return -1;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.rope_cos = rope_cos;
  a.rope_sin = rope_sin;
  a.row = token_row;
  a.slot = token_slot;
  a.pos = token_pos;
  a.q_out = q_out;
  a.slot_pos = slot_pos;
  a.slot_weight = slot_weight;
  a.q_stride = q_stride;
  a.q_head_stride = q_head_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.track_stride = track_stride;
  a.tokens = tokens;
  a.H = heads;
  a.rot = rot_dim;
  a.rope_rows = rope_rows;
  a.rows = cache->rows;
  a.interleaved = interleaved ? 1 : 0;
  a.eps = eps;
  const bool ok = cache->type == 0 ? launch_append<float>(a, hd, st)
                                   : cache->type == 1 ? launch_append<_Float16>(a, hd, st) : launch_append<Bf16>(a, hd, st);
  return ok ? 0 : -3;
}
