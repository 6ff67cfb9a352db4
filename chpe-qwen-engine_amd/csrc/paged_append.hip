// paged_append.hip -- chpe_paged_append: what a layer writes into the paged cache, in one pass over the
// projections' outputs.  Per token and head: RMSNorm of the query or key over the head's dims (where
// gains are given), the rotary embedding of its first rot dims, y0 = x0 c - x1 s, y1 = x0 s + x1 c with
// the pair (i, i + rot/2) or (2i, 2i + 1); keys and values are rounded once to the cache's type, queries
// stay f32.  The arithmetic of k_hyb_qk (hybrid.hip) on caller buffers.
#include <utility>

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

template <int HD, class T>
__global__ void __launch_bounds__(HD) k_paged_append(AppendArgs a) {
#pragma clang fp contract(off)
  const uint32_t per = a.H + 2 * a.c.KV, t = blockIdx.x / per, b = blockIdx.x % per, d = threadIdx.x;
  const bool is_q = b < a.H, is_k = !is_q && b < a.H + a.c.KV;
  const uint32_t h = is_q ? b : (is_k ? b - a.H : b - a.H - a.c.KV);
  __shared__ float s_x[HD], s_red[HD / 64];
  const int32_t pos = gld(a.pos + t);
  float x = is_q ? gld(a.q + t * a.q_stride + h * a.q_head_stride + d)
                 : gld((is_k ? a.k + t * a.k_stride : a.v + t * a.v_stride) + h * HD + d);
  const float* gain = is_q ? a.q_norm : a.k_norm;
  const bool turns = a.rot == 0 || (pos >= 0 && uint32_t(pos) < a.rope_rows);
  if (is_q || is_k) {
    if (gain) {
      const float s2 = wave_sum(x * x);
      if ((d & 63) == 0) s_red[d >> 6] = s2;
      __syncthreads();
      float tot = 0.0f;
      for (int w = 0; w < HD / 64; ++w) tot += s_red[w];
      x = x * (1.0f / sqrtf(tot / float(HD) + a.eps)) * gain[d];
    }
    s_x[d] = x;
    __syncthreads();
    const uint32_t half = a.rot / 2;
    if (d < a.rot && turns) {
      const uint32_t i = a.interleaved ? d / 2 : (d < half ? d : d - half);
      const bool first = a.interleaved ? (d & 1) == 0 : d < half;
      const float c = a.rope_cos[size_t(pos) * half + i], s = a.rope_sin[size_t(pos) * half + i];
      const float x0 = a.interleaved ? s_x[2 * i] : s_x[i], x1 = a.interleaved ? s_x[2 * i + 1] : s_x[i + half];
      x = first ? x0 * c - x1 * s : x0 * s + x1 * c;
    }
  }
  if (is_q) {
    a.q_out[(size_t(t) * a.H + h) * HD + d] = turns ? x : __builtin_nanf("");
    return;
  }
  const int32_t row = gld(a.row + t), slot = gld(a.slot + t);
  if (row < 0 || uint32_t(row) >= a.rows || slot < 0 || uint32_t(slot) >= a.c.capacity || !turns) return;
  uint32_t page;
  if (!a.c.page_of(row, slot, &page)) return;
  reinterpret_cast<T*>(is_k ? a.c.k : a.c.v)[a.c.at(page, h, slot) + d] = Elem<T>::put(x);
  if (is_k && d == 0 && uint64_t(slot) < a.track_stride) {
    const size_t at = (size_t(row) * a.c.KV + h) * a.track_stride + slot;
    if (a.slot_pos) a.slot_pos[at] = pos;
    if (a.slot_weight) a.slot_weight[at] = 0.0f;
  }
}

template <class T>
bool launch_append(const AppendArgs& a, uint32_t hd, hipStream_t st) {
  const uint64_t blocks = uint64_t(a.tokens) * (a.H + 2 * a.c.KV);
  if (hd == 64) return launch(&k_paged_append<64, T>, blocks, 64, st, a);
  if (hd == 128) return launch(&k_paged_append<128, T>, blocks, 128, st, a);
  return launch(&k_paged_append<256, T>, blocks, 256, st, a);
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
  if (heads != 0 && (q_head_stride < hd || (tokens > 1 && q_stride < (heads - 1) * q_head_stride + hd))) return -1;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(q_norm) || !aligned16(k_norm) ||
      q_stride % 4 || q_head_stride % 4 || k_stride % 4 || v_stride % 4)
    return -1;
  if (rot_dim > hd || rot_dim % 8 != 0 || (rot_dim != 0 && (!rope_cos || !rope_sin || rope_rows == 0))) return -1;
  if (!aligned16(rope_cos) || !aligned16(rope_sin)) return -1;
  if ((slot_pos || slot_weight) && track_stride == 0) return -1;
  if (heads > 65536 || cache->kv_heads > 65536 || uint64_t(tokens) * (heads + 2 * cache->kv_heads) > kMaxBlocks) return -1;
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
