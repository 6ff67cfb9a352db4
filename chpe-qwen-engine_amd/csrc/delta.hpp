// delta.hpp -- what the operators of the gated delta rule over a pool of states share: rows of tokens and
// their slots on the device, typed loads and stores, the checks of their descriptions on the host.
#pragma once
#include "paged.hpp"

namespace chpe {

// The rows of a call: row r is tokens starts[r] .. starts[r + 1] - 1 (starts null: token r alone); its state is
// read from slot_in[r] and left in slot_out[r].
struct DeltaRows {
  const int32_t *starts, *slot_in, *slot_out;
  uint32_t tokens, rows, n_slots;

  // false for a row whose range does not lie in the tokens: it is left out
  __device__ bool range(uint32_t row, uint32_t* lo, uint32_t* hi) const {
    if (!starts) {
      *lo = row;
      *hi = row + 1;
      return true;
    }
    *lo = uint32_t(dev::gld(starts + row));
    *hi = uint32_t(dev::gld(starts + row + 1));
    return *lo <= *hi && *hi <= tokens;
  }
  // A launch does not know the rows' lengths, so a row's blocks of 1 << shift tokens have the numbers from
  // starts[r] / block + r on: at most the next row's first number, tokens / block + rows in all, and a row
  // without tokens has one too.  The row that holds block `b` (-1: none), 64 candidates a step.
  __device__ int row_of(uint32_t b, int shift, int lane) const {
    uint32_t at = 0, n = rows;
    do {
      const uint32_t step = (n + 63) / 64, r = at + min(uint32_t(lane) * step, n - 1);
      const uint32_t first = uint32_t(max(dev::gld(starts + r), 0)) >> shift;
      const uint64_t in = __ballot(uint32_t(lane) * step < n && first + r <= b);
      if (in == 0) return -1;
      const uint32_t last = 63u - uint32_t(__builtin_clzll(in));
      at += last * step;
      n = min(step, n - last * step);
    } while (n > 1);
    return int(at);
  }
  __device__ uint32_t first_block(uint32_t row, uint32_t lo, int shift) const { return (lo >> shift) + row; }
  // slot of the pool (*fill is not used), or -1: all values before are *fill, 0 for a new sequence (slot -1) and
  // NaN for a slot outside the pool
  __device__ int before(uint32_t row, float* fill) const {
    const int s = dev::gld(slot_in + row);
    *fill = s == -1 ? 0.0f : __builtin_nanf("");
    return uint32_t(s) < n_slots ? s : -1;
  }
  // slot that receives the state, or -1: it is not kept
  __device__ int after(uint32_t row) const {
    const int s = dev::gld(slot_out + row);
    return uint32_t(s) < n_slots ? s : -1;
  }
};

// A chpe_delta_states and a chpe_delta_tokens on the device.
struct DeltaArgs {
  DeltaRows r;
  float* state;
  uint64_t slot_stride;
  const void *q, *k, *v, *z;
  void* out;
  uint64_t q_stride, k_stride, v_stride, z_stride, out_stride, a_stride, b_stride;
  const float *a, *b, *A_log, *dt_bias, *norm_w;
  uint32_t NV, NK;
  float eps;
};

// The rows of up to `longest` tokens, token by token (delta_step.hip).
bool launch_delta_tokens(const DeltaArgs& a, uint32_t head_dim, int type, uint32_t longest, hipStream_t st);
namespace {

// N consecutive elements (16 bytes, or all N where they are fewer) widened to f32, and rounded from it
template <int N>
__device__ __forceinline__ void ld_row(const float* p, float (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = dev::ld_f4(p + i);
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = dev::gld(p + i);
  }
}
template <int N, class T>
__device__ __forceinline__ void widen(const uint32_t (&w)[N / 2], float (&x)[N], const T*) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, Bf16)) {
      x[2 * i] = dev::half_lo(w[i]);
      x[2 * i + 1] = dev::half_hi(w[i]);
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int N, class T>
__device__ __forceinline__ void ld_row(const T* p, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = Elem<T>::get(p);
    return;
  } else {
    uint32_t w[N / 2];
    const uint32_t* s = reinterpret_cast<const uint32_t*>(p);
    if constexpr (N % 8 == 0) {
#pragma unroll
      for (int i = 0; i < N / 2; i += 4) {
        const dev::u32x4_t v = dev::gld(reinterpret_cast<const dev::u32x4_t*>(s + i));
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else if constexpr (N == 4) {
      const dev::u32x2_t v = dev::gld(reinterpret_cast<const dev::u32x2_t*>(s));
      w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = dev::gld(s + i);
    }
    widen<N>(w, x, p);
  }
}
template <int N>
__device__ __forceinline__ void st_row(float* p, const float (&x)[N]) {
  static_assert(N % 4 == 0, "");
#pragma unroll
  for (int i = 0; i < N; i += 4) st_once(reinterpret_cast<dev::f32x4_t*>(p + i), dev::f32x4_t{x[i], x[i + 1], x[i + 2], x[i + 3]});
}
template <int N, class T>
__device__ __forceinline__ void st_row(T* p, const float (&x)[N]) {
  static_assert(N % 4 == 0, "");
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = uint32_t(__builtin_bit_cast(uint16_t, Elem<T>::put(x[2 * i]))) |
           uint32_t(__builtin_bit_cast(uint16_t, Elem<T>::put(x[2 * i + 1]))) << 16;
  uint32_t* d = reinterpret_cast<uint32_t*>(p);
#pragma unroll
  for (int i = 0; i < N / 2; i += 4) {
    if constexpr (N % 8 == 0)
      st_once(reinterpret_cast<dev::u32x4_t*>(d + i), dev::u32x4_t{w[i], w[i + 1], w[i + 2], w[i + 3]});
    else
      st_once(reinterpret_cast<dev::u32x2_t*>(d + i), dev::u32x2_t{w[i], w[i + 1]});
  }
}

// x / (1 + e^-x), off by at most 8 u of itself from x = -87 on, u = 2^-24: e^-x as 2^t (2 u) times 1 + what the product t lost
// (2 u), the sum 1 u, the reciprocal 2 u, the product 1 u.  Below, the reciprocal is no normal number and may come out as 0,
// and so may the result: off by 87 e^-87 = 1.4e-36 at most.  (x / (1 + expf(-x)) loses e^-x from -88.7 on, too.)  With expf and
// a division the convolution was bound by them: 78 us instead of 54 for 67 million bf16 values.  (Beyond 200 e^-x is 0 or
// infinite either way.)
__device__ __forceinline__ float delta_silu(float x) {
  const float y = __builtin_amdgcn_fmed3f(x, -200.0f, 200.0f), t = y * -1.44269502f;  // log2 e rounded, and the rest of it
  const float lost = fmaf(y, -1.92596303e-8f, fmaf(y, -1.44269502f, -t));
  const float e = __builtin_amdgcn_exp2f(t) * fmaf(lost, 0.693147182f, 1.0f);
  return x * __builtin_amdgcn_rcpf(1.0f + e);
}
// log of a token's decay, -exp(A_log) softplus(a + dt_bias), and its beta
__device__ __forceinline__ float delta_log_decay(float A_log, float x) {
  return -expf(A_log) * (x > 20.0f ? x : log1pf(expf(x)));
}
__device__ __forceinline__ float delta_beta(float b) { return 1.0f / (1.0f + expf(-b)); }

// ---- host -------------------------------------------------------------------------------------------------
constexpr uint32_t kMaxTokens = 0x7fffffffu;
constexpr uint64_t kMaxExtent = uint64_t(1) << 60;  // elements between the first and the last of a stride's steps

// `n` rows of `width` elements (16-bit or 32-bit by type) that start at 16-byte boundaries, `stride` apart
inline bool rows_ok(const void* p, uint64_t stride, uint64_t width, uint64_t n, int type) {
  if (!p || !aligned16(p)) return false;
  return n <= 1 || (stride >= width && stride % (type == 0 ? 4 : 8) == 0 && stride <= kMaxExtent / n);
}

inline bool delta_rows_ok(uint32_t tokens, uint32_t rows, const int32_t* slot_in, const int32_t* slot_out) {
  return tokens <= kMaxTokens && rows <= kMaxTokens && (rows == 0 || (slot_in && slot_out));
}

inline bool delta_states_ok(const chpe_delta_states* s) {
  if (!s || s->n_slots == 0 || s->n_slots > kMaxTokens || (s->head_dim != 64 && s->head_dim != 128)) return false;
  if (s->k_heads == 0 || s->v_heads == 0 || s->v_heads % s->k_heads != 0 || s->v_heads > 65536) return false;
  return rows_ok(s->state, s->slot_stride, uint64_t(s->v_heads) * s->head_dim * s->head_dim, s->n_slots, 0);
}

inline bool delta_from(const chpe_delta_states* s, const chpe_delta_tokens* t, uint32_t tokens, uint32_t rows,
                       const int32_t* starts, const int32_t* slot_in, const int32_t* slot_out, DeltaArgs* out) {
  if (!delta_states_ok(s) || !t || t->type < 0 || t->type > 2) return false;
  if (!delta_rows_ok(tokens, rows, slot_in, slot_out)) return false;
  const uint64_t kw = uint64_t(s->k_heads) * s->head_dim, vw = uint64_t(s->v_heads) * s->head_dim;
  if (tokens != 0) {
    if (!rows_ok(t->q, t->q_stride, kw, tokens, t->type) || !rows_ok(t->k, t->k_stride, kw, tokens, t->type) ||
        !rows_ok(t->v, t->v_stride, vw, tokens, t->type) || !rows_ok(t->out, t->out_stride, vw, tokens, t->type))
      return false;
    if (t->z && !rows_ok(t->z, t->z_stride, vw, tokens, t->type)) return false;
    if (!t->a || !t->b || !t->A_log || !t->dt_bias || (t->z == nullptr) != (t->norm_w == nullptr) || !aligned16(t->norm_w)) return false;
    if (tokens > 1 && (t->a_stride < s->v_heads || t->b_stride < s->v_heads || t->a_stride > kMaxExtent / tokens ||
                       t->b_stride > kMaxExtent / tokens))
      return false;
  }
  *out = DeltaArgs{{starts, slot_in, slot_out, tokens, rows, s->n_slots}, s->state, s->n_slots > 1 ? s->slot_stride : 0,
                   t->q, t->k, t->v, t->z, t->out, t->q_stride, t->k_stride, t->v_stride, t->z_stride, t->out_stride,
                   t->a_stride, t->b_stride, t->a, t->b, t->A_log, t->dt_bias, t->norm_w, s->v_heads, s->k_heads, t->eps};
  return true;
}

}  // namespace
}  // namespace chpe
