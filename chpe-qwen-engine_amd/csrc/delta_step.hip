// delta_step.hip -- chpe_delta_step: one token per row of the gated delta rule over a pool of states.
// Per value head, with q, k l2-normalised, q over sqrt(head_dim) too, d the token's decay and b its beta:
//   S' = d S,  S = S' + k (b (v - S'^T k))^T,  o = S^T q,  and optionally w * o / rms(o) * silu(z).
#include "delta.hpp"

namespace chpe {
namespace {
using namespace dev;

// A workgroup takes one value head of one row: its threads hold the state, 4 columns of D / 16 or D / 8 rows each (16 or 8
// groups of rows), 16 bytes a lane, read once and written once.  The column sums (S^T k before the update, S^T q after it) meet
// over the groups of a wave, then over the waves in LDS, in a fixed order.
// Bound by memory: 2 x 64 KB a head of 128 (256 rows of the 9B layout, 1.08 GB: 189 us, 5.7 TB/s; 33 rows, 141 MB: 25 us; one
// row, 4 MB: 6.5 us, the latencies of the slot's number, the state and the sums).  ONE: a token per row, with nothing to load ahead; else rows of up to `longest`, the
// next token's inputs on the way meanwhile.  (16 groups for one token at D = 128: 256 rows take 207 us with 8; 8 for
// more: 32 rows of 5 tokens take 54 us with 16, 46 with 8.)
template <int D, bool ONE>
constexpr int kGroups = D == 64 || ONE ? 16 : 8;
template <int D, class T, bool ONE>
__global__ void __launch_bounds__((kGroups<D, ONE> * D / 4)) k_delta_step(DeltaArgs a, uint32_t longest) {
  constexpr int LPR = D / 4, RG = kGroups<D, ONE>, RPT = D / RG, PL = D / 64, NW = RG * LPR / 64;
  const uint32_t h = blockIdx.x % a.NV, row = blockIdx.x / a.NV, kh = h / (a.NV / a.NK);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = tid % LPR * 4, rg = tid / LPR;
  __shared__ float s_q[D], s_k[D];
  __shared__ __align__(16) float s_sum[2][NW][D];
  uint32_t lo, hi;
  float fill;
  const bool there = a.r.range(row, &lo, &hi);
  const int slot = a.r.before(row, &fill), to = a.r.after(row);
  if (!there || hi - lo > longest) return;
  const bool any = ONE || lo < hi;
  float A_log = 0.0f, dt = 0.0f, w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (any) {  // (a call without tokens has none of these)
    A_log = gld(a.A_log + h);
    dt = gld(a.dt_bias + h);
    if (a.z) ld_row(a.norm_w + c, w);
  }
  struct Token {
    float v[4], x[PL], y[PL], z[4], a, b;
  };
  auto load = [&](uint32_t t) {
    Token k;
    ld_row(static_cast<const T*>(a.q) + t * a.q_stride + kh * D + lane * PL, k.x);
    ld_row(static_cast<const T*>(a.k) + t * a.k_stride + kh * D + lane * PL, k.y);
    ld_row(static_cast<const T*>(a.v) + t * a.v_stride + h * D + c, k.v);
    if (a.z) ld_row(static_cast<const T*>(a.z) + t * a.z_stride + h * D + c, k.z);
    k.a = gld(a.a + t * a.a_stride + h);
    k.b = gld(a.b + t * a.b_stride + h);
    return k;
  };
  Token next;  // (requested before the state, whose slot is on its way)
  if (any) next = load(lo);
  float s[RPT][4];
  // (the head's place is the same for all lanes: scalar registers hold the rows' addresses)
  const uint32_t at = rg * D + c;
  if (slot >= 0) {
    const float* S = a.state + uniform(slot) * a.slot_stride + size_t(h) * D * D;
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      const f32x4_t v = ld_once(reinterpret_cast<const f32x4_t*>(S + r * RG * D + at));
      s[r][0] = v.x, s[r][1] = v.y, s[r][2] = v.z, s[r][3] = v.w;
    }
  } else {
#pragma unroll
    for (int r = 0; r < RPT; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] = fill;
  }
  // a column's total over the row groups, in every thread
  auto total = [&](float (&p)[4], int buf) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (LPR == 16) p[e] = pair_sum(p[e], 16);
      p[e] = pair_sum(p[e], 32);
    }
    if (lane < LPR) *reinterpret_cast<float4*>(&s_sum[buf][wave][c]) = make_float4(p[0], p[1], p[2], p[3]);
    __syncthreads();
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(&s_sum[buf][w][c]);
      t.x += x.x, t.y += x.y, t.z += x.z, t.w += x.w;
    }
    p[0] = t.x, p[1] = t.y, p[2] = t.z, p[3] = t.w;
  };
  for (uint32_t t = lo; t < hi; ++t) {
    const Token now = next;
    const float(&v)[4] = now.v, (&x)[PL] = now.x, (&y)[PL] = now.y, (&z)[4] = now.z;
    if (!ONE && t + 1 < hi) next = load(t + 1);
    const float decay = expf(delta_log_decay(A_log, now.a + dt)), beta = delta_beta(now.b);
    float q2 = 0.0f, k2 = 0.0f;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      q2 = fmaf(x[i], x[i], q2);
      k2 = fmaf(y[i], y[i], k2);
    }
    const float qi = 1.0f / sqrtf(wave_sum(q2) + 1e-6f) * (1.0f / sqrtf(float(D))), ki = 1.0f / sqrtf(wave_sum(k2) + 1e-6f);
    if (!ONE && t != lo) __syncthreads();  // (s_q, s_k)
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        s_q[lane * PL + i] = x[i] * qi;
        s_k[lane * PL + i] = y[i] * ki;
      }
    }
    __syncthreads();
    float p[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      const float k = s_k[rg + r * RG];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[r][e] *= decay;
        p[e] = fmaf(s[r][e], k, p[e]);
      }
    }
    total(p, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = (v[e] - p[e]) * beta;
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      const float k = s_k[rg + r * RG], q = s_q[rg + r * RG];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[r][e] = fmaf(k, p[e], s[r][e]);
        o[e] = fmaf(s[r][e], q, o[e]);
      }
    }
    total(o, 1);
    if (a.z) {  // (every group of D / 4 lanes holds the head's outputs)
      float s2 = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) s2 = fmaf(o[e], o[e], s2);
#pragma unroll
      for (int m = 1; m < LPR; m <<= 1) s2 = pair_sum(s2, m);
      const float rr = 1.0f / sqrtf(s2 / float(D) + a.eps);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = w[e] * (o[e] * rr) * delta_silu(z[e]);
    }
    if (rg == 0) st_row(static_cast<T*>(a.out) + t * a.out_stride + h * D + c, o);
  }
  if (to >= 0) {
    float* S = a.state + uniform(to) * a.slot_stride + size_t(h) * D * D;
#pragma unroll
    for (int r = 0; r < RPT; ++r) st_row(S + r * RG * D + at, s[r]);
  }
}

template <int D>
bool launch_step(const DeltaArgs& a, int type, uint32_t longest, hipStream_t st) {
  const uint64_t blocks = uint64_t(a.r.rows) * a.NV;
  auto run = [&](auto one, auto many) {
    return a.r.starts ? launch(many, blocks, kGroups<D, false> * D / 4, st, a, longest)
                      : launch(one, blocks, kGroups<D, true> * D / 4, st, a, longest);
  };
  return type == 0   ? run(&k_delta_step<D, float, true>, &k_delta_step<D, float, false>)
         : type == 1 ? run(&k_delta_step<D, _Float16, true>, &k_delta_step<D, _Float16, false>)
                     : run(&k_delta_step<D, Bf16, true>, &k_delta_step<D, Bf16, false>);
}

}  // namespace

bool launch_delta_tokens(const DeltaArgs& a, uint32_t head_dim, int type, uint32_t longest, hipStream_t st) {
  return head_dim == 128 ? launch_step<128>(a, type, longest, st) : launch_step<64>(a, type, longest, st);
}

}  // namespace chpe

using namespace chpe;

extern "C" int chpe_delta_step(const chpe_delta_states* states, const chpe_delta_tokens* t, uint32_t rows,
                               const int32_t* slot_in, const int32_t* slot_out, void* stream) {
  DeltaArgs a{};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!delta_from(states, t, rows, rows, nullptr, slot_in, slot_out, &a) || !stream_here(st)) return -1;
  if (uint64_t(rows) * a.NV > kMaxItems / 512) return -1;
  if (rows == 0) return 0;
  return launch_delta_tokens(a, states->head_dim, t->type, 1, st) ? 0 : -3;
}
