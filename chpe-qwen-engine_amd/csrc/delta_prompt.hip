// delta_prompt.hip -- chpe_delta_prompt: the gated delta rule over prompts, in chunks of 64 tokens.
// Within a chunk, with g_i the sum of the tokens' log decays up to i, G its value at the chunk's end, S the state
// before it, k and q normalised:
//   A_ij = b_i (k_i . k_j) e^(g_i - g_j) for j < i,  T = (I + A)^-1,  u = T diag(b) (v - e^g (K S))
//   o_i = e^g_i q_i S + sum_(j <= i) (q_i . k_j) e^(g_i - g_j) u_j,   S <- e^G S + sum_j e^(G - g_j) k_j u_j^T
// which is the recurrence of chpe_delta_step unrolled: u_j are the updates b (v - S'^T k) of its tokens.
// k_delta_prep forms T and the matrix of o for every chunk at once, k_delta_scan carries the state over a row's chunks
// and writes the outputs, k_delta_gnorm applies the gated norm, which needs a head's whole row.
#include <type_traits>

#include "delta.hpp"

namespace chpe {
namespace {
using namespace dev;

constexpr int kChunkShift = 6, kChunk = 1 << kChunkShift;
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// What a chunk of a value head leaves for the scan, as operands (mma below): u's matrix T diag(b) and o's matrix in
// fragments of 16 x 32, row w of 16 tokens in w / 2 + 1 of them; then per token the factors of K S, Q S and k u^T, e^G
// and whether all is finite.
constexpr int kFrag = 3 * 256;  // words
__device__ __host__ constexpr int frag_of(int w) { return w < 2 ? w : 2 * w - 2; }  // row w's first
constexpr int kOffO = 6 * kFrag, kOffScale = 12 * kFrag, kChunkFloats = kOffScale + 256;

struct PromptArgs {
  DeltaArgs d;
  float *chunks, *o32;  // o32 [token][NV][D]: the outputs before the gated norm, null without it
  uint32_t shortest;    // tokens of the shortest row that is theirs: the others run token by token (delta_step.hip)

  // the row's range; false for a row that is left out or not theirs
  __device__ bool range(uint32_t row, uint32_t* lo, uint32_t* hi) const {
    return d.r.range(row, lo, hi) && *hi - *lo >= shortest;
  }
  // The n-th longest of up to 64 rows that are theirs, -1 behind the last (of more rows: row n; of equal ones in their order):
  // workgroups start in order, and where they are several rounds a long row that starts late ends alone (24 rows of 1 to 4097
  // tokens in random orders: the scan 1.04 to 1.2 ms as they come, 1.0 so).
  __device__ int nth_longest(uint32_t n, uint32_t lane) const {
    if (d.r.rows > 64) return int(n);
    uint32_t lo = 0, hi = 0, rank = 0;
    const bool there = lane < d.r.rows && range(lane, &lo, &hi);
    const uint64_t all = __ballot(there);
    if (n >= uint32_t(__builtin_popcountll(all))) return -1;
    const uint32_t len = hi - lo;
    for (uint64_t left = all; left != 0; left &= left - 1) {
      const uint32_t j = uint32_t(__builtin_ctzll(left)), other = lane_of(len, int(j));
      rank += other > len || (other == len && j < lane) ? 1u : 0u;
    }
    return int(__builtin_ctzll(__ballot(there && rank == n)));
  }
  // the x-th of a row's value heads in workgroups' order: those of one key head on one XCD (workgroup i runs on XCD i % 8), whose
  // L2 they share (with two value heads a key head 8189 tokens in f32 fetch 151 and 424 MB in the two launches instead of 286 and 558)
  __device__ uint32_t head_of(uint32_t x) const {
    const uint32_t r = d.NV / d.NK;
    return d.NK % 8 != 0 ? x : (x % 8 + 8 * (x / (8 * r))) * r + x / 8 % r;
  }
};

// ---- products in 32 bits on the 16-bit matrix cores ---------------------------------------------------------
// A value is taken apart into bf16 parts: three hold all 24 bits of an f32, two an fp16, one a bf16.  Of the products of
// two values' parts those below 2^-25 of the whole are left out (three by three: six of nine remain), less than
// the rounding of the f32 sums.
template <class T>
constexpr int kParts = 0;
template <>
constexpr int kParts<float> = 3;
template <>
constexpr int kParts<_Float16> = 2;
template <>
constexpr int kParts<Bf16> = 1;

// the parts of two values, as words of two bf16
template <int N>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&w)[N]) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    w[p] = __builtin_bit_cast(uint32_t, b2_t{__bf16(x), __bf16(y)});
    x -= __uint_as_float(w[p] << 16);
    y -= __uint_as_float(w[p] & 0xffff0000u);
  }
}
template <int NA, int NB>
__device__ __forceinline__ f4_t mma(const u32x4_t (&a)[NA], const u32x4_t (&b)[NB], f4_t c) {
#pragma unroll
  for (int o = 2; o >= 0; --o)  // the small ones first
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (o - i >= 0 && o - i < NB)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a[i]), __builtin_bit_cast(b8_t, b[o - i]), c, 0, 0, 0);
  return c;
}
template <int N>
__device__ __forceinline__ void ld_parts(const u32x4_t (&src)[N][64], int lane, u32x4_t (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = src[i][lane];
}
// 16 x 16 by 16 x 16 in f32: a lane (G, n) holds row (or column) n, inner indexes 4 G + r
__device__ __forceinline__ f4_t mma16(f4_t a, f4_t b, f4_t c) {
#pragma unroll
  for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
  return c;
}

// A token's key or query row in a wave that holds 16 tokens: lane (G, i) = (lane / 16, lane % 16) has every fourth 16
// bytes of token i, from the G-th on (the four lanes of a token load next to each other).  Product s of D / 32 takes
// the next 8 of each lane's dims, in halves u: the inner index of a product is free as long as both sides agree, and
// so 16-bit rows are operands as they come.
template <int D, class T>
struct Row16 {
  static constexpr int W = D / 4 * int(sizeof(T)) / 16;
  u32x4_t w[W];
  // the dim of product s, half u, element r < 4
  static __device__ constexpr int dim(int G, int s, int u, int r) {
    return sizeof(T) == 4 ? 32 * s + 16 * u + 4 * G + r : 32 * s + 8 * G + 4 * u + r;
  }
  __device__ void load(const T* row, int G) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = gld(reinterpret_cast<const u32x4_t*>(row) + 4 * i + G);
  }
  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = u32x4_t{0, 0, 0, 0};
  }
  __device__ void pair(int e, float* x, float* y) const {  // elements e, e + 1 (e even)
    if constexpr (sizeof(T) == 4) {
      *x = __uint_as_float(w[e / 4][e % 4]);
      *y = __uint_as_float(w[e / 4][e % 4 + 1]);
    } else {
      const uint32_t v = w[e / 8][e / 2 % 4];
      if constexpr (__is_same(T, Bf16)) {
        *x = __uint_as_float(v << 16);
        *y = __uint_as_float(v & 0xffff0000u);
      } else {
        *x = half_lo(v);
        *y = half_hi(v);
      }
    }
  }
  __device__ void operand(int s, u32x4_t (&out)[kParts<T>]) const {
    if constexpr (__is_same(T, Bf16)) {
      out[0] = w[s];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x, y;
        uint32_t p[kParts<T>];
        pair(8 * s + 2 * e, &x, &y);
        split2(x, y, p);
#pragma unroll
        for (int i = 0; i < kParts<T>; ++i) out[i][e] = p[i];
      }
    }
  }
  __device__ float sum2() const {  // of the token's squares, in all its lanes
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 4; e += 2) {
      float x, y;
      pair(e, &x, &y);
      a = fmaf(x, x, a);
      b = fmaf(y, y, b);
    }
    return pair_sum(pair_sum(a + b, 16), 32);
  }
};

// one element as it lies in memory, and its value
template <class T>
struct Raw {
  static __device__ uint16_t bits(const T* p) { return gld(reinterpret_cast<const uint16_t*>(p)); }
  static __device__ float value(uint16_t b) {
    if constexpr (__is_same(T, Bf16)) return bf2f(b);
    else return h2f(b);
  }
};
template <>
struct Raw<float> {
  static __device__ float bits(const float* p) { return gld(p); }
  static __device__ float value(float b) { return b; }
};

// Keys and queries longer than 1e8, values from 1e20 on, states from 1e25 on, and gates that are NaN, make a chunk run token by
// token: the products above take keys before their norm, and 0 times what is not finite would reach earlier tokens.  Within
// these bounds a product of a key and a state stays below 1e8 sqrt(128) 1.5e25, a thousandth of f32's range over the 1e3 that a
// row behind the end multiplies it by.  (In such chunks a state's columns grow by 1e20 sqrt(tokens) at most, 5e24 in 2^31 of them.)
__device__ __forceinline__ bool in_range(float sum2) { return sum2 <= 1e16f; }
__device__ __forceinline__ bool value_in_range(float v) { return fabsf(v) < 1e20f; }
// (what is infinite or NaN in a state stays in its column either way)
__device__ __forceinline__ bool state_in_range(float s) { return !(fabsf(s) >= 1e25f && fabsf(s) < INFINITY); }

// ---- T and o's matrix of a chunk --------------------------------------------------------------------------------
// A workgroup per (chunk, value head); wave w forms o's row w (16 tokens) and A's row 3 - w, as many products for each.
// Both are formed transposed (rows: j, columns: i), which is the order in which the scan takes them.
// (I + A)^-1: the four 16 x 16 blocks on the diagonal by substitution, a column a lane; then row i from the right,
// T_ij = -(sum_(j < k <= i) T_ik A_kj) T_jj, in a wave's registers.  |k| <= 1 and b < 1 keep T's elements within products
// of contractions; a series in powers of A would not stay there.
// Bound by its chain of steps (three workgroups a CU overlap theirs) and by the 38 KB of operands that it leaves: 128 chunks
// of 32 heads in f32, 155 MB, 95 us; with bf16 keys, one product where f32 takes six, 8 chunks 11.2 us.  T and o's matrix
// as f32 would be two thirds of the bytes, but each of the scan's workgroups would take them apart in its chain, which was slower.
template <int D, class T>
__global__ void __launch_bounds__(256, 3) k_delta_prep(PromptArgs pa) {
  const DeltaArgs& a = pa.d;
  constexpr int NP = kParts<T>, KS = D / 32, AS = 68;
  constexpr int kBytesK = 4 * KS * NP * 1024, kBytesA = 64 * AS * 4, kBytesD = 4 * 16 * 20 * 4;
  // (49 KB for f32 keys of 128: three workgroups on a CU)
  __shared__ __align__(16) uint8_t s_mem[kBytesK > kBytesA + kBytesD ? kBytesK : kBytesA + kBytesD];
  __shared__ double s_g[64];
  __shared__ __align__(16) float s_beta[64], s_rk[64], s_rq[64];
  auto s_k = reinterpret_cast<u32x4_t(*)[KS][NP][64]>(s_mem);
  auto s_A = reinterpret_cast<float(*)[AS]>(s_mem);
  auto s_diag = reinterpret_cast<float(*)[16][20]>(s_mem + kBytesA);
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, G = lane >> 4, n = lane & 15;
  const uint32_t h = pa.head_of(blockIdx.x % a.NV), b = blockIdx.x / a.NV, kh = h / (a.NV / a.NK);
  const int row = a.r.row_of(b, kChunkShift, lane);
  uint32_t lo, hi;
  if (row < 0 || !pa.range(row, &lo, &hi)) return;
  const uint32_t t0 = lo + (b - a.r.first_block(row, lo, kChunkShift)) * kChunk;
  if (t0 >= hi) return;
  const uint32_t nt = min(hi - t0, uint32_t(kChunk)), mine = 16 * wave + n;
  float* out = pa.chunks + (size_t(b) * a.NV + h) * kChunkFloats;
  Row16<D, T> kr, qr;
  if (mine < nt) {
    kr.load(static_cast<const T*>(a.k) + (t0 + mine) * a.k_stride + kh * D, G);
    qr.load(static_cast<const T*>(a.q) + (t0 + mine) * a.q_stride + kh * D, G);
  } else {
    kr.clear();
    qr.clear();
  }
  float ld = 0.0f, beta = 0.0f;
  bool fine = true;
  if (wave == 0 && uint32_t(lane) < nt) {
    ld = delta_log_decay(gld(a.A_log + h), gld(a.a + (t0 + lane) * a.a_stride + h) + gld(a.dt_bias + h));
    beta = delta_beta(gld(a.b + (t0 + lane) * a.b_stride + h));
    fine = ld == ld && beta == beta;
    ld = ld < -200.0f ? -200.0f : ld;  // e^-200 is 0 in f32; differences of sums stay numbers
  }
  const float k2 = kr.sum2(), q2 = qr.sum2();
  const float rk = 1.0f / sqrtf(k2 + 1e-6f), rq = 1.0f / sqrtf(q2 + 1e-6f) * (1.0f / sqrtf(float(D)));
  if (G == 0) {
    s_rk[mine] = in_range(k2) ? rk : -1.0f;  // (told below)
    s_rq[mine] = in_range(q2) ? rq : -1.0f;
  }
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    u32x4_t f[NP];
    kr.operand(s, f);
#pragma unroll
    for (int p = 0; p < NP; ++p) s_k[wave][s][p][lane] = f[p];
  }
  if (wave == 0) {
    // sums in 64 bits: their differences are what counts, and in 32 bits 1e3 - 1e3 leaves 6e-5
    double g = double(ld);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double p = __shfl_up(g, o);
      g += lane >= o ? p : 0.0;
    }
    s_g[lane] = g;
    s_beta[lane] = beta;
  }
  __syncthreads();
  if (wave == 0) {
    const double g = s_g[lane], end = s_g[63];
    const float k = s_rk[lane], q = s_rq[lane];
    fine = fine && k >= 0.0f && q >= 0.0f;
    const bool all = __ballot(!fine) == 0;
    float* sc = out + kOffScale;
    sc[lane] = expf(float(g)) * k;
    sc[64 + lane] = expf(float(g)) * q;
    sc[128 + lane] = expf(float(end - g)) * k;
    if (lane == 0) {
      sc[192] = expf(float(end));
      sc[193] = all ? 1.0f : 0.0f;
    }
  }
  // row `wave` of a matrix, as the scan's operands
  auto leave = [&](float* dst, const f4_t (&v)[4]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > wave >> 1) break;
      u32x4_t f[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t p[3];
        split2(v[2 * s + e / 2][e % 2 * 2], v[2 * s + e / 2][e % 2 * 2 + 1], p);
#pragma unroll
        for (int i = 0; i < 3; ++i) f[i][e] = p[i];
      }
#pragma unroll
      for (int i = 0; i < 3; ++i)
        *reinterpret_cast<u32x4_t*>(dst + (frag_of(wave) + s) * kFrag + (i * 64 + lane) * 4) = f[i];
    }
  };
  // tiles (j, i) transposed: lane (G, n) gets tokens j = 16 jt + 4 G + r of i = 16 it + n
  f4_t At[4];
  const int R = 3 - wave;
  auto weight = [&](int it, int jt, f4_t v, bool below, float fi) {
    const int i = 16 * it + n;
    const double gi = s_g[i];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = 16 * jt + 4 * G + r;
      v[r] = j < i || (j == i && !below) ? v[r] * (fi * s_rk[j]) * expf(float(gi - s_g[j])) : 0.0f;
    }
    return v;
  };
  {
    u32x4_t qf[KS][NP];
#pragma unroll
    for (int s = 0; s < KS; ++s) qr.operand(s, qf[s]);
    f4_t o[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      f4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (jt <= wave) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          u32x4_t f[NP];
          ld_parts(s_k[jt][s], lane, f);
          v = mma(f, qf[s], v);
        }
        v = weight(wave, jt, v, false, s_rq[16 * wave + n]);
      }
      o[jt] = v;
    }
    leave(out + kOffO, o);
  }
  {
    u32x4_t kf[KS][NP];
#pragma unroll
    for (int s = 0; s < KS; ++s)
      ld_parts(s_k[R][s], lane, kf[s]);
    const float fi = s_beta[16 * R + n] * s_rk[16 * R + n];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      if (jt > R) break;
      f4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        u32x4_t f[NP];
        ld_parts(s_k[jt][s], lane, f);
        v = mma(f, kf[s], v);
      }
      At[jt] = weight(R, jt, v, true, fi);
    }
  }
  __syncthreads();  // (the keys have been read: A takes their place)
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
    if (jt <= R) *reinterpret_cast<f4_t*>(&s_A[16 * R + n][16 * jt + 4 * G]) = At[jt];
  __syncthreads();
  {
    float t[16];  // column n of T_ww; what a row has taken off the others first, so that few sums wait for each other
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = i == n ? 1.0f : 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j += 4)
#pragma unroll
      for (int i = j + 1; i < 16; ++i) {
        const f4_t x = *reinterpret_cast<const f4_t*>(&s_A[16 * wave + i][16 * wave + j]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < i) t[i] = fmaf(-x[e], t[j + e], t[i]);
      }
    if (G == 0) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(&s_diag[wave][n][i]) = make_float4(t[i], t[i + 1], t[i + 2], t[i + 3]);
    }
  }
  __syncthreads();
  f4_t Tt[4];  // T_wj transposed: lane (G, n) has row n, columns 4 G + r
#pragma unroll
  for (int j = 3; j >= 0; --j) {
    if (j > wave) {
      Tt[j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    } else if (j == wave) {
#pragma unroll
      for (int r = 0; r < 4; ++r) Tt[j][r] = s_diag[j][4 * G + r][n];
    } else {
      f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 3; k > j; --k) {
        if (k > wave) continue;
        f4_t x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = s_A[16 * k + 4 * G + r][16 * j + n];
        acc = mma16(x, Tt[k], acc);
      }
      const f4_t d = -*reinterpret_cast<const f4_t*>(&s_diag[j][n][4 * G]);
      Tt[j] = mma16(d, acc, f4_t{0.0f, 0.0f, 0.0f, 0.0f});
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) Tt[j] *= *reinterpret_cast<const f4_t*>(&s_beta[16 * j + 4 * G]);
  leave(out, Tt);
}

// ---- the state over a row's chunks --------------------------------------------------------------------------------
// A workgroup takes 16 NT columns of a value head's state over all chunks of a row.  A chunk is three steps with a
// barrier behind each, what one leaves to the others in LDS as operands.  Four waves carry the state, each with 16 tokens
// of a chunk and D / 4 rows of S: 1. v - e^g (K S) of their tokens, 2. u of their tokens, 3. their rows of S.  Four others
// form the outputs of 16 tokens each: Q S in 2., o in 3.  Everybody loads its own operands of the next chunk where the
// others leave it time.  (Rows behind the end are the last token again: b, and so u, is 0 there.)
// Keys as operands of k u^T have tokens inside: the transposing reads of LDS give them so.
// Bound, for few rows, by the chain of a chunk's three steps, each a wait on LDS, a run of dependent products and a barrier: 3.6 us a
// chunk of f32 keys (8189 tokens of 32 heads on 256 workgroups, 460 us; with four waves for everything 6.5),
// 2.7 of bf16; with 64 columns of bf16, where a CU's LDS holds one workgroup, 5.2 (24 prompts of 49 thousand tokens
// together, 192 such chunks a CU: 1.0 ms, 0.6 PFLOP/s of parts' products).
template <int D, class T, int NT>
__global__ void __launch_bounds__(512, D == 64 ? 4 : 2) k_delta_scan(PromptArgs pa) {
  const DeltaArgs& a = pa.d;
  constexpr int NP = kParts<T>, KS = D / 32, RT = D / 64, CB = D / (16 * NT);
  constexpr int KR = D / 8 + 2;  // a token's keys in LDS, with room so that neither side's accesses meet in a few banks
  __shared__ u32x4_t s_k[NP][kChunk][KR];
  __shared__ u32x4_t s_s[KS][NT][3][64];
  __shared__ u32x4_t s_x[NT][2][3][64], s_u[NT][2][3][64], s_us[NT][2][3][64];
  __shared__ __align__(16) float s_scale[2][256];
  __shared__ float s_red[2][4], s_col[2][4][16 * NT];
  __shared__ __align__(16) uint32_t s_bad[2][4];  // of each wave that carries the state
  const int wave8 = uniform(threadIdx.x >> 6), wave = wave8 & 3, lane = threadIdx.x & 63, G = lane >> 4, n = lane & 15;
  const bool carry = wave8 < 4;  // (uniform)
  // the column blocks of a head on one XCD (workgroup i runs on XCD i % 8), whose L2 they share
  const uint32_t item = blockIdx.x / (8 * CB) * 8 + blockIdx.x % 8, c0 = blockIdx.x / 8 % CB * (16 * NT);
  if (item >= a.r.rows * a.NV) return;
  const int nth = gridDim.x > 256 ? pa.nth_longest(item / a.NV, lane) : int(item / a.NV);
  uint32_t lo, hi;
  float fill;
  if (nth < 0 || !pa.range(uint32_t(nth), &lo, &hi)) return;
  const uint32_t row = uniform(uint32_t(nth)), h = pa.head_of(item % a.NV), kh = h / (a.NV / a.NK);
  const int slot = a.r.before(row, &fill), to = a.r.after(row);
  // the wave's rows of the state: those of its two (D = 64: of its one) operands' elements
  auto dim = [&](int r, int u) { return RT == 2 ? Row16<D, T>::dim(G, wave, u, r) : Row16<D, T>::dim(G, wave >> 1, wave & 1, r); };
  f4_t S[RT][NT];
  if (carry) {
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
      for (int ct = 0; ct < NT; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          S[u][ct][r] = slot >= 0 ? gld(a.state + uint64_t(slot) * a.slot_stride + (size_t(h) * D + dim(r, u)) * D + c0 + 16 * ct + n) : fill;
  }
  auto is_bad = [&](int turn) {
    const uint4 b = *reinterpret_cast<const uint4*>(s_bad[turn]);
    return (b.x | b.y | b.z | b.w) != 0;
  };
  // has chunk `turn` run token by token if S is out of range
  auto look_at_s = [&](int turn) {
    bool large = false;
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
      for (int ct = 0; ct < NT; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) large |= !state_in_range(S[u][ct][r]);
    if (__ballot(large) != 0 && lane == 0) s_bad[turn][wave] = 1;
  };
  // leaves S as operands
  auto leave_s = [&] {
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      uint32_t p[2 * RT][3];
#pragma unroll
      for (int e = 0; e < 2 * RT; ++e) split2(S[e / 2][ct][e % 2 * 2], S[e / 2][ct][e % 2 * 2 + 1], p[e]);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        if constexpr (RT == 2) s_s[wave][ct][i][lane] = u32x4_t{p[0][i], p[1][i], p[2][i], p[3][i]};
        else reinterpret_cast<u32x2_t*>(&s_s[wave >> 1][ct][i][lane])[wave & 1] = u32x2_t{p[0][i], p[1][i]};
      }
    }
  };
  // leaves 16 tokens of one column tile as half of an operand with tokens inside
  auto leave_u = [&](u32x4_t (&dst)[2][3][64], f4_t v) {
    uint32_t p[2][3];
    split2(v[0], v[1], p[0]);
    split2(v[2], v[3], p[1]);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      reinterpret_cast<u32x2_t*>(&dst[wave >> 1][i][lane])[wave & 1] = u32x2_t{p[0][i], p[1][i]};
  };
  using Bits = __typeof__(Raw<T>::bits(nullptr));
  const int ns = (wave >> 1) + 1;  // products of 32 tokens in the wave's row of a matrix
  const uint32_t first = a.r.first_block(row, lo, kChunkShift);
  const T* v_at = static_cast<const T*>(a.v) + h * D + c0 + n;
  auto chunk_at = [&](uint32_t t0) { return pa.chunks + (size_t(first + ((t0 - lo) >> kChunkShift)) * a.NV + h) * kChunkFloats; };
  // the values of the tokens of a wave that carries S
  Bits v16[NT][4];  // (as they lie there: widened here, they would be waited for at once)
  auto load_v = [&](uint32_t t0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const T* p = v_at + min(t0 + 16 * wave + 4 * G + r, hi - 1) * a.v_stride;
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) v16[ct][r] = Raw<T>::bits(p + 16 * ct);
    }
  };
  // 16 tokens' keys or queries, the wave's row of a chunk's matrix
  auto load_x = [&](Row16<D, T>& x, const void* p, uint64_t stride, uint32_t t0) {
    x.load(static_cast<const T*>(p) + min(t0 + 16 * wave + n, hi - 1) * stride + kh * D, G);
  };
  auto load_m = [&](u32x4_t (&m)[2][3], uint32_t t0, int at) {
    const float* p = chunk_at(t0) + at + frag_of(wave) * kFrag + lane * 4;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= ns) break;
#pragma unroll
      for (int i = 0; i < 3; ++i) m[s][i] = gld(reinterpret_cast<const u32x4_t*>(p + s * kFrag + i * 256));
    }
  };
  auto put = [&](uint32_t t, int ct, float v) {
    const size_t at = size_t(h) * D + c0 + 16 * ct + n;
    if (pa.o32) pa.o32[size_t(t) * a.NV * D + at] = v;
    else static_cast<T*>(a.out)[t * a.out_stride + at] = Elem<T>::put(v);
  };
  auto put4 = [&](uint32_t t, int ct, f4_t v) {  // columns 4 G ..
    const size_t at = size_t(h) * D + c0 + 16 * ct + 4 * G;
    const float x[4] = {v.x, v.y, v.z, v.w};
    if (pa.o32) *reinterpret_cast<f4_t*>(pa.o32 + size_t(t) * a.NV * D + at) = v;
    else st_row(static_cast<T*>(a.out) + t * a.out_stride + at, x);
  };
  // the recurrence itself, token by token (inputs that are not finite: see in_range), by the waves that carry S: three barriers a token
  auto tokens = [&](uint32_t t0, uint32_t t1) {
    const float A_log = gld(a.A_log + h), dt = gld(a.dt_bias + h);
    for (uint32_t t = t0; t < t1; ++t) {
      float k[RT][4], q[RT][4], k2 = 0.0f, q2 = 0.0f, p[NT], o[NT];
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const size_t d = kh * D + dim(r, u);
          k[u][r] = Elem<T>::get(static_cast<const T*>(a.k) + t * a.k_stride + d);
          q[u][r] = Elem<T>::get(static_cast<const T*>(a.q) + t * a.q_stride + d);
          k2 = fmaf(k[u][r], k[u][r], k2);
          q2 = fmaf(q[u][r], q[u][r], q2);
        }
      k2 = pair_sum(pair_sum(k2, 16), 32);
      q2 = pair_sum(pair_sum(q2, 16), 32);
      if (lane == 0) {
        s_red[0][wave] = k2;
        s_red[1][wave] = q2;
      }
      lds_barrier();
      k2 = (s_red[0][0] + s_red[0][1]) + (s_red[0][2] + s_red[0][3]);
      q2 = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
      const float ki = 1.0f / sqrtf(k2 + 1e-6f), qi = 1.0f / sqrtf(q2 + 1e-6f) * (1.0f / sqrtf(float(D)));
      const float decay = expf(delta_log_decay(A_log, gld(a.a + t * a.a_stride + h) + dt));
      const float beta = delta_beta(gld(a.b + t * a.b_stride + h));
      auto total = [&](float (&p)[NT], int buf) {
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
          p[ct] = pair_sum(pair_sum(p[ct], 16), 32);
          if (G == 0) s_col[buf][wave][16 * ct + n] = p[ct];
        }
        lds_barrier();
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
          const int c = 16 * ct + n;
          p[ct] = (s_col[buf][0][c] + s_col[buf][1][c]) + (s_col[buf][2][c] + s_col[buf][3][c]);
        }
      };
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        p[ct] = o[ct] = 0.0f;
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            S[u][ct][r] *= decay;
            p[ct] = fmaf(S[u][ct][r], k[u][r] * ki, p[ct]);
          }
      }
      total(p, 0);
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const float x = (Elem<T>::get(v_at + t * a.v_stride + 16 * ct) - p[ct]) * beta;
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            S[u][ct][r] = fmaf(k[u][r] * ki, x, S[u][ct][r]);
            o[ct] = fmaf(S[u][ct][r], q[u][r] * qi, o[ct]);
          }
      }
      total(o, 1);
      if (wave == 0 && G == 0) {
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) put(t, ct, o[ct]);
      }
    }
  };

  // X S of the wave's tokens: lane (G, n) gets tokens 4 G + r of column n, or (the operands the other way round) columns
  // 4 G + r of token n, so that outputs are stored 4 at a time
  auto times_s = [&](const u32x4_t (&x)[KS][NP], f4_t (&y)[NT], auto turned) {
    constexpr int N = KS * NT, AHEAD = 2;  // (operands are read two products ahead: LDS answers in some 100 cycles)
    u32x4_t f[AHEAD + 1][3];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ld_parts(s_s[i % KS][i / KS], lane, f[i]);
    f4_t sum[2];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + AHEAD < N) ld_parts(s_s[(i + AHEAD) % KS][(i + AHEAD) / KS], lane, f[(i + AHEAD) % (AHEAD + 1)]);
      __builtin_amdgcn_sched_barrier(0);
      const int s = i % KS;
      if (s == 0) sum[0] = sum[1] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};  // (two chains of products)
      const auto& g = f[i % (AHEAD + 1)];
      sum[s & 1] = turned ? mma(g, x[s], sum[s & 1]) : mma(x[s], g, sum[s & 1]);
      if (s == KS - 1) y[i / KS] = sum[0] + sum[1];
    }
  };
  // M x of the wave's row of a matrix, the same ways
  auto times_x = [&](const u32x4_t (&m)[2][3], const u32x4_t (&x)[2][3][64], f4_t y, auto turned) {
    f4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    u32x4_t f[3];
    ld_parts(x[0], lane, f);
    y = turned ? mma(f, m[0], y) : mma(m[0], f, y);
    if (ns > 1) {
      ld_parts(x[1], lane, f);
      sum = turned ? mma(f, m[1], sum) : mma(m[1], f, sum);
    }
    return y + sum;
  };
  Row16<D, T> x16;
  u32x4_t m16[2][3];
  int turn = 0;
  if (!carry) {
    f4_t f16;
    auto load_scale = [&](uint32_t t0) {
      if (wave == 0) f16 = gld(reinterpret_cast<const f4_t*>(chunk_at(t0) + kOffScale + lane * 4));
    };
    auto leave_scale = [&](int turn) {
      if (wave == 0) *reinterpret_cast<f4_t*>(&s_scale[turn][lane * 4]) = f16;
    };
    u32x4_t xf[KS][NP];
    auto take_x = [&] {
#pragma unroll
      for (int s = 0; s < KS; ++s) x16.operand(s, xf[s]);
    };
    f4_t y[NT], done[NT];
    uint32_t from = hi;  // tokens of `done`
    auto store = [&] {
      const uint32_t t = from + 16 * wave + n;
      if (t >= hi) return;
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) put4(t, ct, done[ct]);
    };
    if (lo < hi) {
      load_scale(lo);
      load_x(x16, a.q, a.q_stride, lo);
      load_m(m16, lo, kOffO);
      leave_scale(0);
    }
    lds_barrier();
    for (uint32_t t0 = lo; t0 < hi; t0 += kChunk, turn ^= 1) {
      const uint32_t next = t0 + kChunk < hi ? t0 + kChunk : t0;  // (behind the last chunk: that one again, not used)
      take_x();
      load_x(x16, a.q, a.q_stride, next);
      load_scale(next);
      store();
      lds_barrier();
      const float g = s_scale[turn][64 + 16 * wave + n];
      if (is_bad(turn)) {  // (the same for all)
        for (uint32_t i = 3 * min(hi - t0, uint32_t(kChunk)); i != 0; --i) lds_barrier();
        from = hi;
      } else {
        times_s(xf, y, std::true_type{});
        lds_barrier();
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) done[ct] = times_x(m16, s_u[ct], y[ct] * g, std::true_type{});
        from = t0;
      }
      load_m(m16, next, kOffO);
      leave_scale(turn ^ 1);
      lds_barrier();
    }
    store();
    return;
  }

  if (lo < hi) {
    load_x(x16, a.k, a.k_stride, lo);
    load_v(lo);
    load_m(m16, lo, 0);
  }
  if (lane < 2) s_bad[lane][wave] = 0;
  look_at_s(0);
  leave_s();
  lds_barrier();
  for (uint32_t t0 = lo; t0 < hi; t0 += kChunk, turn ^= 1) {
    const uint32_t next = t0 + kChunk < hi ? t0 + kChunk : t0;
    // 1.
    f4_t v[NT], y[NT];
    u32x4_t xf[KS][NP];
    bool bad = s_scale[turn][193] != 1.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      x16.operand(s, xf[s]);
#pragma unroll
      for (int p = 0; p < NP; ++p) s_k[p][16 * wave + n][4 * s + G] = xf[s][p];
    }
#pragma unroll
    for (int ct = 0; ct < NT; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[ct][r] = Raw<T>::value(v16[ct][r]);
        bad |= !value_in_range(v[ct][r]);
      }
    if (__ballot(bad) != 0 && lane == 0) s_bad[turn][wave] = 1;
    times_s(xf, y, std::false_type{});
    const float* scale = s_scale[turn] + 16 * wave + 4 * G;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) leave_u(s_x[ct], v[ct] - *reinterpret_cast<const f4_t*>(scale) * y[ct]);
    lds_barrier();
    if (is_bad(turn)) {  // (the same for all)
      tokens(t0, min(hi, t0 + kChunk));
      look_at_s(turn ^ 1);
      leave_s();
      load_x(x16, a.k, a.k_stride, next);
      load_v(next);
      load_m(m16, next, 0);
      lds_barrier();
      if (lane == 0) s_bad[turn][wave] = 0;
      continue;
    }
    // 2.
    f4_t u[NT];
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) u[ct] = times_x(m16, s_x[ct], f4_t{0.0f, 0.0f, 0.0f, 0.0f}, std::false_type{});
    load_x(x16, a.k, a.k_stride, next);
    load_v(next);
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      leave_u(s_u[ct], u[ct]);
      leave_u(s_us[ct], u[ct] * *reinterpret_cast<const f4_t*>(scale + 128));
    }
    const float end = s_scale[turn][192];
    lds_barrier();
    // 3.
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4_t kt[RT][NP];
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          // lane n of a group of 16 names 4 keys of token n / 4 and gets key n of the four tokens
          const int at = 4 * (RT == 2 ? wave : wave >> 1) + n % 4, half = RT == 2 ? u : wave & 1;
          const u32x2_t lo4 = ld_transposed(reinterpret_cast<const u32x2_t*>(&s_k[p][32 * s + 4 * G + n / 4][at]) + half);
          const u32x2_t hi4 = ld_transposed(reinterpret_cast<const u32x2_t*>(&s_k[p][32 * s + 16 + 4 * G + n / 4][at]) + half);
          kt[u][p] = u32x4_t{lo4.x, lo4.y, hi4.x, hi4.y};
        }
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        u32x4_t f[3];
        ld_parts(s_us[ct][s], lane, f);
#pragma unroll
        for (int u = 0; u < RT; ++u) S[u][ct] = mma(kt[u], f, s == 0 ? S[u][ct] * end : S[u][ct]);
      }
    }
    load_m(m16, next, 0);
    leave_s();
    lds_barrier();
  }
  if (to < 0) return;
#pragma unroll
  for (int u = 0; u < RT; ++u)
#pragma unroll
    for (int ct = 0; ct < NT; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        st_once(a.state + uint64_t(to) * a.slot_stride + (size_t(h) * D + dim(r, u)) * D + c0 + 16 * ct + n, S[u][ct][r]);
}

// ---- the gated norm: w * o / rms(o) * silu(z), a workgroup per 16 tokens of a (chunk, value head), 4 dims a lane.  Its f32
// outputs come from the scan's stores, of few tokens mostly out of the caches (501 tokens of 32 heads of 128, 16 MB: 5.1 us, a
// launch's time; 49 thousand, 1.6 GB: 279 us, 5.8 TB/s) -----------------------------------------------------------------------------
constexpr int kNormTokens = 16;
template <int D, class T>
__global__ void __launch_bounds__(256) k_delta_gnorm(PromptArgs pa) {
  const DeltaArgs& a = pa.d;
  constexpr int LPR = D / 4, RG = 256 / LPR, PARTS = kChunk / kNormTokens;
  const int c = threadIdx.x % LPR * 4;
  const uint32_t part = blockIdx.x % PARTS, h = blockIdx.x / PARTS % a.NV, b = blockIdx.x / (PARTS * a.NV);
  const int row = a.r.row_of(b, kChunkShift, threadIdx.x & 63);
  uint32_t lo, hi;
  if (row < 0 || !pa.range(row, &lo, &hi)) return;
  const uint32_t t0 = lo + (b - a.r.first_block(row, lo, kChunkShift)) * kChunk + part * kNormTokens;
  if (t0 >= hi) return;
  float w[4], o[kNormTokens / RG][4], z[kNormTokens / RG][4];
  ld_row(a.norm_w + c, w);
#pragma unroll
  for (int i = 0; i < kNormTokens / RG; ++i) {  // (behind the row's end: its last token again)
    const size_t t = min(t0 + i * RG + threadIdx.x / LPR, hi - 1);
    ld_row(pa.o32 + (t * a.NV + h) * D + c, o[i]);
    ld_row(static_cast<const T*>(a.z) + t * a.z_stride + h * D + c, z[i]);
  }
#pragma unroll
  for (int i = 0; i < kNormTokens / RG; ++i) {
    const uint32_t t = t0 + i * RG + threadIdx.x / LPR;
    float s2 = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s2 = fmaf(o[i][e], o[i][e], s2);
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) s2 = pair_sum(s2, m);
    const float rr = 1.0f / sqrtf(s2 / float(D) + a.eps);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = w[e] * (o[i][e] * rr) * delta_silu(z[i][e]);
    if (t < hi) st_row(static_cast<T*>(a.out) + t * a.out_stride + h * D + c, o[i]);
  }
}

// ---- host -----------------------------------------------------------------------------------------------------
struct PromptPlan {
  bool ok = false;
  uint64_t chunks = 0;  // (chunk, value head) pairs
  size_t off_o = 0, bytes = 0;
};
PromptPlan prompt_plan(const chpe_delta_states* s, uint32_t tokens, uint32_t rows, bool norm) {
  PromptPlan p;
  const uint64_t blocks = (uint64_t(tokens) >> kChunkShift) + rows, vw = uint64_t(s->v_heads) * s->head_dim;
  if (tokens > kMaxTokens || rows > kMaxTokens || blocks * s->v_heads > kMaxItems / 1024) return p;  // (the norm's launch)
  p.chunks = blocks * s->v_heads;
  if ((uint64_t(rows) * s->v_heads + 7) / 8 * 8 * (s->head_dim / 16) > kMaxItems / 512) return p;
  p.off_o = p.chunks * kChunkFloats * 4;
  p.bytes = p.off_o + (norm ? tokens * vw * 4 : 0);
  p.ok = true;
  return p;
}

// Rows of up to this many tokens run token by token, each state read and written once for all of them, and no launch
// knows the rows' lengths: where there are several rows both kinds are launched and leave the other's rows alone.
// A token costs the one kind some 2 us beside the states' bytes, a chunk is the same work for the other however few tokens
// it has (9B layout, f32 / bf16, us: one row in chunks 24 / 21, of 8 tokens token by token 23 / 23, of 16 38 / 40; 8 rows 55 / 41
// in chunks, of 16 tokens 48 / 50; 16 rows 88 / 63, of 16 62 / 61, of 24 86 / 85; 32 rows 150 / 105, of 8 68 / 65; 64 rows
// 297 / 201, of 16 180 / 184).
uint32_t short_rows(uint32_t rows, uint32_t v_heads) { return uint64_t(rows) * v_heads >= 512 ? 16 : 8; }

template <int D, class T>
bool launch_prompt(const PromptArgs& a, const PromptPlan& p, hipStream_t st) {
  const uint64_t items = (uint64_t(a.d.r.rows) * a.d.NV + 7) / 8 * 8;
  if (a.d.r.tokens != 0 && !launch(&k_delta_prep<D, T>, p.chunks, 256, st, a)) return false;
  // Columns of a workgroup: 16, so that few rows reach all CUs; where head dim 128 gives more workgroups than those, 32 (one
  // row of 1000 tokens of the 9B layout in f32 79 us with 16, 91 with 32; four rows 279 and 207; bf16 49 / 61 and
  // 160 / 128; at head dim 64 16 is ahead or within 11 % throughout), and 64 for many bf16 rows, where LDS holds
  // that (8 rows 247 us with 32, 233 with 64; 6 rows 182 and 210).
  const uint64_t many = uint64_t(a.d.r.rows) * a.d.NV;
  bool ok;
  if constexpr (D == 128 && __is_same(T, Bf16)) {
    ok = many * 2 >= 512  ? launch(&k_delta_scan<D, T, 4>, items * 2, 512, st, a)
         : many * 8 > 256 ? launch(&k_delta_scan<D, T, 2>, items * 4, 512, st, a)
                          : launch(&k_delta_scan<D, T, 1>, items * 8, 512, st, a);
  } else if constexpr (D == 128) {
    ok = many * 8 > 256 ? launch(&k_delta_scan<D, T, 2>, items * 4, 512, st, a)
                        : launch(&k_delta_scan<D, T, 1>, items * 8, 512, st, a);
  } else {
    ok = launch(&k_delta_scan<D, T, 1>, items * 4, 512, st, a);
  }
  if (!ok) return false;
  return !a.o32 || a.d.r.tokens == 0 || launch(&k_delta_gnorm<D, T>, p.chunks * (kChunk / kNormTokens), 256, st, a);
}
template <int D>
bool launch_prompt(const PromptArgs& a, const PromptPlan& p, int type, hipStream_t st) {
  return type == 0   ? launch_prompt<D, float>(a, p, st)
         : type == 1 ? launch_prompt<D, _Float16>(a, p, st)
                     : launch_prompt<D, Bf16>(a, p, st);
}

}  // namespace
}  // namespace chpe

using namespace chpe;

extern "C" size_t chpe_delta_prompt_workspace(const chpe_delta_states* states, uint32_t tokens, uint32_t rows, int norm) {
  if (!delta_states_ok(states)) return 0;
  const PromptPlan p = prompt_plan(states, tokens, rows, norm != 0);
  return p.ok ? p.bytes : 0;
}

extern "C" int chpe_delta_prompt(const chpe_delta_states* states, const chpe_delta_tokens* t, uint32_t tokens,
                                 uint32_t rows, const int32_t* starts, const int32_t* slot_in, const int32_t* slot_out,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  PromptArgs a{};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!delta_from(states, t, tokens, rows, starts, slot_in, slot_out, &a.d) || !stream_here(st)) return -1;
  if (rows == 0) return 0;
  const PromptPlan p = prompt_plan(states, tokens, rows, t->z != nullptr);
  if (!p.ok || !starts || !workspace || !aligned16(workspace)) return -1;
  if (workspace_bytes < p.bytes) return -2;
  a.chunks = static_cast<float*>(workspace);
  a.o32 = t->z ? a.chunks + p.off_o / 4 : nullptr;
  const uint32_t few = short_rows(rows, states->v_heads);
  const bool some_short = rows > 1 || tokens <= few, some_long = tokens > few;
  a.shortest = some_short ? few + 1 : 0;
  if (some_short && !launch_delta_tokens(a.d, states->head_dim, t->type, few, st)) return -3;
  if (!some_long) return 0;
  return (states->head_dim == 128 ? launch_prompt<128>(a, p, t->type, st) : launch_prompt<64>(a, p, t->type, st)) ? 0 : -3;
}
