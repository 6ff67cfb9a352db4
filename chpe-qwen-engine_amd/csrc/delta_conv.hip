// delta_conv.hip -- chpe_delta_conv: the causal depthwise convolution in front of the gated delta rule, with SiLU:
// y_t = silu(sum_j w_j x_(t - taps + 1 + j)) per channel, over the tokens of many rows; what came before a row's
// first token is its state, the taps - 1 last inputs, which is left anew.
#include "delta.hpp"

namespace chpe {
namespace {
using namespace dev;

constexpr int kConvShift = 3, kConvTokens = 1 << kConvShift;  // tokens of a workgroup: at least taps - 1
static_assert(kConvTokens >= int(kDnMaxTaps) - 1, "");
constexpr int kConvThreads = 64;

struct ConvArgs {
  DeltaRows r;
  float* state;            // [slot][channels][taps - 1], oldest first
  const void* x;
  const float* w;          // [channels][taps]
  void* y;
  uint64_t slot_stride, x_stride, y_stride;
  uint32_t channels, parts;  // parts: workgroups of a block of tokens
};

// A wave takes 64 x 16 bytes of channels (V of them a lane) of a block of 8 tokens of one row; the taps slide through
// registers.  A row's first block reads the state before and writes the one after (whose inputs are x and the state
// before), so that both may be the same slot.
// Bound by memory: every input is read once, and by the next block's taps (8196 bf16 tokens of 8192 channels, 316 MB so:
// 53 us, 6.0 TB/s, on inputs that change from call to call 58; with 16 tokens 54, with 32 and a slower SiLU 90 instead of 78).
template <class T, int TAPS>
__global__ void __launch_bounds__(kConvThreads) k_delta_conv(ConvArgs a) {
  constexpr int V = 16 / sizeof(T), P = TAPS - 1;
  const int lane = threadIdx.x;
  const uint32_t part = blockIdx.x % a.parts, b = blockIdx.x / a.parts;
  int row = int(b);
  uint32_t lo, hi, i = 0;
  if (a.r.starts) {
    row = a.r.row_of(b, kConvShift, lane);
    if (row < 0) return;
  }
  if (!a.r.range(row, &lo, &hi)) return;
  if (a.r.starts) i = b - a.r.first_block(row, lo, kConvShift);
  const uint32_t t0 = lo + i * kConvTokens, c = (part * kConvThreads + lane) * V;
  if ((i != 0 && t0 >= hi) || c >= a.channels) return;
  const T* x = static_cast<const T*>(a.x) + c;
  float tap[P][V];  // the inputs before token t, oldest first
  if (i == 0) {
    float fill, old[V * P];
    const int slot = a.r.before(row, &fill), to = a.r.after(row);
    if (slot >= 0) {
      ld_row(a.state + uint64_t(slot) * a.slot_stride + size_t(c) * P, old);
    } else {
#pragma unroll
      for (int e = 0; e < V * P; ++e) old[e] = fill;
    }
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) tap[p][e] = old[e * P + p];
    if (to >= 0) {
      const uint32_t n = hi - lo;
      float now[V * P];
#pragma unroll
      for (int p = 0; p < P; ++p) {  // input n - P + p of the row, or n + p of the state before
        float in[V];
        if (n + p >= uint32_t(P)) {
          ld_row(x + size_t(lo + (n + p - P)) * a.x_stride, in);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            in[e] = 0.0f;
#pragma unroll
            for (int o = 0; o < P; ++o)
              if (uint32_t(o) == n + p) in[e] = tap[o][e];
          }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) now[e * P + p] = in[e];
      }
      st_row(a.state + uint64_t(to) * a.slot_stride + size_t(c) * P, now);
    }
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) ld_row(x + size_t(t0 - P + p) * a.x_stride, tap[p]);
  }
  if (t0 >= hi) return;
  float w[V * TAPS];
  ld_row(a.w + size_t(c) * TAPS, w);
  T* y = static_cast<T*>(a.y) + c;
  const uint32_t n = min(hi - t0, uint32_t(kConvTokens));
#pragma unroll 4
  for (uint32_t k = 0; k < n; ++k) {
    float in[V], out[V];
    ld_row(x + size_t(t0 + k) * a.x_stride, in);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float s = 0.0f;  // oldest first
#pragma unroll
      for (int p = 0; p < P; ++p) s = fmaf(w[e * TAPS + p], tap[p][e], s);
      s = fmaf(w[e * TAPS + P], in[e], s);
      out[e] = delta_silu(s);
#pragma unroll
      for (int p = 0; p + 1 < P; ++p) tap[p][e] = tap[p + 1][e];
      tap[P - 1][e] = in[e];
    }
    st_row(y + size_t(t0 + k) * a.y_stride, out);
  }
}

template <int TAPS>
bool launch_conv(const ConvArgs& a, int type, uint64_t blocks, hipStream_t st) {
  return type == 0   ? launch(&k_delta_conv<float, TAPS>, blocks, kConvThreads, st, a)
         : type == 1 ? launch(&k_delta_conv<_Float16, TAPS>, blocks, kConvThreads, st, a)
                     : launch(&k_delta_conv<Bf16, TAPS>, blocks, kConvThreads, st, a);
}

}  // namespace
}  // namespace chpe

using namespace chpe;

extern "C" int chpe_delta_conv(float* conv_state, uint64_t slot_stride, uint32_t n_slots, uint32_t channels,
                               uint32_t taps, const float* w, int type, const void* x, uint64_t x_stride, void* y,
                               uint64_t y_stride, uint32_t tokens, uint32_t rows, const int32_t* starts,
                               const int32_t* slot_in, const int32_t* slot_out, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (taps < 2 || taps > kDnMaxTaps || channels == 0 || channels % 8 != 0 || channels > kMaxTokens) return -1;
  if (type < 0 || type > 2 || n_slots == 0 || n_slots > kMaxTokens || !w || !aligned16(w)) return -1;
  if (!rows_ok(conv_state, slot_stride, uint64_t(channels) * (taps - 1), n_slots, 0) || !stream_here(st)) return -1;
  if (!delta_rows_ok(tokens, rows, slot_in, slot_out) || (!starts && tokens != rows)) return -1;
  if (tokens != 0 && (!rows_ok(x, x_stride, channels, tokens, type) || !rows_ok(y, y_stride, channels, tokens, type)))
    return -1;
  if (rows == 0) return 0;
  const uint32_t wide = kConvThreads * (type == 0 ? 4 : 8);
  ConvArgs a{{starts, slot_in, slot_out, tokens, rows, n_slots}, conv_state, x, w, y, n_slots > 1 ? slot_stride : 0,
             x_stride, y_stride, channels, (channels + wide - 1) / wide};
  const uint64_t blocks = (starts ? uint64_t(tokens >> kConvShift) + rows : rows) * a.parts;
  if (blocks > kMaxItems / kConvThreads) return -1;
  bool ok = false;
  switch (taps) {
    case 2: ok = launch_conv<2>(a, type, blocks, st); break;
    case 3: ok = launch_conv<3>(a, type, blocks, st); break;
    case 4: ok = launch_conv<4>(a, type, blocks, st); break;
    case 5: ok = launch_conv<5>(a, type, blocks, st); break;
    case 6: ok = launch_conv<6>(a, type, blocks, st); break;
    case 7: ok = launch_conv<7>(a, type, blocks, st); break;
    default: ok = launch_conv<8>(a, type, blocks, st); break;
  }
  return ok ? 0 : -3;
}
