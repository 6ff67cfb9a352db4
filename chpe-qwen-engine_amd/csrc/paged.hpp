// paged.hpp -- what the operators of the paged key/value cache share: the cache's addressing on the
// device, the checks of its description and of the stream on the host, the launch.
#pragma once
#include <utility>

#include "../../include/chpe.h"
#include "device_common.hpp"

namespace chpe {
namespace {

// A chpe_kv_pages on the device: strides in elements, the page size as a shift.
struct Pages {
  uint8_t *k, *v;
  const int32_t* table;
  uint64_t page_stride, head_stride, slot_stride;
  uint32_t n_pages, table_stride, capacity, KV;
  int shift;

  // the page that holds `slot` of a row's table; false (and page 0) for an id outside the pool
  __device__ bool page_of(uint32_t row, uint32_t slot, uint32_t* page) const {
    const uint32_t id = uint32_t(dev::gld(table + size_t(row) * table_stride + (slot >> shift)));
    *page = id < n_pages ? id : 0u;
    return id < n_pages;
  }
  // element offset of a head's row at `slot` in `page`
  __device__ size_t at(uint32_t page, uint32_t head, uint32_t slot) const {
    return page * page_stride + head * head_stride + (slot & ((1u << shift) - 1u)) * slot_stride;
  }
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The description's own checks: known type and head dim, whole pages, rows that start at 16-byte
// boundaries and do not lie in each other.
inline bool pages_from(const chpe_kv_pages* c, Pages* out) {
  if (!c || !c->k || !c->v || !aligned16(c->k) || !aligned16(c->v)) return false;
  if (c->type < 0 || c->type > 2 || c->kv_heads == 0 || c->n_pages == 0 || c->n_pages > 0x7fffffffu) return false;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return false;
  if (c->page_size == 0 || (c->page_size & (c->page_size - 1)) != 0) return false;
  if (c->rows > 0 && (!c->table || c->pages_per_row == 0 || c->table_stride < c->pages_per_row)) return false;
  if (uint64_t(c->pages_per_row) * c->page_size > 0x7fffffffu) return false;
  uint64_t st[3] = {c->page_stride, c->head_stride, c->slot_stride};
  uint64_t n[3] = {c->n_pages, c->kv_heads, c->page_size};
  const uint64_t per16 = c->type == 0 ? 4 : 8;
  // a dimension of one entry may have any stride; the others, from the innermost outwards, have to
  // step over what lies inside them
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (st[j] < st[i]) { std::swap(st[i], st[j]); std::swap(n[i], n[j]); }
  uint64_t extent = c->head_dim;
  for (int i = 0; i < 3; ++i) {
    if (n[i] == 1) continue;
    if (st[i] < extent || st[i] % per16 != 0 || st[i] > (uint64_t(1) << 60) / n[i]) return false;
    extent = st[i] * n[i];
  }
  int shift = 0;
  while ((1u << shift) < c->page_size) ++shift;
  *out = Pages{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->table, c->n_pages > 1 ? c->page_stride : 0,
               c->kv_heads > 1 ? c->head_stride : 0, c->page_size > 1 ? c->slot_stride : 0, c->n_pages, c->table_stride,
               c->pages_per_row * c->page_size, c->kv_heads, shift};
  return true;
}

// false for a stream of another device than the current one, whose kernels would run there
inline bool stream_here(hipStream_t st) {
  if (st == nullptr || st == hipStreamLegacy || st == hipStreamPerThread) return true;
  int cur = 0;
  hipDevice_t dev = 0;
  if (hipGetDevice(&cur) == hipSuccess && hipStreamGetDevice(st, &dev) == hipSuccess) return dev == cur;
  (void)hipGetLastError();
  return false;
}

constexpr uint64_t kMaxItems = (uint64_t(1) << 32) - 1;  // work-items of a launch
constexpr uint64_t kMaxBlocks = uint64_t(1) << 23;       // of 256 threads: half of that

// one launch; its own error, not one that an earlier call of the program left
template <class... P, class... A>
inline bool launch(void (*kernel)(P...), uint64_t blocks, uint32_t threads, hipStream_t st, A... args) {
  void* argv[] = {static_cast<void*>(&args)...};
  if (hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(uint32_t(blocks)), dim3(threads), argv, 0, st) ==
      hipSuccess)
    return true;
  (void)hipGetLastError();
  return false;
}

// inclusive prefix sum over the wave on the vector ALU: row_shr 1, 2, 4, 8 within rows of 16 lanes, then the
// last lane of row 0 / 2 to row 1 / 3 (row_bcast 15) and lane 31 to the upper half (row_bcast 31)
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x111, 0xf, 0xf, false));
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x112, 0xf, 0xf, false));
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x114, 0xf, 0xf, false));
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x118, 0xf, 0xf, false));
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x142, 0xa, 0xf, false));
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x143, 0xc, 0xf, false));
  return v;
}
// the value of lane `at`, which is the same in all lanes
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int at) { return uint32_t(__builtin_amdgcn_readlane(int(v), at)); }

// Loads and stores of what a launch touches once and in bulk: keys, values, activations.  Marked as not to be
// kept, they leave the caches to the rest (1.1 GB read once: 7.1 TB/s, without the mark 6.3).
template <class T>
__device__ __forceinline__ T ld_once(const T* p) {
  return __builtin_nontemporal_load(dev::as_global(p));
}
template <class T>
__device__ __forceinline__ void st_once(T* p, T v) {
  __builtin_nontemporal_store(v, (__attribute__((address_space(1))) T*)p);
}
// a value that is the same in all lanes, as a scalar
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return uint32_t(__builtin_amdgcn_readfirstlane(int(v))); }
__device__ __forceinline__ uint64_t uniform64(uint64_t v) { return uint64_t(uniform(uint32_t(v >> 32))) << 32 | uniform(uint32_t(v)); }

// element types of the cache
struct Bf16 {
  uint16_t bits;
};
template <class T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ float get(const float* p) { return dev::gld(p); }
  static __device__ float put(float v) { return v; }
};
template <>
struct Elem<_Float16> {
  static __device__ float get(const _Float16* p) { return float(dev::gld(p)); }
  static __device__ _Float16 put(float v) { return _Float16(v); }
};
template <>
struct Elem<Bf16> {
  static __device__ float get(const Bf16* p) { return dev::bf2f(dev::gld(reinterpret_cast<const uint16_t*>(p))); }
  // round to nearest, ties to even; a NaN stays one
  static __device__ Bf16 put(float v) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return Bf16{uint16_t((u >> 16) | 0x40u)};
    return Bf16{uint16_t((u + 0x7fffu + ((u >> 16) & 1u)) >> 16)};
  }
};

}  // namespace
}  // namespace chpe
