// The paged key/value cache as its kernels see it: addressing, and the widening of its element types.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace stb {

// The kernels of a batch of several requests start while the one before drains.  The rule they keep: before its wait a kernel
// reads only what was complete before its predecessor started, writes nothing that one reads or writes, and every block
// waits before it exits -- so a kernel that is done means that all before it are.  Norm and rotation, the cache's kernels,
// attention and pool_small_kernel wait first, read then, and let the next one start only then.  Two differ (adapter_pool.cu):
// pool_up_kernel lets the next one start at once and reads the rows' slots, ranks, scales and B before its wait: they were
// complete when pool_down_kernel, having waited, let the next one start.  pool_down_kernel behind a vector product (`behind`)
// reads and writes at once and waits at its end: that product was launched plainly, after all before it, and touches
// neither thin nor what the plan reads.
// One after another in a stream, norm and rotation of one token 3.0 -> 2.7 us, a cache write 2.2 -> 1.7, attention over 33
// tokens 5.9 -> 5.1; from Python 8.2 -> 5.3 us per call of the last.

// A cache of the caller's (stb_paged_cache), with the page table of the call.
struct PagedView {
  void *kv[2];        // keys, values: (pages, kv_heads, page_size, width)
  uint8_t *scale[2];  // E4M3: exponent + 127 per (page, head, slot)
  int pages, page_size, kv_heads, width;
  const int *tables;  // [batch][blocks]
  int batch, blocks;
  int *err;
};

// Host checks of a cache and its tables; throws STB_ERR_INVALID.
PagedView paged_view(stb_session *s, const stb_paged_cache *c, uint64_t tables, int batch, int blocks);

// The page of token `pos` of request `seq`, or -1 (recorded) where the indices name none.  Both >= 0.
__device__ __forceinline__ int paged_lookup(const PagedView &c, int seq, int pos, int block) {
  if (seq < c.batch && block < c.blocks) {
    const int page = c.tables[(size_t)seq * c.blocks + block];
    if ((unsigned)page < (unsigned)c.pages) return page;
  }
  *c.err = DEV_BAD_INDEX;
  return -1;
}

// Index of the (page, head, slot) row in the cache; 64-bit, a long cache passes 2^31 elements.
__device__ __forceinline__ size_t paged_row(const PagedView &c, int page, int head, int slot) {
  return ((size_t)page * c.kv_heads + head) * c.page_size + slot;
}

// 2^(byte - 127) for bytes 1 .. 254 (what an append writes); 0 and 255 are read as they are in Float32.
__device__ __forceinline__ float scale_of(uint8_t e) { return __uint_as_float((uint32_t)e << 23); }

// Two packed E4M3 bytes (low byte first) to Float32, exactly.
__device__ __forceinline__ float2 widen_e4m3x2(uint16_t u) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)u, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

template <int DTYPE>
__device__ __forceinline__ float paged_load(const void *base, size_t i) {
  if constexpr (DTYPE == STB_F32) return ((const float *)base)[i];
  else if constexpr (DTYPE == STB_BF16) return widen1<__nv_bfloat16>(((const uint16_t *)base)[i]);
  else if constexpr (DTYPE == STB_F16) return widen1<__half>(((const uint16_t *)base)[i]);
  else return widen_e4m3x2(((const uint8_t *)base)[i]).x;
}

// Exponent of the smallest power of two that brings `top` (finite, >= 0) to 448 or below, at least -126;
// 0 for 0.  top = m 2^x with m in [1, 2): 448 = 1.75 2^8, so the exponent is x - 8, or x - 7 where
// m > 1.75 -- adding 0x1fffff to the bits carries into the exponent field exactly then.
__device__ __forceinline__ int e4m3_exponent(float top) {
  if (top == 0.0f) return 0;
  const int e = (int)((__float_as_uint(top) + 0x1fffffu) >> 23) - 127 - 8;
  return e < -126 ? -126 : e;
}

template <typename F>
void dispatch_paged(int dtype, F &&f) {
  switch (dtype) {
    case STB_F32: f(std::integral_constant<int, STB_F32>()); break;
    case STB_BF16: f(std::integral_constant<int, STB_BF16>()); break;
    case STB_F16: f(std::integral_constant<int, STB_F16>()); break;
    default: f(std::integral_constant<int, STB_E4M3>()); break;
  }
}

}  // namespace stb
