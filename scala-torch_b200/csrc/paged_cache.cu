// The paged cache as it is written and read back (stb_op_paged_append, stb_op_paged_read).
//
// append: element x of a (token, head) row is stored as x (F32), rne(x) (BF16, F16), or for E4M3 as
// rne(x / 2^e) with the row's own scale 2^e, the smallest power of two with max |x| <= 448 * 2^e.  A power
// of two costs no accuracy in a floating type (the row's largest value still lands in (224, 448]), and
// makes x / 2^e and the way back exact, so a cached value is the same whichever kernel widens it.
// read: the stored value times its scale, exact in Float32.
//
// What bounds both: the bytes, 4 per Float32 element and 1 to 4 per stored one, each moved once.  A group of 16 or 32 lanes
// takes the keys and values of a head for R tokens in a row, a float4 per lane each, all sent for at once (append) or
// as soon as the tokens' pages are known (read); the lanes look the R pages up side by side.  R = 4 keeps 64 to 128 KB
// under way per SM; calls too small to fill the SMs that way take R = 1.  E4M3, 8 heads of 128: append of 14273 tokens 29 us =
// 5.1 TB/s, read of 20005 38 us = 5.4 TB/s, 3 us of each the launch and the ramp (26 and 35 us on the same buffers again, partly out
// of L2).
#include <cmath>

#include "paged.cuh"
#include "tc_common.cuh"

namespace stb {

PagedView paged_view(stb_session *s, const stb_paged_cache *c, uint64_t tables, int batch, int blocks) {
  STB_REQUIRE(c, "paged cache is null");
  STB_REQUIRE(c->dtype >= STB_F32 && c->dtype <= STB_E4M3, "paged cache type");
  STB_REQUIRE(c->pages > 0 && c->page_size > 0 && c->kv_heads > 0 && c->width > 0 && c->width <= 512,
              "invalid paged cache dimensions");
  const uint64_t size = c->dtype == STB_F32 ? 4 : (c->dtype == STB_E4M3 ? 1 : 2);
  STB_REQUIRE(c->keys && c->values && c->keys % size == 0 && c->values % size == 0,
              "paged cache: null or misaligned buffer");
  STB_REQUIRE((c->dtype == STB_E4M3) == (c->key_scales != 0) && (c->dtype == STB_E4M3) == (c->value_scales != 0),
              "an E4M3 cache has scales, the other types have none");
  STB_REQUIRE(batch >= 0 && blocks >= 0, "invalid page tables");
  STB_REQUIRE(batch == 0 || blocks == 0 || (tables && tables % 4 == 0), "null or misaligned page tables");
  STB_REQUIRE((int64_t)blocks * c->page_size <= 0x7fffffff, "page tables longer than Int positions");
  PagedView v;
  v.kv[0] = (void *)c->keys;
  v.kv[1] = (void *)c->values;
  v.scale[0] = (uint8_t *)c->key_scales;
  v.scale[1] = (uint8_t *)c->value_scales;
  v.pages = c->pages;
  v.page_size = c->page_size;
  v.kv_heads = c->kv_heads;
  v.width = c->width;
  v.tables = (const int *)tables;
  v.batch = batch;
  v.blocks = blocks;
  v.err = session_error_word(s);
  return v;
}

namespace {

struct Rows {
  float *data[2];
  int64_t row[2], head[2];
  const int *sequences, *positions;
  int rows;
};

// One warp per (token, head), keys then values: any width and alignment.
template <int DTYPE>
__global__ void __launch_bounds__(256) paged_append_any_kernel(const PagedView c, const Rows r) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (unit >= (int64_t)r.rows * c.kv_heads) return;
  const int row = (int)(unit / c.kv_heads), head = (int)(unit % c.kv_heads);
  const int seq = r.sequences[row], pos = r.positions[row];
  if (seq < 0 || pos < 0) return;
  const int page = paged_lookup(c, seq, pos, pos / c.page_size);
  if (page < 0) return;
  const size_t at = paged_row(c, page, head, pos % c.page_size);
  for (int side = 0; side < 2; side++) {
    const float *x = r.data[side] + row * r.row[side] + head * r.head[side];
    if constexpr (DTYPE == STB_E4M3) {
      float top = 0.0f;
      for (int d = lane; d < c.width; d += 32) {
        const float a = fabsf(x[d]);
        if (a <= 3.402823466e38f) top = fmaxf(top, a);
      }
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const int e = e4m3_exponent(top);
      const float inverse = scale_of((uint8_t)(127 - e));
      for (int d = lane; d < c.width; d += 32) {
        const float v = x[d];
        ((uint8_t *)c.kv[side])[at * c.width + d] =
            isfinite(v) ? __nv_cvt_float_to_fp8(v * inverse, __NV_SATFINITE, __NV_E4M3) : (uint8_t)0x7f;
      }
      if (lane == 0) c.scale[side][at] = (uint8_t)(e + 127);
    } else {
      for (int d = lane; d < c.width; d += 32) {
        const size_t i = at * c.width + d;
        if constexpr (DTYPE == STB_F32) ((float *)c.kv[side])[i] = x[d];
        else if constexpr (DTYPE == STB_BF16) ((uint16_t *)c.kv[side])[i] = f32_to_bf16_rne(x[d]);
        else ((__half *)c.kv[side])[i] = __float2half_rn(x[d]);
      }
    }
  }
}

template <int DTYPE>
__global__ void __launch_bounds__(256) paged_read_any_kernel(const PagedView c, const Rows r) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (unit >= (int64_t)r.rows * c.kv_heads) return;
  const int row = (int)(unit / c.kv_heads), head = (int)(unit % c.kv_heads);
  const int seq = r.sequences[row], pos = r.positions[row];
  if (seq < 0 || pos < 0) return;
  const int page = paged_lookup(c, seq, pos, pos / c.page_size);
  if (page < 0) return;
  const size_t at = paged_row(c, page, head, pos % c.page_size);
  for (int side = 0; side < 2; side++) {
    float *y = r.data[side] + row * r.row[side] + head * r.head[side];
    const float scale = DTYPE == STB_E4M3 ? scale_of(c.scale[side][at]) : 1.0f;
    for (int d = lane; d < c.width; d += 32) {
      const float v = paged_load<DTYPE>(c.kv[side], at * c.width + d);
      y[d] = DTYPE == STB_E4M3 ? v * scale : v;
    }
  }
}

// Rows of the cache that tokens r0 .. r0 + R - 1 take at head `head` (-1: none), one per lane of the group, lanes 0 .. R - 1.
template <int R>
__device__ __forceinline__ int64_t token_row(const PagedView &c, const Rows &r, int64_t r0, int head, int lane) {
  if (lane >= R || r0 + lane >= r.rows) return -1;
  const int seq = r.sequences[r0 + lane], pos = r.positions[r0 + lane];
  if (seq < 0 || pos < 0) return -1;
  const int page = paged_lookup(c, seq, pos, pos / c.page_size);
  return page < 0 ? -1 : (int64_t)paged_row(c, page, head, pos % c.page_size);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return (uint32_t)f32_to_bf16_rne(a) | (uint32_t)f32_to_bf16_rne(b) << 16;
}

// L lanes of V float4 each per head (4 L V >= width); the group's unit is (R tokens, head).
template <int DTYPE, int L, int V, int R>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedView c, const Rows r) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
  const int lane = threadIdx.x % L, head = (int)(unit % c.kv_heads);
  const int64_t r0 = unit / c.kv_heads * R;
  float4 x[2][R][V];
  pdl_wait();
  pdl_trigger();
#pragma unroll
  for (int side = 0; side < 2; side++)
#pragma unroll
    for (int k = 0; k < R; k++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int d = (v * L + lane) * 4;
        const float *from = side ? r.data[1] + (r0 + k) * r.row[1] + head * r.head[1] : r.data[0] + (r0 + k) * r.row[0] + head * r.head[0];
        x[side][k][v] = r0 + k < r.rows && d < c.width ? __ldcs((const float4 *)(from + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
  const int64_t mine = token_row<R>(c, r, r0, head, lane);
#pragma unroll
  for (int k = 0; k < R; k++) {
    const int64_t at = __shfl_sync(0xffffffffu, mine, k, L);
#pragma unroll
    for (int side = 0; side < 2; side++) {
      int e = 0;
      float inverse = 1.0f;
      bool infinite = false;
      if (DTYPE == STB_E4M3) {  // every group of the warp takes part in the reductions
        auto widest = [&](bool finite_only) {
          float top = 0.0f;
#pragma unroll
          for (int v = 0; v < V; v++) {
            const float f[4] = {x[side][k][v].x, x[side][k][v].y, x[side][k][v].z, x[side][k][v].w};
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (!finite_only || fabsf(f[i]) < INFINITY) top = fmaxf(top, fabsf(f[i]));  // drops NaNs
          }
          if constexpr (L == 32) {
            return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
          } else {
#pragma unroll
            for (int off = L / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            return top;
          }
        };
        float top = widest(false);
        infinite = top == INFINITY;
        if (__any_sync(0xffffffffu, infinite)) top = widest(true);
        e = e4m3_exponent(top);
        inverse = scale_of((uint8_t)(127 - e));
      }
      if (at < 0) continue;
      if (DTYPE == STB_E4M3 && lane == 0) (side ? c.scale[1] : c.scale[0])[at] = (uint8_t)(e + 127);
      void *base = side ? c.kv[1] : c.kv[0];
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int d = (v * L + lane) * 4;
        if (d >= c.width) continue;
        const float4 f = x[side][k][v];
        const size_t i = (size_t)at * c.width + d;
        if constexpr (DTYPE == STB_F32) {
          *(float4 *)((float *)base + i) = f;
        } else if constexpr (DTYPE == STB_BF16) {
          *(uint2 *)((uint16_t *)base + i) = make_uint2(pack_bf16(f.x, f.y), pack_bf16(f.z, f.w));
        } else if constexpr (DTYPE == STB_F16) {
          const __half2 a = __floats2half2_rn(f.x, f.y), b = __floats2half2_rn(f.z, f.w);
          *(uint2 *)((uint16_t *)base + i) = make_uint2(*(const uint32_t *)&a, *(const uint32_t *)&b);
        } else {
          uint32_t u = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.x * inverse, f.y * inverse), __NV_SATFINITE, __NV_E4M3) |
                       (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.z * inverse, f.w * inverse), __NV_SATFINITE, __NV_E4M3) << 16;
          if (infinite) {  // the conversion would saturate it
            const float g[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int b = 0; b < 4; b++)
              if (isinf(g[b])) u = (u & ~(0xffu << (8 * b))) | 0x7fu << (8 * b);
          }
          *(uint32_t *)((uint8_t *)base + i) = u;
        }
      }
    }
  }
}

template <int DTYPE, int L, int V, int R>
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedView c, const Rows r) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
  const int lane = threadIdx.x % L, head = (int)(unit % c.kv_heads);
  const int64_t r0 = unit / c.kv_heads * R;
  pdl_wait();
  pdl_trigger();
  const int64_t mine = token_row<R>(c, r, r0, head, lane);
  uint4 raw[2][R][V];  // as stored: 4 elements
  uint8_t e[2][R];
#pragma unroll
  for (int k = 0; k < R; k++) {
    const int64_t at = __shfl_sync(0xffffffffu, mine, k, L);
#pragma unroll
    for (int side = 0; side < 2; side++) {
      const void *base = side ? c.kv[1] : c.kv[0];
      e[side][k] = DTYPE == STB_E4M3 && at >= 0 ? (side ? c.scale[1] : c.scale[0])[at] : (uint8_t)127;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int d = (v * L + lane) * 4;
        raw[side][k][v] = make_uint4(0, 0, 0, 0);
        if (at < 0 || d >= c.width) continue;
        const size_t i = (size_t)at * c.width + d;
        if constexpr (DTYPE == STB_F32) {
          raw[side][k][v] = *(const uint4 *)((const float *)base + i);
        } else if constexpr (DTYPE == STB_E4M3) {
          raw[side][k][v].x = *(const uint32_t *)((const uint8_t *)base + i);
        } else {
          const uint2 u = *(const uint2 *)((const uint16_t *)base + i);
          raw[side][k][v].x = u.x;
          raw[side][k][v].y = u.y;
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < R; k++) {
    if (__shfl_sync(0xffffffffu, mine, k, L) < 0) continue;
#pragma unroll
    for (int side = 0; side < 2; side++) {
      float *to = side ? r.data[1] + (r0 + k) * r.row[1] + head * r.head[1] : r.data[0] + (r0 + k) * r.row[0] + head * r.head[0];
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int d = (v * L + lane) * 4;
        if (d >= c.width) continue;
        const uint4 u = raw[side][k][v];
        float4 f;
        if constexpr (DTYPE == STB_F32) {
          f = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
        } else if constexpr (DTYPE == STB_E4M3) {
          const float2 a = widen_e4m3x2((uint16_t)u.x), b = widen_e4m3x2((uint16_t)(u.x >> 16));
          const float s = scale_of(e[side][k]);
          f = make_float4(a.x * s, a.y * s, b.x * s, b.y * s);
        } else {
          using T = std::conditional_t<DTYPE == STB_BF16, __nv_bfloat16, __half>;
          const float2 a = widen2<T>(u.x), b = widen2<T>(u.y);
          f = make_float4(a.x, a.y, b.x, b.y);
        }
        __stcs((float4 *)(to + d), f);
      }
    }
  }
}

Rows paged_rows(const PagedView &c, uint64_t k, int64_t k_row, int64_t k_head, uint64_t v, int64_t v_row, int64_t v_head,
                uint64_t sequences, uint64_t positions, int rows) {
  STB_REQUIRE(k && v && k % 4 == 0 && v % 4 == 0, "paged rows: null or misaligned Float32 buffer");
  STB_REQUIRE(sequences && positions && sequences % 4 == 0 && positions % 4 == 0, "null or misaligned row indices");
  STB_REQUIRE(rows == 1 || (k_row >= c.width && v_row >= c.width), "paged rows overlap");
  STB_REQUIRE(c.kv_heads == 1 || (k_head >= c.width && v_head >= c.width), "paged heads overlap");
  Rows r;
  r.data[0] = (float *)k;
  r.data[1] = (float *)v;
  r.row[0] = k_row;
  r.row[1] = v_row;
  r.head[0] = k_head;
  r.head[1] = v_head;
  r.sequences = (const int *)sequences;
  r.positions = (const int *)positions;
  r.rows = rows;
  return r;
}

// Whether rows and cache can be moved four elements at a time.
bool in_quads(const PagedView &c, const Rows &r, int dtype) {
  const uint64_t size = dtype == STB_F32 ? 16 : (dtype == STB_E4M3 ? 4 : 8);
  bool ok = c.width % 4 == 0 && c.width <= 256;
  for (int i = 0; i < 2; i++)
    ok &= (uint64_t)c.kv[i] % size == 0 && (uint64_t)r.data[i] % 16 == 0 && (r.rows == 1 || r.row[i] % 4 == 0) && (c.kv_heads == 1 || r.head[i] % 4 == 0);
  return ok;
}

// launch(L, V, R) with integral constants: lanes per head, float4 per lane, tokens per group.
template <typename F>
void by_shape(stb_session *s, const PagedView &c, int rows, F &&launch) {
  auto go = [&](auto l, auto v) {
    constexpr int L = decltype(l)::value;
    // four tokens per group once that still gives every SM 16 warps
    if ((int64_t)rows * c.kv_heads * L >= (int64_t)tc::sm_count(s->device) * 512 * 4) launch(l, v, std::integral_constant<int, 4>());
    else launch(l, v, std::integral_constant<int, 1>());
  };
  using std::integral_constant;
  if (c.width <= 64) go(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (c.width <= 128) go(integral_constant<int, 32>(), integral_constant<int, 1>());
  else go(integral_constant<int, 32>(), integral_constant<int, 2>());
}

unsigned grid_of(const PagedView &c, int rows, int lanes, int tokens) {
  const int64_t units = ((int64_t)rows + tokens - 1) / tokens * c.kv_heads, blocks = (units * lanes + 255) / 256;
  STB_REQUIRE(blocks <= 0x7fffffff, "too many rows");
  return (unsigned)blocks;
}

}  // namespace
}  // namespace stb

using namespace stb;

extern "C" {

int stb_op_paged_append(stb_session *s, const stb_paged_cache *cache, uint64_t k, int64_t k_row, int64_t k_head,
                        uint64_t v, int64_t v_row, int64_t v_head, uint64_t tables, int batch, int blocks,
                        uint64_t sequences, uint64_t positions, int rows) {
  return guarded([&] {
    enter(s);
    STB_REQUIRE(rows >= 0, "negative row count");
    const PagedView c = paged_view(s, cache, tables, batch, blocks);
    if (!rows) return;
    const Rows r = paged_rows(c, k, k_row, k_head, v, v_row, v_head, sequences, positions, rows);
    dispatch_paged(cache->dtype, [&](auto t) {
      constexpr int DT = decltype(t)::value;
      if (!in_quads(c, r, DT)) {
        launch_kernel(paged_append_any_kernel<DT>, dim3(grid_of(c, rows, 32, 1)), dim3(256), 0, s->stream, true, c, r);
        return;
      }
      by_shape(s, c, rows, [&](auto l, auto v, auto k) {
        constexpr int L = decltype(l)::value, V = decltype(v)::value, R = decltype(k)::value;
        launch_kernel(paged_append_kernel<DT, L, V, R>, dim3(grid_of(c, rows, L, R)), dim3(256), 0, s->stream, true, c, r);
      });
    });
    count_launch(s);
  });
}

int stb_op_paged_read(stb_session *s, const stb_paged_cache *cache, uint64_t tables, int batch, int blocks,
                      uint64_t sequences, uint64_t positions, int rows, uint64_t k, int64_t k_row, int64_t k_head,
                      uint64_t v, int64_t v_row, int64_t v_head) {
  return guarded([&] {
    enter(s);
    STB_REQUIRE(rows >= 0, "negative row count");
    const PagedView c = paged_view(s, cache, tables, batch, blocks);
    if (!rows) return;
    const Rows r = paged_rows(c, k, k_row, k_head, v, v_row, v_head, sequences, positions, rows);
    dispatch_paged(cache->dtype, [&](auto t) {
      constexpr int DT = decltype(t)::value;
      if (!in_quads(c, r, DT)) {
        launch_kernel(paged_read_any_kernel<DT>, dim3(grid_of(c, rows, 32, 1)), dim3(256), 0, s->stream, true, c, r);
        return;
      }
      by_shape(s, c, rows, [&](auto l, auto v, auto k) {
        constexpr int L = decltype(l)::value, V = decltype(v)::value, R = decltype(k)::value;
        launch_kernel(paged_read_kernel<DT, L, V, R>, dim3(grid_of(c, rows, L, R)), dim3(256), 0, s->stream, true, c, r);
      });
    });
    count_launch(s);
  });
}

}  // extern "C"
