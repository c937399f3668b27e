// The paged cache as it is written and read back (stb_op_paged_append, stb_op_paged_read).
//
// append: element x of a (token, head) row is stored as x (F32), rne(x) (BF16, F16), or for E4M3 as
// rne(x / 2^e) with the row's own scale 2^e, the smallest power of two with max |x| <= 448 * 2^e.  A power
// of two costs no accuracy in a floating type (the row's largest value still lands in (224, 448]), and
// makes x / 2^e and the way back exact, so a cached value is the same whichever kernel widens it.
// read: the stored value times its scale, exact in Float32.
#include <cmath>

#include "paged.cuh"

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

// One warp per (token, head), keys then values.
template <int DTYPE>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedView c, const Rows r) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
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
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedView c, const Rows r) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
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

unsigned grid_of(const PagedView &c, int rows) {
  const int64_t blocks = ((int64_t)rows * c.kv_heads + 7) / 8;
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
      launch_kernel(paged_append_kernel<decltype(t)::value>, dim3(grid_of(c, rows)), dim3(256), 0, s->stream, false, c,
                    r);
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
      launch_kernel(paged_read_kernel<decltype(t)::value>, dim3(grid_of(c, rows)), dim3(256), 0, s->stream, false, c, r);
    });
    count_launch(s);
  });
}

}  // extern "C"
