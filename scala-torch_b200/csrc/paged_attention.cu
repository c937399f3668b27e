// Attention of one new token per request over its paged cache (stb_op_paged_attention):
//   y[b, h] = sum_j softmax_j(q[b, h] . k_j / sqrt(width)) v_j,   j < lengths[b],  h on kv head h / group,
// zeros where lengths[b] <= 0.  Softmax with the running maximum and sum, everything in Float32.
#include <cmath>

#include "paged.cuh"

namespace stb {
namespace {

struct AttendArgs {
  const float *q;
  float *y;
  int64_t q_row, y_row;
  const int *lengths;
  int heads, group;
  float scale_log2;  // log2(e) / sqrt(width)
};

__device__ __forceinline__ int attend_length(const PagedView &c, const AttendArgs &a, int b) {
  const int n = a.lengths[b], most = c.blocks * c.page_size;
  if (n > most) *c.err = DEV_BAD_INDEX + 1;
  return min(n, most);
}

// One block per (request, query head): its warps take keys in turn, a lane every 32nd dimension.
template <int DTYPE>
__global__ void __launch_bounds__(256) paged_attention_kernel(const PagedView c, const AttendArgs a) {
  constexpr int W = 8, D = 16;  // warps; dimensions of a lane (width <= 512)
  __shared__ float s_max[W], s_sum[W], s_acc[W][512];
  const int b = blockIdx.y, h = blockIdx.x, kvh = h / a.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = attend_length(c, a, b);
  float q[D], acc[D];
#pragma unroll
  for (int i = 0; i < D; i++) {
    const int d = i * 32 + lane;
    q[i] = d < c.width ? a.q[b * a.q_row + (size_t)h * c.width + d] * a.scale_log2 : 0.0f;
    acc[i] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;
  for (int j = warp; j < n; j += W) {
    const int page = paged_lookup(c, b, j, j / c.page_size);
    if (page < 0) continue;
    const size_t at = paged_row(c, page, kvh, j % c.page_size);
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < D; i++)
      if (i * 32 + lane < c.width) dot = fmaf(q[i], paged_load<DTYPE>(c.kv[0], at * c.width + i * 32 + lane), dot);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    if (DTYPE == STB_E4M3) dot *= scale_of(c.scale[0][at]);
    const float now = fmaxf(top, dot), keep = top == now ? 1.0f : exp2f(top - now), p = exp2f(dot - now);
    const float pv = DTYPE == STB_E4M3 ? p * scale_of(c.scale[1][at]) : p;
    sum = sum * keep + p;
#pragma unroll
    for (int i = 0; i < D; i++)
      if (i * 32 + lane < c.width)
        acc[i] = fmaf(acc[i], keep, pv * paged_load<DTYPE>(c.kv[1], at * c.width + i * 32 + lane));
    top = now;
  }
  if (lane == 0) {
    s_max[warp] = top;
    s_sum[warp] = sum;
  }
#pragma unroll
  for (int i = 0; i < D; i++) s_acc[warp][i * 32 + lane] = acc[i];
  __syncthreads();
  float m = s_max[0];
  for (int w = 1; w < W; w++) m = fmaxf(m, s_max[w]);
  float total = 0.0f;
  for (int w = 0; w < W; w++)
    if (s_sum[w] != 0.0f) total += s_sum[w] * exp2f(s_max[w] - m);
  for (int d = threadIdx.x; d < c.width; d += 256) {
    float v = 0.0f;
    for (int w = 0; w < W; w++)
      if (s_sum[w] != 0.0f) v = fmaf(s_acc[w][d], exp2f(s_max[w] - m), v);
    a.y[b * a.y_row + (size_t)h * c.width + d] = total != 0.0f ? v / total : 0.0f;
  }
}

}  // namespace
}  // namespace stb

using namespace stb;

extern "C" int stb_op_paged_attention(stb_session *s, const stb_paged_cache *cache, uint64_t q, int64_t q_row, int heads,
                                      uint64_t tables, int batch, int blocks, uint64_t lengths, uint64_t y,
                                      int64_t y_row) {
  return guarded([&] {
    enter(s);
    const PagedView c = paged_view(s, cache, tables, batch, blocks);
    STB_REQUIRE(heads > 0 && heads % c.kv_heads == 0, "invalid grouped attention heads");
    if (!batch) return;
    STB_REQUIRE(batch <= 65535, "paged attention takes at most 65535 requests");
    STB_REQUIRE(q && y && q % 4 == 0 && y % 4 == 0, "paged attention: null or misaligned Float32 buffer");
    STB_REQUIRE(lengths && lengths % 4 == 0, "null or misaligned lengths");
    STB_REQUIRE(batch == 1 || (q_row >= (int64_t)heads * c.width && y_row >= (int64_t)heads * c.width),
                "paged attention rows overlap");
    AttendArgs a;
    a.q = (const float *)q;
    a.y = (float *)y;
    a.q_row = q_row;
    a.y_row = y_row;
    a.lengths = (const int *)lengths;
    a.heads = heads;
    a.group = heads / c.kv_heads;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)c.width));
    dispatch_paged(cache->dtype, [&](auto t) {
      launch_kernel(paged_attention_kernel<decltype(t)::value>, dim3(heads, batch), dim3(256), 0, s->stream, false, c, a);
    });
    count_launch(s);
  });
}
