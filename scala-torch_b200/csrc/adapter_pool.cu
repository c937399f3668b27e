// Adapters of many requests beside one shared projection (stb_linear_pool):
//   y[m] = x[m].W^T + scale_t ((x[m].A_t^T).B_t^T) + bias,   t = rows[m] (none where negative),
// the shared product as stb_linear does it, the thin products in Float32.
#include "gemv.cuh"

namespace stb {

void linear(stb_session *s, uint64_t x, int ldx, uint64_t w, int w_dtype, uint64_t bias, uint64_t y, int ldy,
            int M, int N, int K);

namespace {

struct Pool {
  const void *a, *b;
  const int *ranks;
  const float *scales;
  int slots, max_rank;
  const int *rows;
  int *err;
};

template <int DTYPE>
__device__ __forceinline__ float factor(const void *p, size_t i) {
  if constexpr (DTYPE == STB_F32) return ((const float *)p)[i];
  else if constexpr (DTYPE == STB_BF16) return widen1<__nv_bfloat16>(((const uint16_t *)p)[i]);
  else return widen1<__half>(((const uint16_t *)p)[i]);
}

// The slot of row m, or -1; a slot behind the pool is recorded.
__device__ __forceinline__ int slot_of(const Pool &p, int m) {
  const int t = p.rows[m];
  if (t >= p.slots) {
    *p.err = DEV_BAD_INDEX + 2;
    return -1;
  }
  return t;
}

__device__ __forceinline__ int rank_of(const Pool &p, int t) { return max(0, min(p.ranks[t], p.max_rank)); }

// thin[m][j] = x[m] . A_t[j]: one warp per output.
template <int DTYPE>
__global__ void __launch_bounds__(256) pool_down_kernel(const Pool p, const float *x, float *thin, int M, int K) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (unit >= (int64_t)M * p.max_rank) return;
  const int m = (int)(unit / p.max_rank), j = (int)(unit % p.max_rank);
  const int t = slot_of(p, m);
  if (t < 0 || j >= rank_of(p, t)) return;
  float acc = 0.0f;
  for (int k = lane; k < K; k += 32)
    acc = fmaf(x[(size_t)m * K + k], factor<DTYPE>(p.a, ((size_t)t * p.max_rank + j) * K + k), acc);
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if (lane == 0) thin[unit] = acc;
}

// y[m][n] += scale_t thin[m] . B_t[n] + bias[n]: one thread per output.
template <int DTYPE>
__global__ void __launch_bounds__(256) pool_up_kernel(const Pool p, const float *thin, const float *bias, float *y, int M,
                                                      int N) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)M * N) return;
  const int m = (int)(i / N), n = (int)(i % N);
  const int t = slot_of(p, m);
  float v = y[i];
  if (t >= 0) {
    float u = 0.0f;
    const int r = rank_of(p, t);
    for (int j = 0; j < r; j++)
      u = fmaf(thin[(size_t)m * p.max_rank + j], factor<DTYPE>(p.b, ((size_t)t * N + n) * p.max_rank + j), u);
    v += u * p.scales[t];
  }
  y[i] = bias ? v + bias[n] : v;
}

}  // namespace
}  // namespace stb

using namespace stb;

extern "C" int stb_linear_pool(stb_session *s, uint64_t x, uint64_t w, int w_dtype, uint64_t bias,
                               const stb_adapter_pool *pool, uint64_t rows, uint64_t y, int M, int N, int K) {
  return guarded([&] {
    enter(s);
    STB_REQUIRE(pool, "adapter pool is null");
    STB_REQUIRE(pool->dtype == STB_F32 || pool->dtype == STB_BF16 || pool->dtype == STB_F16, "unsupported adapter type");
    STB_REQUIRE(pool->slots > 0 && pool->max_rank > 0 && pool->max_rank <= 256, "invalid adapter pool dimensions");
    const uint64_t size = pool->dtype == STB_F32 ? 4 : 2;
    STB_REQUIRE(pool->a && pool->b && pool->a % size == 0 && pool->b % size == 0,
                "adapter factors: null or misaligned buffer");
    STB_REQUIRE(pool->ranks && pool->scales && pool->ranks % 4 == 0 && pool->scales % 4 == 0,
                "adapter ranks or scales: null or misaligned buffer");
    STB_REQUIRE(M >= 0 && N >= 0 && K >= 0, "Linear dimensions must be nonnegative");
    if (!M || !N || !K) {
      linear(s, x, K, w, w_dtype, bias, y, N, M, N, K);
      return;
    }
    STB_REQUIRE(rows && rows % 4 == 0, "null or misaligned row slots");
    STB_REQUIRE(x && y && x % 4 == 0 && y % 4 == 0 && bias % 4 == 0, "Linear: null or misaligned Float32 buffer");
    Pool p;
    p.a = (const void *)pool->a;
    p.b = (const void *)pool->b;
    p.ranks = (const int *)pool->ranks;
    p.scales = (const float *)pool->scales;
    p.slots = pool->slots;
    p.max_rank = pool->max_rank;
    p.rows = (const int *)rows;
    p.err = session_error_word(s);
    const int64_t units = (int64_t)M * p.max_rank, outs = (int64_t)M * N;
    STB_REQUIRE(units / 8 < 0x7fffffff && outs / 256 < 0x7fffffff, "adapted Linear too large");
    linear(s, x, K, w, w_dtype, 0, y, N, M, N, K);
    float *thin = (float *)session_scratch(s, units * sizeof(float));
    auto go = [&](auto t) {
      constexpr int DT = decltype(t)::value;
      launch_kernel(pool_down_kernel<DT>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, s->stream, false, p,
                    (const float *)x, thin, M, K);
      launch_kernel(pool_up_kernel<DT>, dim3((unsigned)((outs + 255) / 256)), dim3(256), 0, s->stream, false, p,
                    (const float *)thin, (const float *)bias, (float *)y, M, N);
    };
    if (pool->dtype == STB_F32) go(std::integral_constant<int, STB_F32>());
    else if (pool->dtype == STB_BF16) go(std::integral_constant<int, STB_BF16>());
    else go(std::integral_constant<int, STB_F16>());
    count_launch(s, 2);
  });
}
