// Adapters of many requests beside one shared projection (stb_linear_pool):
//   y[m] = x[m].W^T + scale_t ((x[m].A_t^T).B_t^T) + bias,   t = rows[m] (none where negative),
// the shared product and bias as stb_linear does them, the thin products by two kernels around it.
//
// What bounds them: the factors of every slot in use, read once (the rows of a slot go through them 16 at a time), and the
// launches.  One block serves one slot: the block of the slot's first row, which finds the others in `rows`; blocks of
// other rows leave at once.  Both products run on the tensor cores in TF32 terms (the 16 rows are the product's rows):
// BF16 and F16 factors are TF32 values already, Float32 factors and the activations are split into two terms, so the
// result keeps 22 bits; sums of 32 products are joined in Float32.  A lane reads whole 16-byte pieces of a factor's row:
// the order of the summed index within 32 is the lanes', the same in both operands.
//   1. down: thin[s][m][j] = x[m] . A_t[j] over the s-th stretch of K (split so that the blocks cover the SMs even
//      for a single row), by warps in turn, joined in shared memory;
//   2. the shared product, launched as a dependent (its weights stream in while the first kernel drains);
//   3. up: adds the stretches in order, multiplies by B_t, adds to y.  Its factors are read before it waits for y.
#include <algorithm>

#include "gemv.cuh"
#include "tf32.cuh"

namespace stb {
namespace {

struct Pool {
  const void *a, *b;
  const int *ranks;
  const float *scales;
  int slots, max_rank;
  const int *rows;
  int *err;
};

constexpr int DOWN_RANKS = 32;   // ranks of a block of the first kernel
constexpr int UP_COLUMNS = 256;  // outputs of a block of the second
constexpr int MAX_RANK = 256;

__device__ __forceinline__ int rank_of(const Pool &p, int t) { return max(0, min(p.ranks[t], p.max_rank)); }

// The slot that this block serves (for rows m and later), or -1: a row without one, or not the slot's first row.
__device__ __forceinline__ int slot_served(const Pool &p, int m) {
  const int t = p.rows[m];
  if (t < 0) return -1;
  if (t >= p.slots) {
    *p.err = DEV_BAD_INDEX + 2;
    return -1;
  }
  bool before = false;
  for (int i = threadIdx.x; i < m; i += blockDim.x) before |= p.rows[i] == t;
  return __syncthreads_or(before) ? -1 : t;
}

// The next 16 rows of slot t from row `from` on, -1 behind the last; returns where to go on.  Ends with a barrier.
__device__ __forceinline__ int gather_rows(const Pool &p, int t, int from, int M, int (&s_rows)[16], int &s_next) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    if (lane < 16) s_rows[lane] = -1;
    __syncwarp();
    int count = 0, next = M;
    for (int i = from; i < M; i += 32) {
      const bool has = i + lane < M && p.rows[i + lane] == t;
      const uint32_t which = __ballot_sync(0xffffffffu, has);
      const int at = count + __popc(which & ((1u << lane) - 1));
      if (has && at < 16) s_rows[at] = i + lane;
      const uint32_t over = __ballot_sync(0xffffffffu, has && at >= 16);
      count += __popc(which);
      if (over) {
        next = i + __ffs(over) - 1;
        break;
      }
    }
    if (lane == 0) s_next = next;
  }
  __syncthreads();
  return s_next;
}

// Eight neighbouring factor elements from index `at`, the first `live` of them (the others are zero).  VEC: 16-byte loads.
template <int DTYPE, bool VEC>
struct Eight {
  uint4 raw[DTYPE == STB_F32 ? 2 : 1];

  __device__ __forceinline__ void load(const void *base, size_t at, int live) {
#pragma unroll
    for (int i = 0; i < (DTYPE == STB_F32 ? 2 : 1); i++) raw[i] = make_uint4(0, 0, 0, 0);
    if (live <= 0) return;
    if (VEC) {
      const uint4 *p = (const uint4 *)((const char *)base + at * (DTYPE == STB_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < (DTYPE == STB_F32 ? 2 : 1); i++) raw[i] = __ldg(p + i);
      if (live >= 8) return;
      uint32_t *w = (uint32_t *)raw;
#pragma unroll
      for (int i = 0; i < (DTYPE == STB_F32 ? 8 : 4); i++) {
        if (DTYPE == STB_F32) w[i] = i < live ? w[i] : 0u;
        else w[i] = 2 * i + 1 < live ? w[i] : (2 * i < live ? w[i] & 0xffffu : 0u);
      }
    } else {
      uint32_t *w = (uint32_t *)raw;
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < live) {
          if (DTYPE == STB_F32) w[i] = ((const uint32_t *)base)[at + i];
          else w[i / 2] |= (uint32_t)((const uint16_t *)base)[at + i] << (16 * (i & 1));
        }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t *w = (const uint32_t *)raw;
    if constexpr (DTYPE == STB_F32) return __uint_as_float(w[i]);
    else if constexpr (DTYPE == STB_BF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __half2float(__ushort_as_half((uint16_t)(w[i / 2] >> (16 * (i & 1)))));
  }
};

// c += x . f over eight elements of each lane: hi and lo are x's terms (rows g, g + 8 by element), f the factor's.
template <int DTYPE, typename E>
__device__ __forceinline__ void eight_products(float (&c)[4], const uint32_t (&hi)[4][4], const uint32_t (&lo)[4][4], const E &f) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float f0 = f.get(2 * j), f1 = f.get(2 * j + 1);
    if constexpr (DTYPE == STB_F32) {
      uint32_t h0, l0, h1, l1;
      split_tf32(f0, h0, l0);
      split_tf32(f1, h1, l1);
      product_tf32(c, hi[j], l0, l1);
      product_tf32(c, lo[j], h0, h1);
      product_tf32(c, hi[j], h0, h1);
    } else {
      product_tf32(c, lo[j], __float_as_uint(f0), __float_as_uint(f1));
      product_tf32(c, hi[j], __float_as_uint(f0), __float_as_uint(f1));
    }
  }
}

// thin[blockIdx.y][m][j] for the rows of one slot, ranks 32 blockIdx.z .. + 31, columns blockIdx.y * stretch .. + stretch - 1
// (a multiple of 256).  VEC: x and A have rows of whole 16-byte pieces.
template <int DTYPE, bool VEC>
__global__ void __launch_bounds__(256) pool_down_kernel(const Pool p, const float *x, float *thin, int M, int K, int stretch) {
  constexpr int NT = DOWN_RANKS / 8;
  __shared__ float s_sum[8][16][DOWN_RANKS + 1];
  __shared__ int s_rows[16], s_next;
  const int m = blockIdx.x, j0 = blockIdx.z * DOWN_RANKS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  pdl_trigger();
  const int t = slot_served(p, m);
  if (t < 0) return;
  const int rank = rank_of(p, t) - j0;
  if (rank <= 0) return;
  const int k0 = blockIdx.y * stretch + warp * 32 + t4 * 8, k1 = min(K, (int)(blockIdx.y + 1) * stretch);
  for (int next = m; next < M;) {
    next = gather_rows(p, t, next, M, s_rows, s_next);
    const int m0 = s_rows[g], m1 = s_rows[g + 8];
    Eight<DTYPE, VEC> f[NT];
    Eight<STB_F32, VEC> x0, x1;
    auto read = [&](int k) {
      const int live = min(8, k1 - k);
#pragma unroll
      for (int n = 0; n < NT; n++)
        f[n].load(p.a, ((size_t)t * p.max_rank + j0 + n * 8 + g) * K + k, n * 8 + g < rank ? live : 0);
      x0.load(x, (size_t)max(m0, 0) * K + k, m0 >= 0 ? live : 0);
      x1.load(x, (size_t)max(m1, 0) * K + k, m1 >= 0 ? live : 0);
    };
    float acc[NT][4] = {};
    read(k0);
#pragma unroll 1
    for (int k = k0 - t4 * 8; k < k1; k += 256) {
      uint32_t hi[4][4], lo[4][4];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          split_tf32(x0.get(2 * j + i), hi[j][2 * i], lo[j][2 * i]);
          split_tf32(x1.get(2 * j + i), hi[j][2 * i + 1], lo[j][2 * i + 1]);
        }
      Eight<DTYPE, VEC> now[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) now[n] = f[n];
      read(k + 256 + t4 * 8);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        if (n * 8 >= rank) continue;
        float c[4] = {};
        eight_products<DTYPE>(c, hi, lo, now[n]);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] += c[i];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) s_sum[warp][g + 8 * (i >> 1)][n * 8 + 2 * t4 + (i & 1)] = acc[n][i];
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * DOWN_RANKS; e += 256) {
      const int i = e / DOWN_RANKS, j = e % DOWN_RANKS;
      if (s_rows[i] < 0 || j >= rank) continue;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; w++) v += s_sum[w][i][j];
      thin[((size_t)blockIdx.y * M + s_rows[i]) * p.max_rank + j0 + j] = v;
    }
    __syncthreads();
  }
}

// y[m][n] += scale_t thin[m] . B_t[n] for the rows of one slot, columns 256 blockIdx.y .. + 255; `stretches` partial sums
// of thin.  VEC: B has rows of whole 16-byte pieces.
template <int DTYPE, bool VEC>
__global__ void __launch_bounds__(256) pool_up_kernel(const Pool p, const float *thin, float *y, int M, int N, int stretches) {
  constexpr int NT = UP_COLUMNS / 64;  // 8-column results of a warp
  __shared__ float s_thin[16][MAX_RANK + 4];
  __shared__ int s_rows[16], s_next;
  const int m = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int n0 = blockIdx.y * UP_COLUMNS + warp * (UP_COLUMNS / 8);
  const int t = slot_served(p, m);
  const int rank = t >= 0 ? rank_of(p, t) : 0;
  if (rank == 0) return;
  const int blocks = (rank + 31) / 32;  // of 32 ranks
  const float scale = p.scales[t];
  Eight<DTYPE, VEC> f[NT];
  auto read = [&](int kb) {
    const int j = kb * 32 + t4 * 8;
#pragma unroll
    for (int n = 0; n < NT; n++)
      f[n].load(p.b, ((size_t)t * N + n0 + n * 8 + g) * p.max_rank + j, n0 + n * 8 + g < N ? min(8, rank - j) : 0);
  };
  read(0);
  int next = gather_rows(p, t, m, M, s_rows, s_next);
  pdl_wait();  // thin, and the shared product in y
  while (true) {
    for (int e = threadIdx.x; e < 16 * blocks * 32; e += 256) {
      const int i = e / (blocks * 32), j = e % (blocks * 32), row = s_rows[i];
      float v = 0.0f;
      if (row >= 0 && j < rank) {
        const float *at = thin + (size_t)row * p.max_rank + j;
#pragma unroll 8
        for (int s = 0; s < stretches; s++) v += __ldcg(at + (size_t)s * M * p.max_rank);
      }
      s_thin[i][j] = v;
    }
    __syncthreads();
    float acc[NT][4] = {};
#pragma unroll 1
    for (int kb = 0; kb < blocks; kb++) {
      uint32_t hi[4][4], lo[4][4];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int at = kb * 32 + t4 * 8 + 2 * j + i;
          split_tf32(s_thin[g][at], hi[j][2 * i], lo[j][2 * i]);
          split_tf32(s_thin[g + 8][at], hi[j][2 * i + 1], lo[j][2 * i + 1]);
        }
      Eight<DTYPE, VEC> now[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) now[n] = f[n];
      if (kb + 1 < blocks || next < M) read(kb + 1 < blocks ? kb + 1 : 0);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float c[4] = {};
        eight_products<DTYPE>(c, hi, lo, now[n]);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] += c[i];
      }
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int row = s_rows[g + 8 * half];
      if (row < 0) continue;
      float *to = y + (size_t)row * N;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int col = n0 + n * 8 + 2 * t4 + i;
          if (col < N) to[col] += scale * acc[n][2 * half + i];
        }
    }
    if (next >= M) return;
    __syncthreads();
    next = gather_rows(p, t, next, M, s_rows, s_next);
  }
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
    STB_REQUIRE(pool->slots > 0 && pool->max_rank > 0 && pool->max_rank <= MAX_RANK, "invalid adapter pool dimensions");
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
    STB_REQUIRE(w && (w_dtype == STB_F32 || w_dtype == STB_BF16 || w_dtype == STB_F16), "Linear: null weight or unsupported type");
    Pool p;
    p.a = (const void *)pool->a;
    p.b = (const void *)pool->b;
    p.ranks = (const int *)pool->ranks;
    p.scales = (const float *)pool->scales;
    p.slots = pool->slots;
    p.max_rank = pool->max_rank;
    p.rows = (const int *)rows;
    p.err = session_error_word(s);
    // About 1200 blocks of the first kernel were every row of a slot of its own, at least 256 columns each (measured at
    // 32 rows of 12 slots, K = 14336, rank 64: 1024 columns).
    const int chunks = (p.max_rank + DOWN_RANKS - 1) / DOWN_RANKS;
    const int64_t want = std::max<int64_t>(1, 1184 / ((int64_t)M * chunks));
    const int stretch = (int)(((K + want - 1) / want + 255) / 256 * 256);
    const int stretches = (K + stretch - 1) / stretch;
    const int columns = (N + UP_COLUMNS - 1) / UP_COLUMNS;
    STB_REQUIRE(columns <= 65535, "adapted Linear too wide");
    // The partial sums lie behind the shared product's own scratch.
    const uint64_t base = (skinny_eligible(M, N, K, w_dtype, (const void *)w) ? skinny_scratch_bytes(M, N, K, s->device) : 0) + 255 & ~255ull;
    float *thin = (float *)(session_scratch(s, base + (uint64_t)stretches * M * p.max_rank * sizeof(float)) + base);
    const bool vec_down = K % 8 == 0 && x % 16 == 0 && pool->a % 16 == 0;
    const bool vec_up = p.max_rank % 8 == 0 && pool->b % 16 == 0;
    auto go = [&](auto type) {
      constexpr int DT = decltype(type)::value;
      launch_kernel(vec_down ? pool_down_kernel<DT, true> : pool_down_kernel<DT, false>, dim3(M, stretches, chunks), dim3(256), 0,
                    s->stream, false, p, (const float *)x, thin, M, K, stretch);
      linear(s, x, K, w, w_dtype, bias, y, N, M, N, K, true);
      launch_kernel(vec_up ? pool_up_kernel<DT, true> : pool_up_kernel<DT, false>, dim3(M, columns), dim3(256), 0, s->stream, true, p,
                    (const float *)thin, (float *)y, M, N, stretches);
    };
    if (pool->dtype == STB_F32) go(std::integral_constant<int, STB_F32>());
    else if (pool->dtype == STB_BF16) go(std::integral_constant<int, STB_BF16>());
    else go(std::integral_constant<int, STB_F16>());
    count_launch(s, 2);
  });
}
