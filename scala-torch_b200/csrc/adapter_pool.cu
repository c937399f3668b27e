// Adapters of many requests beside one shared projection (stb_linear_pool):
//   y[m] = x[m].W^T + scale_t ((x[m].A_t^T).B_t^T) + bias,   t = rows[m] (none where negative),
// the shared product and bias as stb_linear does them, the thin products by two kernels around it.
//
// One or two rows with small factors take one launch (pool_small_kernel): every block works the thin product out for
// itself.  The others take three.
//
// What bounds those: the factors of every slot in use, read once (the rows of a slot go through them 16 at a time), and
// the launches' own starts and ends.  32 rows of 4096 x 14336 with 12 slots of rank 64 take 43.5 us, 21.6 for their bytes
// at the copy rate: 12 us down (2.5 for the plan, 2.5 to send, 2.5 until the first factors are there, 4.5 for the
// products), 20 the shared product, 10 up (6 of them for the pieces and thin out of L2).  The shared product's weights
// prefetched into L2 meanwhile made it 44 to 47.  Every block plans the rows by slot for itself and takes units of the
// plan in turn.  Both products run on the tensor cores in TF32 terms (the rows of a slot are the product's 16 rows): BF16
// and F16 factors are TF32 values already, Float32 factors and the activations are split into two terms, so the result
// keeps 22 bits; sums of 32 products are joined in Float32.  A lane reads whole 16-byte pieces of a factor's row: the
// order of the summed index within 32 is the lanes', the same in both operands.
//   1. down: thin[s][m][j] = x[m] . A_t[j] over the s-th stretch of K; beside it the shared product's own prologue, the
//      three BF16 terms of x, where the product takes the skinny tensor-core form;
//   2. the shared product, launched as a dependent (its weights stream in while the first kernel drains); where it takes
//      the vector form, it comes first and the first kernel runs beside it;
//   3. up: adds the stretches in order, multiplies by B_t; it also adds up the skinny form's pieces of the shared
//      product (or reads y), and the bias.  Its factors are read before it waits.
// Rows go through in blocks of 64, the skinny form's.
#include <algorithm>
#include <mutex>

#include "gemv.cuh"
#include "tc_common.cuh"
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

constexpr int DOWN_RANKS = 32;     // ranks of a unit of the first kernel
constexpr int DOWN_COLUMNS = 512;  // columns of it: 32 for each of 16 warps
constexpr int UP_COLUMNS = 256;    // outputs of a unit of the second
constexpr int MAX_RANK = 256;
constexpr int WINDOW = 64;         // rows of one launch
// Multiply-adds of thin that every block may repeat for one row, twice as many as for each of two.  One launch against
// three: 1 x 1536 x 576 rank 8 4.1 against 10.0 us, rank 64 8.5 against 10.9; 1 x 1024 x 4096 rank 16 (2^16) 9.1 against
// 12.2, rank 64 23 against 13; 2 x 576 x 576 rank 16 5.7 against 10.0, rank 56 11.9 against 10.9.
// A warp takes an output's whole row, so wide rows and many outputs lose: 1 x 64 x 16384 rank 4 23 against 16, 1 x 32000 x
// 512 rank 8 21 against 14.
constexpr int SMALL_WORK = 1 << 16, SMALL_INNER = 4096, SMALL_OUTPUTS = 2;  // outputs of a warp

// The launch's rows by slot: groups of up to 16 rows that name the same slot (or none).
struct Plan {
  int groups, widest;  // of them; most rows of one with a slot
  int slot[WINDOW];    // per group: -1 without a slot
  short rank[WINDOW], count[WINDOW], first[WINDOW];
  signed char rows[WINDOW][16];
  // (group, chunk of 32 ranks) pairs, and into how many parts each one's columns are split: as many as give every block
  // of the first kernel one (both kernels plan alike).
  int pairs, parts, per;  // per: stretches of 512 columns in a part
  signed char group_of[WINDOW * (MAX_RANK / DOWN_RANKS)];
};

// By the first warp alone, lane i for rows i and i + 32, in registers; short code that runs cold.  Ends with a barrier.
__device__ __forceinline__ void make_plan(const Pool &p, int M, int stretches, int blocks, Plan &s) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const uint32_t below = (1u << lane) - 1;
    int known[4];  // a small pool's ranks, on their way beside the rows' slots rather than behind them
    const bool small = p.slots <= 128;
#pragma unroll
    for (int k = 0; k < 4; k++) known[k] = small && k * 32 + lane < p.slots ? p.ranks[k * 32 + lane] : 0;
    int t[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      t[h] = -2;  // behind the last row
      if (h * 32 + lane < M) {
        t[h] = p.rows[h * 32 + lane];
        if (t[h] >= p.slots) *p.err = DEV_BAD_INDEX + 2;
        if (t[h] < 0 || t[h] >= p.slots) t[h] = -1;
      }
    }
    uint64_t same[2] = {__match_any_sync(0xffffffffu, t[0]), (uint64_t)__match_any_sync(0xffffffffu, t[1]) << 32};
    if (M > 32) {
#pragma unroll 1
      for (int k = 0; k < 32; k++) {
        same[0] |= (uint64_t)(__shfl_sync(0xffffffffu, t[1], k) == t[0]) << (32 + k);
        same[1] |= (uint64_t)(__shfl_sync(0xffffffffu, t[0], k) == t[1]) << k;
      }
    }
    const int at[2] = {__popc((uint32_t)same[0] & below), __popcll(same[1] & ((1ull << (32 + lane)) - 1))};  // place among the slot's rows
    const uint64_t starts = __ballot_sync(0xffffffffu, t[0] != -2 && at[0] % 16 == 0) |
                            (uint64_t)__ballot_sync(0xffffffffu, t[1] != -2 && at[1] % 16 == 0) << 32;
    int chunks[2] = {0, 0}, group[2], widest = 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      uint64_t mine = same[h] & starts;  // its group starts at the (at / 16)-th of these
      for (int k = 0; k < at[h] / 16; k++) mine &= mine - 1;
      const int start = t[h] == -2 ? 0 : __ffsll((long long)mine) - 1;
      group[h] = __popcll(starts & ((1ull << start) - 1));
      int rank = 0;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int r = __shfl_sync(0xffffffffu, known[k], t[h] & 31);
        if (t[h] >= 0 && t[h] / 32 == k) rank = r;
      }
      if (!small && t[h] >= 0) rank = p.ranks[t[h]];
      rank = max(0, min(rank, p.max_rank));
      if (t[h] != -2) {
        s.rows[group[h]][at[h] % 16] = (signed char)(h * 32 + lane);
        if (at[h] % 16 == 0) {
          const int count = min(16, __popcll(same[h]) - at[h]);
          s.slot[group[h]] = t[h];
          s.rank[group[h]] = (short)rank;
          s.count[group[h]] = (short)count;
          if (t[h] >= 0) chunks[h] = (rank + DOWN_RANKS - 1) / DOWN_RANKS, widest = max(widest, count);
        }
      }
    }
    // pairs in the order of the rows that start their groups
    int before[2] = {chunks[0], chunks[1]};
#pragma unroll
    for (int off = 1; off < 32; off <<= 1)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int v = __shfl_up_sync(0xffffffffu, before[h], off);
        if (lane >= off) before[h] += v;
      }
    const int half = __shfl_sync(0xffffffffu, before[0], 31), pairs = half + __shfl_sync(0xffffffffu, before[1], 31);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if (!(starts >> (h * 32 + lane) & 1)) continue;
      const int from = before[h] - chunks[h] + (h ? half : 0);
      s.first[group[h]] = (short)from;
      for (int k = 0; k < chunks[h]; k++) s.group_of[from + k] = (signed char)group[h];
    }
    widest = __reduce_max_sync(0xffffffffu, widest);
    if (lane == 0) {
      s.groups = __popcll(starts);
      s.widest = widest;
      s.pairs = pairs;
      const int parts = max(1, min(stretches, blocks / max(1, pairs)));
      s.per = (stretches + parts - 1) / parts;
      s.parts = (stretches + s.per - 1) / s.per;
    }
  }
  __syncthreads();
}

// Eight neighbouring factor elements from index `at`, the first `live` of them at least (all of a piece that has one, with
// VEC: 16-byte loads).
template <int DTYPE, bool VEC>
struct Eight {
  uint4 raw[DTYPE == STB_F32 ? 2 : 1];

  __device__ __forceinline__ void load(const void *base, size_t at, int live) {
#pragma unroll
    for (int i = 0; i < (DTYPE == STB_F32 ? 2 : 1); i++) raw[i] = make_uint4(0, 0, 0, 0);
    if (VEC) {
      const uint4 *p = (const uint4 *)((const char *)base + at * (DTYPE == STB_F32 ? 4 : 2));
      if (live > 0) {
#pragma unroll
        for (int i = 0; i < (DTYPE == STB_F32 ? 2 : 1); i++) raw[i] = __ldg(p + i);
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
  // Zeros behind the first `live` elements, which may hold anything: at the use, a load would have to be waited for.
  __device__ __forceinline__ void trim(int live) {
    uint32_t *w = (uint32_t *)raw;
#pragma unroll
    for (int i = 0; i < (DTYPE == STB_F32 ? 8 : 4); i++) {
      if (DTYPE == STB_F32) w[i] = i < live ? w[i] : 0u;
      else w[i] = 2 * i + 1 < live ? w[i] : (2 * i < live ? w[i] & 0xffffu : 0u);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t *w = (const uint32_t *)raw;
    if constexpr (DTYPE == STB_F32) return __uint_as_float(w[i]);
    else if constexpr (DTYPE == STB_BF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __half2float(__ushort_as_half((uint16_t)(w[i / 2] >> (16 * (i & 1)))));
  }
};

// The terms of an activation: rounded beside Float32 factors, whose own are cut; beside exact factors nothing is left out.
template <int DTYPE>
__device__ __forceinline__ void split_row(float x, uint32_t &hi, uint32_t &lo) {
  if (DTYPE == STB_F32) split_tf32(x, hi, lo);
  else cut_tf32(x, hi, lo);
}

// c += x . f over eight elements of each lane: hi and lo are x's terms (rows g, g + 8 by element), f the factor's.
template <int DTYPE, typename E>
__device__ __forceinline__ void eight_products(float (&c)[4], const uint32_t (&hi)[4][4], const uint32_t (&lo)[4][4], const E &f) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float f0 = f.get(2 * j), f1 = f.get(2 * j + 1);
    if constexpr (DTYPE == STB_F32) {
      uint32_t h0, l0, h1, l1;
      cut_tf32(f0, h0, l0);
      cut_tf32(f1, h1, l1);
      product_tf32(c, hi[j], l0, l1);
      product_tf32(c, lo[j], h0, h1);
      product_tf32(c, hi[j], h0, h1);
    } else {
      product_tf32(c, lo[j], __float_as_uint(f0), __float_as_uint(f1));
      product_tf32(c, hi[j], __float_as_uint(f0), __float_as_uint(f1));
    }
  }
}

// The skinny form's terms x3 [3][NT][K] of four neighbouring values (zeros for rows M and behind).
__device__ __forceinline__ void write_terms(float4 v, uint16_t *x3, int m, int NT, int K, int k) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  uint16_t h[3][4];
#pragma unroll
  for (int e = 0; e < 4; e++) split3_bf16(f[e], h[0][e], h[1][e], h[2][e]);
#pragma unroll
  for (int i = 0; i < 3; i++) {
    uint2 u;
    u.x = (uint32_t)h[i][0] | ((uint32_t)h[i][1] << 16);
    u.y = (uint32_t)h[i][2] | ((uint32_t)h[i][3] << 16);
    *(uint2 *)(x3 + ((size_t)i * NT + m) * K + k) = u;
  }
}

template <int DTYPE>
struct Down {
  static constexpr int ESZ = DTYPE == STB_F32 ? 4 : 2;
  static constexpr int A_ROW = DOWN_COLUMNS * ESZ, X_ROW = DOWN_COLUMNS * 4;
  static constexpr int RING = 196608, SMEM = RING + 16 * 16 * DOWN_RANKS * 4;  // the stretches' slots, then the warps' sums
  static_assert(RING / (DOWN_RANKS * A_ROW + 16 * X_ROW) >= 2 && SMEM + sizeof(Plan) <= 232448, "shared memory");
};

__device__ __forceinline__ void copy16_async(void *dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(live ? 16 : 0)
               : "memory");
}

// thin[part][m][j] for all rows: units (pair of a group of rows and a chunk of 32 ranks, part of the columns), one block per
// SM and, where the plan can, one unit per block; with x3 the blocks also write the terms of x.  The factors come from
// memory that nothing has touched lately (2 to 3 us away, behind the shared product's weights), so a block sends for all
// that its shared memory holds (two to six stretches of 512 columns, by the rows of the widest group) before it waits.  VEC: x and A have
// rows of whole 16-byte pieces (plain loads otherwise).
template <int DTYPE, bool VEC>
__global__ void __launch_bounds__(512, 1) pool_down_kernel(const Pool p, const float *x, float *thin, int M, int K, int stretches,
                                                           uint16_t *x3, int terms_rows, bool behind) {
  using D = Down<DTYPE>;
  constexpr int NT = DOWN_RANKS / 8, ESZ = D::ESZ;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Plan s_plan;
  float(*s_sum)[16][DOWN_RANKS] = (float(*)[16][DOWN_RANKS])(smem + D::RING);  // row r turned by 8 (r & 3)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  if (!behind) pdl_wait();
  pdl_trigger();  // after the wait: what starts early may read weights and factors at once
  make_plan(p, M, stretches, gridDim.x, s_plan);
  const int units = s_plan.pairs * s_plan.parts, per = s_plan.per;
  const int slot_bytes = DOWN_RANKS * D::A_ROW + s_plan.widest * D::X_ROW, slots = D::RING / slot_bytes;

  // 16-byte chunk c of row r: XORed so that the chunks that eight rows read at once lie in different banks.
  auto a_at = [&](uint8_t *slot, int r, int c) {
    return slot + r * D::A_ROW + ((c ^ (ESZ == 4 ? r & 7 : (r & 1) << 2 | (r >> 1 & 3))) << 4);
  };
  auto x_at = [&](uint8_t *slot, int r, int c) { return slot + DOWN_RANKS * D::A_ROW + r * D::X_ROW + ((c ^ (r & 7)) << 4); };
  // One stretch s of unit u, and the next one to send for.
  int ahead = blockIdx.x, ahead_s = 0;
  auto send = [&](uint8_t *slot) {
    if (ahead < units) {
      const int pair = ahead / s_plan.parts, e = s_plan.group_of[pair], j0 = (pair - s_plan.first[e]) * DOWN_RANKS;
      const int s0 = ahead % s_plan.parts * per, s = s0 + ahead_s;
      const int live = min(DOWN_RANKS, (int)s_plan.rank[e] - j0), rows = (live + 7) / 8 * 8, k0 = s * DOWN_COLUMNS;
      const size_t base = ((size_t)s_plan.slot[e] * p.max_rank + j0) * K + k0;
      if (++ahead_s == per || s + 1 == stretches) {
        ahead_s = 0;
        ahead += gridDim.x;
      }
      constexpr int AC = D::A_ROW / 16, XC = D::X_ROW / 16, PER = 16 / ESZ;
      for (int i = threadIdx.x; i < rows * AC; i += 512) {
        const int r = i / AC, c = i % AC, k = c * PER;
        if (VEC) {
          const bool in = r < live && k0 + k < K;
          copy16_async(a_at(slot, r, c), (const uint8_t *)p.a + (base + (in ? (size_t)r * K + k : 0)) * ESZ, in);
        } else {
          uint8_t *to = a_at(slot, r, c);
          for (int h = 0; h < PER; h++) {
            const bool in = r < live && k0 + k + h < K;
            if (ESZ == 4) ((uint32_t *)to)[h] = in ? ((const uint32_t *)p.a)[base + (size_t)r * K + k + h] : 0u;
            else ((uint16_t *)to)[h] = in ? ((const uint16_t *)p.a)[base + (size_t)r * K + k + h] : (uint16_t)0;
          }
        }
      }
      for (int i = threadIdx.x; i < s_plan.count[e] * XC; i += 512) {
        const int r = i / XC, c = i % XC, k = c * 4;
        const float *from = x + (size_t)s_plan.rows[e][r] * K + k0;
        if (VEC) {
          copy16_async(x_at(slot, r, c), from + (k0 + k < K ? k : 0), k0 + k < K);
        } else {
          for (int h = 0; h < 4; h++) ((float *)x_at(slot, r, c))[h] = k0 + k + h < K ? from[k + h] : 0.0f;
        }
      }
    }
  };

  auto send_all = [&](int n) {  // the next n stretches, into the first slots
#pragma unroll 1
    for (int i = 0; i < n; i++) send(smem + i * slot_bytes);
  };
  if ((int)blockIdx.x < units) send_all(min(slots, min(per, stretches - (int)blockIdx.x % s_plan.parts * per)));
  if (x3) {
    const int quads = K / 4, all = terms_rows * quads, step = gridDim.x * 512;
    for (int i = blockIdx.x * 512 + threadIdx.x; i < all; i += 2 * step) {  // two in flight
      float4 v[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int e = i + h * step;
        v[h] = e < M * quads ? *(const float4 *)(x + (size_t)e * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int e = i + h * step;
        if (e < all) write_terms(v[h], x3, e / quads, terms_rows, K, e % quads * 4);
      }
    }
  }
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int pair = unit / s_plan.parts, part = unit % s_plan.parts, e = s_plan.group_of[pair];
    const int j0 = (pair - s_plan.first[e]) * DOWN_RANKS, rank = s_plan.rank[e] - j0, count = s_plan.count[e];
    float acc[NT][4] = {};
    const int end = min(per, stretches - part * per);
#pragma unroll 1
    for (int done = 0; done < end; done += slots) {  // what the slots hold, and then the next of it
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < min(slots, end - done); i++) {
        uint8_t *slot = smem + i * slot_bytes;
        uint32_t hi[4][4], lo[4][4];  // the rows' eight values of this lane, in both terms
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int r = g + 8 * h;
          const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          const float4 u = r < count ? *(const float4 *)x_at(slot, r, warp * 8 + t4 * 2) : zero;
          const float4 v = r < count ? *(const float4 *)x_at(slot, r, warp * 8 + t4 * 2 + 1) : zero;
          const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 2; i++) split_row<DTYPE>(f[2 * j + i], hi[j][2 * i + h], lo[j][2 * i + h]);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          Eight<DTYPE, true> f;  // ranks behind the last hold anything, and go nowhere
#pragma unroll
          for (int i = 0; i < ESZ / 2; i++) f.raw[i] = *(const uint4 *)a_at(slot, n * 8 + g, (warp * 4 + t4) * (ESZ / 2) + i);
          float c[4] = {};
          eight_products<DTYPE>(c, hi, lo, f);
#pragma unroll
          for (int i = 0; i < 4; i++) acc[n][i] += c[i];
        }
      }
      __syncthreads();  // the slots have been read
      const int left = end - done - slots;
      if (left > 0) send_all(min(slots, left));
      else if (unit + gridDim.x < units) send_all(min(slots, min(per, stretches - (unit + (int)gridDim.x) % s_plan.parts * per)));
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) s_sum[warp][g + 8 * (i >> 1)][(n * 8 + 2 * t4 + (i & 1) + 8 * (g & 3)) & 31] = acc[n][i];
    __syncthreads();
    float v = 0.0f;  // a warp per row, a lane per rank
#pragma unroll
    for (int w = 0; w < 16; w++) v += s_sum[w][warp][(lane + 8 * (warp & 3)) & 31];
    if (warp < count && lane < rank) thin[((size_t)part * M + s_plan.rows[e][warp]) * p.max_rank + j0 + lane] = v;
    __syncthreads();
  }
  if (behind) pdl_wait();  // the third kernel waits for this one alone: the shared product has to be done by then
}

// y[m][n] = base + scale_t thin[m] . B_t[n] + bias[n]: units (group of rows, 256 columns) in turn over the blocks;
// `stretches` partial sums of thin.  base: the skinny form's pieces (PIECES), or y itself, its bias already in.  VEC: B has
// rows of whole 16-byte pieces.
template <int DTYPE, bool VEC, bool PIECES>
__global__ void __launch_bounds__(256, DTYPE == STB_F32 ? 1 : 2) pool_up_kernel(const Pool p, const float *thin, float *y, int M,
                                                                               int N, int stretches, int down_blocks, const SkinnyParts parts,
                                                                               const float *bias) {
  constexpr int NT = UP_COLUMNS / 64;  // 8-column results of a warp
  __shared__ float s_thin[16][MAX_RANK + 4];
  __shared__ Plan s_plan;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  pdl_trigger();
  make_plan(p, M, stretches, down_blocks, s_plan);
  const int groups = s_plan.groups, columns = (N + UP_COLUMNS - 1) / UP_COLUMNS;
  bool waited = false;
  for (int u = blockIdx.x; u < groups * columns; u += gridDim.x) {
    const int e = u % groups, t = s_plan.slot[e], rank = s_plan.rank[e], count = s_plan.count[e];
    const int n0 = u / groups * UP_COLUMNS + warp * (UP_COLUMNS / 8);
    if (!PIECES && rank == 0) continue;
    const int blocks = (rank + 31) / 32;  // of 32 ranks
    const float scale = t >= 0 ? p.scales[t] : 0.0f;
    const int wide = blocks * 32;
    Eight<DTYPE, VEC> f[2][NT];  // of 32 ranks each: the first 64 are read before the wait
    auto read = [&](int kb, Eight<DTYPE, VEC> (&f)[NT]) {
      const int j = kb * 32 + t4 * 8;
#pragma unroll
      for (int n = 0; n < NT; n++)
        f[n].load(p.b, ((size_t)t * N + n0 + n * 8 + g) * p.max_rank + j, n0 + n * 8 + g < N ? min(8, rank - j) : 0);
    };
    if (rank) {
      read(0, f[0]);
      read(1, f[1]);
    }
    // pieces of the tile of 128 columns that this warp's 32 lie in
    int pieces = 0;
    const float *at_piece = nullptr;
    if (PIECES && n0 < N) {
      const int tile = n0 / 128;
      pieces = skinny_cta_of((long long)(tile + 1) * parts.kbs - 1, parts.T, parts.G) -
               skinny_cta_of((long long)tile * parts.kbs, parts.T, parts.G) + 1;
      at_piece = parts.part + (size_t)tile * parts.pmax * parts.M * 128 + n0 % 128 + 2 * t4;
    }
    if (!waited) pdl_wait();  // thin, and the shared product
    waited = true;
    // thin's first parts for this warp's first 32 ranks, on their way together with the pieces
    auto thin_at = [&](int i) { return thin + (size_t)s_plan.rows[e][i / wide] * p.max_rank + i % wide + lane; };
    auto thin_in = [&](int i) { return i < count * wide && i % wide + lane < rank; };
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; k++)
      w[k] = thin_in(warp * 32) && k < s_plan.parts ? __ldcg(thin_at(warp * 32) + (size_t)k * M * p.max_rank) : 0.0f;
    float2 base[2][NT];
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int n = 0; n < NT; n++) base[h][n] = make_float2(0.0f, 0.0f);
      if (g + 8 * h >= count) continue;
      const int r = s_plan.rows[e][g + 8 * h];
      if (PIECES) {
        for (int i = 0; i < pieces; i += 4) {  // four on their way at a time
          float2 v[4][NT];
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int n = 0; n < NT; n++)
              v[k][n] = i + k < pieces ? __ldcg((const float2 *)(at_piece + ((size_t)(i + k) * parts.M + r) * 128 + n * 8)) : make_float2(0.0f, 0.0f);
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
              base[h][n].x += v[k][n].x;
              base[h][n].y += v[k][n].y;
            }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const int col = n0 + n * 8 + 2 * t4;
          if (col < N) base[h][n].x = y[(size_t)r * N + col];
          if (col + 1 < N) base[h][n].y = y[(size_t)r * N + col + 1];
        }
      }
    }
    for (int i = warp * 32; i < count * wide; i += 256) {  // 32 ranks of one row
      float v = 0.0f;
      if (i == warp * 32) {
#pragma unroll
        for (int k = 0; k < 8; k++) v += w[k];
      }
      for (int s = i == warp * 32 ? 8 : 0; s < s_plan.parts; s += 8) {
        float u[8];
#pragma unroll
        for (int k = 0; k < 8; k++) u[k] = thin_in(i) && s + k < s_plan.parts ? __ldcg(thin_at(i) + (size_t)(s + k) * M * p.max_rank) : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) v += u[k];
      }
      s_thin[i / wide][i % wide + lane] = v;
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
          split_row<DTYPE>(g < count ? s_thin[g][at] : 0.0f, hi[j][2 * i], lo[j][2 * i]);
          split_row<DTYPE>(g + 8 < count ? s_thin[g + 8][at] : 0.0f, hi[j][2 * i + 1], lo[j][2 * i + 1]);
        }
      const int live = rank - (kb * 32 + t4 * 8);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        if (VEC && live < 8) f[0][n].trim(live);
        float c[4] = {};
        eight_products<DTYPE>(c, hi, lo, f[0][n]);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] += c[i];
        f[0][n] = f[1][n];
      }
      if (kb + 2 < blocks) read(kb + 2, f[1]);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if (g + 8 * h >= count) continue;
      float *to = y + (size_t)s_plan.rows[e][g + 8 * h] * N;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int col = n0 + n * 8 + 2 * t4 + i;
          if (col >= N) continue;
          float v = i ? base[h][n].y : base[h][n].x;
          if (rank) v += scale * acc[n][2 * h + i];
          if (PIECES && bias) v += bias[col];
          to[col] = v;
        }
    }
    __syncthreads();  // before thin's sums are replaced
  }
  if (!waited) pdl_wait();  // what waits for this kernel has to find the ones before it done, too
}

// Few rows of a product that a warp per output takes anyway, with factors small enough that every block works out all of
// thin for itself: one launch.  Float32 FMAs; a lane's eight neighbouring elements at a time, four such pieces on their
// way together, those of the first output sent for before anything is known of the rows' slots.
template <typename WT, int DTYPE, int MT>
__global__ void __launch_bounds__(256) pool_small_kernel(const Pool p, const float *x, const uint16_t *w, const float *bias, float *y,
                                                         int M, int N, int K, int per) {
  constexpr int PIECE = DTYPE == STB_F32 ? 2 : 1, BATCH = 4, THIN = 4 / PIECE;  // loads of a factor's piece; a warp's pieces of 256 at a time
  __shared__ float s_thin[MT][MAX_RANK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = (blockIdx.x * 8 + warp) * per;
  auto weights = [&](uint4 (&u)[BATCH], int n, int k0) {
#pragma unroll
    for (int i = 0; i < BATCH; i++) {
      const int k = k0 + i * 256 + lane * 8;
      u[i] = n < N && k < K ? ld_stream_u4(w + (size_t)n * K + k) : make_uint4(0, 0, 0, 0);
    }
  };
  pdl_wait();
  pdl_trigger();
  uint4 first[BATCH];
  weights(first, n0, 0);
  int t = -1, rank = 0;  // of row `lane`
  float scale = 0.0f;
  if (lane < M) {
    t = p.rows[lane];
    if (t >= p.slots) *p.err = DEV_BAD_INDEX + 2;
    if (t < 0 || t >= p.slots) t = -1;
    if (t >= 0) {
      rank = max(0, min(p.ranks[t], p.max_rank));
      scale = p.scales[t];
    }
  }
  auto b_at = [&](int n, int m, int j) {  // the m-th row's factor of output n, rank j
    const size_t i = ((size_t)max(0, __shfl_sync(0xffffffffu, t, m)) * N + n) * p.max_rank + j;
    const bool in = n < N && j < __shfl_sync(0xffffffffu, rank, m);
    if (DTYPE == STB_F32) return in ? ((const float *)p.b)[i] : 0.0f;
    const uint16_t u = in ? ((const uint16_t *)p.b)[i] : (uint16_t)0;
    return DTYPE == STB_BF16 ? widen1<__nv_bfloat16>(u) : widen1<__half>(u);
  };
  float b[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) b[m] = m < M ? b_at(n0, m, lane) : 0.0f;
  auto at_x = [&](int m, int k, bool half) { return k < K ? *(const float4 *)(x + (size_t)m * K + k + half * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f); };
  // thin: a warp per (row, rank)
  int turn = warp;
#pragma unroll 1
  for (int m = 0; m < M; m++) {
    const int r = __shfl_sync(0xffffffffu, rank, m), slot = __shfl_sync(0xffffffffu, t, m);
#pragma unroll 1
    for (int j = turn; j < r; j += 16) {  // ranks j and j + 8
      const size_t row = ((size_t)slot * p.max_rank + j) * K;
      float v[2] = {};
#pragma unroll 1
      for (int k0 = 0; k0 < K; k0 += THIN * 256) {
        uint4 u[2][THIN][PIECE];
        float4 f[THIN][2];
#pragma unroll
        for (int i = 0; i < THIN; i++) {
          const int k = k0 + i * 256 + lane * 8;
#pragma unroll
          for (int q = 0; q < 2; q++)
#pragma unroll
            for (int h = 0; h < PIECE; h++)
              u[q][i][h] = k < K && j + q * 8 < r ? *(const uint4 *)((const uint8_t *)p.a + (row + (size_t)q * 8 * K + k) * (PIECE * 2) + h * 16)
                                                  : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int h = 0; h < 2; h++) f[i][h] = at_x(m, k, h);
        }
#pragma unroll
        for (int i = 0; i < THIN; i++)
#pragma unroll
          for (int q = 0; q < 2; q++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              float2 c, d;
              if constexpr (DTYPE == STB_F32) {
                const uint4 e = u[q][i][h];
                c = make_float2(__uint_as_float(e.x), __uint_as_float(e.y));
                d = make_float2(__uint_as_float(e.z), __uint_as_float(e.w));
              } else {
                using T = std::conditional_t<DTYPE == STB_BF16, __nv_bfloat16, __half>;
                c = widen2<T>(h ? u[q][i][0].z : u[q][i][0].x);
                d = widen2<T>(h ? u[q][i][0].w : u[q][i][0].y);
              }
              v[q] = fmaf(f[i][h].x, c.x, fmaf(f[i][h].y, c.y, fmaf(f[i][h].z, d.x, fmaf(f[i][h].w, d.y, v[q]))));
            }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
#pragma unroll
        for (int q = 0; q < 2; q++) v[q] += __shfl_xor_sync(0xffffffffu, v[q], off);
      if (lane < 2 && j + lane * 8 < r) s_thin[m][j + lane * 8] = lane ? v[1] : v[0];
    }
    turn = (turn - r) & 7;  // the next row's ranks go on where these end
  }
  __syncthreads();
#pragma unroll 1
  for (int o = 0; o < per; o++) {
    const int n = n0 + o;
    if (n >= N) break;
    float acc[MT] = {};
#pragma unroll 1
    for (int k0 = 0; k0 < K; k0 += BATCH * 256) {
      uint4 u[BATCH];
      if (o == 0 && k0 == 0) {
#pragma unroll
        for (int i = 0; i < BATCH; i++) u[i] = first[i];
      } else {
        weights(u, n, k0);
      }
#pragma unroll
      for (int m = 0; m < MT; m++) {
        if (m >= M) continue;
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
          const int k = k0 + i * 256 + lane * 8;
          const float4 e = at_x(m, k, false), f = at_x(m, k, true);
          const float2 c0 = widen2<WT>(u[i].x), c1 = widen2<WT>(u[i].y), c2 = widen2<WT>(u[i].z), c3 = widen2<WT>(u[i].w);
          acc[m] = fmaf(e.x, c0.x, fmaf(e.y, c0.y, fmaf(e.z, c1.x, fmaf(e.w, c1.y, acc[m]))));
          acc[m] = fmaf(f.x, c2.x, fmaf(f.y, c2.y, fmaf(f.z, c3.x, fmaf(f.w, c3.y, acc[m]))));
        }
      }
    }
    float out = 0.0f;
#pragma unroll
    for (int m = 0; m < MT; m++) {
      if (m >= M) continue;
      const int r = __shfl_sync(0xffffffffu, rank, m);
      float v = 0.0f;
      if (lane < r) v = s_thin[m][lane] * b[m];
      for (int j0 = 32; j0 < r; j0 += 32) {
        const float more = b_at(n, m, j0 + lane);
        if (j0 + lane < r) v = fmaf(s_thin[m][j0 + lane], more, v);
      }
      const float by = __shfl_sync(0xffffffffu, scale, m);
      v = r ? fmaf(by, v, acc[m]) : acc[m];
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (lane == m) out = v;
      if (o + 1 < per) b[m] = b_at(n + 1, m, lane);
    }
    if (lane < M) y[(size_t)lane * N + n] = out + (bias ? bias[n] : 0.0f);
  }
}

template <int DTYPE, bool VEC>
void launch_down(stb_session *s, int grid, const Pool &p, const float *x, float *thin, int M, int K, int stretches,
                 uint16_t *x3, int terms_rows, bool behind) {
  constexpr int SMEM = Down<DTYPE>::SMEM;
  {
    static std::mutex mu;
    static bool configured[64] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (s->device < 0 || s->device >= 64 || !configured[s->device]) {
      STB_CUDA(cudaFuncSetAttribute(pool_down_kernel<DTYPE, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
      if (s->device >= 0 && s->device < 64) configured[s->device] = true;
    }
  }
  launch_kernel(pool_down_kernel<DTYPE, VEC>, dim3(grid), dim3(512), (size_t)SMEM, s->stream, true, p, x, thin, M, K, stretches,
                x3, terms_rows, behind);
}

template <typename F>
void dispatch_pool(int dtype, F &&f) {
  if (dtype == STB_F32) f(std::integral_constant<int, STB_F32>());
  else if (dtype == STB_BF16) f(std::integral_constant<int, STB_BF16>());
  else f(std::integral_constant<int, STB_F16>());
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
    p.err = session_error_word(s);
    const int chunks = (p.max_rank + DOWN_RANKS - 1) / DOWN_RANKS, most = std::min(M, WINDOW);
    const int stretches = (K + DOWN_COLUMNS - 1) / DOWN_COLUMNS, columns = (N + UP_COLUMNS - 1) / UP_COLUMNS;
    STB_REQUIRE((int64_t)WINDOW * stretches * chunks <= 0x7fffffff && (int64_t)WINDOW * columns <= 0x7fffffff, "adapted Linear too large");
    const int sms = tc::sm_count(s->device), resident = (pool->dtype == STB_F32 ? 1 : 2) * sms;  // blocks of `up` at once
    auto tensor_cores = [&](int m) { return m > 0 && skinny_eligible(m, N, K, w_dtype, (const void *)w); };
    const bool skinny = K % 8 == 0 && x % 16 == 0 && (tensor_cores(M) || tensor_cores(most) || tensor_cores(M % WINDOW));
    const bool vec_down = K % 8 == 0 && x % 16 == 0 && pool->a % 16 == 0;
    if (!skinny && vec_down && w % 16 == 0 && w_dtype != STB_F32 && M <= 2 && K <= SMALL_INNER &&
        N <= sms * 16 * SMALL_OUTPUTS && (int64_t)M * M * p.max_rank * K <= SMALL_WORK) {
      p.rows = (const int *)rows;
      const int per = (N + sms * 16 - 1) / (sms * 16);
      auto small = [&](auto wt, auto type) {
        using WT = decltype(wt);
        constexpr int DT = decltype(type)::value;
        launch_kernel(M == 1 ? pool_small_kernel<WT, DT, 1> : pool_small_kernel<WT, DT, 2>,
                      dim3((N + per * 8 - 1) / (per * 8)), dim3(256), 0, s->stream, true, p, (const float *)x, (const uint16_t *)w,
                      (const float *)bias, (float *)y, M, N, K, per);
      };
      dispatch_pool(pool->dtype, [&](auto type) {
        if (w_dtype == STB_BF16) small(__nv_bfloat16(), type);
        else small(__half(), type);
      });
      count_launch(s);
      return;
    }
    // The partial sums lie behind the shared product's own scratch.
    const uint64_t base = ((skinny ? skinny_scratch_bytes(M, N, K, s->device) : 0) + 255) & ~255ull;
    const uint64_t scratch = session_scratch(s, base + (uint64_t)stretches * most * p.max_rank * sizeof(float));
    float *thin = (float *)(scratch + base);
    const bool vec_up = p.max_rank % 8 == 0 && pool->b % 16 == 0;
    auto go = [&](auto type) {
      constexpr int DT = decltype(type)::value;
      for (int m0 = 0; m0 < M; m0 += WINDOW) {
        const int mb = std::min(WINDOW, M - m0), terms_rows = skinny ? skinny_nt(mb) : 0;
        const float *xb = (const float *)x + (size_t)m0 * K;
        float *yb = (float *)y + (size_t)m0 * N;
        uint16_t *terms = skinny ? (uint16_t *)scratch : nullptr;
        p.rows = (const int *)rows + m0;
        const int down_grid = skinny ? sms : (int)std::min<int64_t>(sms, (int64_t)mb * stretches * chunks);
        const int up_grid = (int)std::min<int64_t>(resident, (int64_t)mb * columns);
        if (!skinny) linear(s, (uint64_t)xb, K, w, w_dtype, bias, (uint64_t)yb, N, mb, N, K, true);
        if (vec_down) launch_down<DT, true>(s, down_grid, p, xb, thin, mb, K, stretches, terms, terms_rows, !skinny);
        else launch_down<DT, false>(s, down_grid, p, xb, thin, mb, K, stretches, terms, terms_rows, !skinny);
        SkinnyParts parts;
        if (skinny) {
          GemvParams g;
          g.x = xb;
          g.ldx = K;
          g.w = (const void *)w;
          g.M = mb;
          g.N = N;
          g.K = K;
          g.y = yb;
          g.ldy = N;
          g.pdl = true;
          count_launch(s, skinny_launch<EPI_PLAIN>(g, (void *)scratch, base, p.err, s->device, s->stream, terms, nullptr, &parts));
          launch_kernel(vec_up ? pool_up_kernel<DT, true, true> : pool_up_kernel<DT, false, true>, dim3(up_grid), dim3(256), 0,
                        s->stream, true, p, (const float *)thin, yb, mb, N, stretches, down_grid, parts, (const float *)bias);
        } else {
          launch_kernel(vec_up ? pool_up_kernel<DT, true, false> : pool_up_kernel<DT, false, false>, dim3(up_grid), dim3(256), 0,
                        s->stream, true, p, (const float *)thin, yb, mb, N, stretches, down_grid, parts, (const float *)bias);
        }
        count_launch(s, 2);
      }
    };
    dispatch_pool(pool->dtype, go);
  });
}
