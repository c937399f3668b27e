// Attention of one new token per request over its paged cache (stb_op_paged_attention):
//   y[b, h] = sum_j softmax_j(q[b, h] . k_j / sqrt(width)) v_j,   j < lengths[b],  h on kv head h / group,
// zeros where lengths[b] <= 0.
//
// What bounds it: every cached byte is read once per 8 query heads of its kv head (an item takes 8 at a time), with 4 flops
// per element and head: HBM, as long as the arithmetic keeps out of the way.  With 8 query heads on a kv head, Float32 FMAs
// would take 8 flops per BF16 byte (52 TFLOP/s at the copy rate of 6.5 TB/s, near the SM's FP32 peak) and twice that for
// E4M3, so both products run on the tensor cores (mma.sync, fed by each warp's own ring: with 8 columns there is no reuse that
// larger tiles could find), with Float32 accuracy kept by splitting the Float32 side into terms that the products take exactly:
//   * BF16 cache: q and p in three BF16 terms (24 bits);
//   * F16 and E4M3 cache (E4M3 widens to F16 exactly): two F16 terms (22 bits).  q after a power of two that puts the largest
//     of a head at 2^12 (22 bits of that largest one); weights after one per head that follows the tiles' largest, the
//     second term's times 2^12, in a sum of its own.  What both miss of weights 2^26 times lower than their tile's largest
//     is added in Float32, key by key, where the result is not large enough that those bits cannot count;
//   * F32 cache: both sides in two TF32 terms (q and p 23 bits, keys 22, values 21), without the product of the lower ones.
// The tensor core truncates its sums, so chains are kept short (at most 8 products) and joined by Float32 additions.
//
// Work: items (request, kv head, chunk of 8 query heads) are cut into tiles of 16 or 32 keys, all tiles in one line; each
// block takes an equal stretch of the line and each of its warps an equal stretch of that (lengths are known on
// the device only: a captured step is replayed with new ones).  A warp runs alone over its stretch, across items,
// with a ring of cp.async stages of its own: no block barrier until its end.  The cache is the 16-row operand of
// both products (keys, then dimensions, as rows), the 8 heads are the columns, a product per term: no row of the
// tensor core's tile is padding.  Maxima move only when a score passes them by 2^8, which one vote per tile sees.
// Items that a block covers only in part are joined first among its warps in shared memory, then by the last block to
// arrive, always in the order of the keys.  Few short items go to one block each, many to one warp each (no join at all),
// many of medium length to one block each as the line has them (none between blocks).
//
// Measured in a captured graph: 24 requests of up to 16384 BF16 tokens (8 kv heads of 128, 64 heads) 156 us = 6.1 TB/s, 0.94 of
// the copy rate; one request of 60001 E4M3 tokens 38 us = 3.3 TB/s (its stream runs at 6.2; the rest is the start and two joins);
// 8 requests of up to 544 E4M3 tokens 11.6 us; one of 33 tokens 5.0 us.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged.cuh"
#include "tc_common.cuh"
#include "tf32.cuh"

namespace stb {

namespace {

struct AttendArgs {
  const float *q;
  float *y;
  int64_t q_row, y_row;
  const int *lengths;
  int heads, group, batch, first;  // requests first .. first + batch - 1 of the call
  float scale_log2;                // log2(e) / sqrt(width)
  float *pieces;                   // per block: two of its own, then one per warp
  int *arrived;                    // per block and head, zero between calls
};

__device__ __forceinline__ int attend_length(const PagedView &c, const AttendArgs &a, int b) {
  const int n = a.lengths[b], most = c.blocks * c.page_size;
  if (n > most) *c.err = DEV_BAD_INDEX + 1;
  return max(0, min(n, most));
}

// ------------------------------------------------------------------ any width, alignment and type

// One block per (request, query head): its warps take keys in turn, a lane every 32nd dimension, Float32 FMAs.
// For caches whose rows are no multiple of 16 bytes or wider than 256: the cache goes through once per query head.
template <int DTYPE>
__global__ void __launch_bounds__(256) paged_attention_any_kernel(const PagedView c, const AttendArgs a) {
  constexpr int W = 8, D = 16;  // warps; dimensions of a lane (width <= 512)
  __shared__ float s_max[W], s_sum[W], s_acc[W][512];
  const int b = a.first + blockIdx.y, h = blockIdx.x, kvh = h / a.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
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
    const float now = fmaxf(top, dot), keep = top == now ? 1.0f : exp2f(top - now);
    const float p = dot == -INFINITY ? 0.0f : exp2f(dot - now);  // the maximum itself may be -inf still
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

// ------------------------------------------------------------------ rows of whole 16-byte chunks, width <= 256

constexpr int MAX_GRID = 160;
constexpr int DIRECT_TILES = 64;     // most tiles of an item that one block takes alone
constexpr int WHOLE_TILES = 8;       // most tiles of an item that one warp takes alone
// Most tiles of an item that one block takes alone where there are more items than blocks, and twice as many where there
// are half as many again: the blocks' stretches differ by up to an item, and none is joined between blocks.  256 items of
// up to 300 BF16 tokens 21.7 -> 15.6 us, 400 of up to 500 22.3 -> 17.5; 160 of 500 21.6 -> 19.6, of 1000 (63 tiles) 29.6
// against 32.8; 400 of 1000 51 -> 47.  F32 tiles of 16 keys reach the limit at half as many tokens; 160 items of 500 of them
// lose, 33.3 -> 37.5: some blocks take two items and most one.
constexpr int ROUND_TILES = 32;
constexpr int BLOCK_PIECES = 20800;  // floats of a block's pieces, at most: (2 + warps) of 8 heads x (width + 4)
constexpr int MAX_BATCH = 1024;      // requests of one launch (their prefix sums lie in shared memory)
constexpr float LAZY = 8.0f;         // a maximum moves only when a score passes it by 2^8
// F16 weights, in log2: a head's are put around P_SHIFT and stay there while none passes P_TOP and none is below P_LOW.  The rest
// behind the first term's 11 bits goes times 2^12: both terms together keep 22 bits from F16's smallest normal value on, 2^-14,
// 19 from P_LOW on, and are off by 2^-37 at most below.  Where that may count in a result (some sum so far is not 2^22 times
// what a tile could lose), what is missing is added in Float32.  Scores of a standard deviation of 1, 3 and 5 nats, 0.5 GiB of
// E4M3 of width 128: 109, 115 and 156 us; all low weights in Float32 113, 140 and 388; a second pass of the tensor cores for
// them 131, 139 and 176 (registers); looked at before the tile's products 112, 124 and 177.
constexpr float P_SHIFT = 8.0f, P_TOP = 15.0f, P_LOW = -18.0f, P_REST = 4096.0f;

// What two F16 terms miss of a weight.
__device__ __forceinline__ float missing(float w) {
  const float rest = w - __half2float(__float2half_rn(w));
  return rest - __half2float(__float2half_rn(rest * P_REST)) * (1.0f / P_REST);
}

template <int DTYPE, int WP>
struct Shape {
  static constexpr int ESZ = DTYPE == STB_F32 ? 4 : (DTYPE == STB_E4M3 ? 1 : 2);
  static constexpr int ROW = (WP == 96 ? 128 : WP) * ESZ;  // bytes of a key's row in shared memory
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int PAIRS = WP * ESZ / 32;     // pairs of them that the products take
  static constexpr int TK = ROW >= 256 ? 16 : 32; // keys of a tile: 8 KB where the width allows
  static constexpr int TILE = 2 * TK * ROW;       // keys and values of a tile
  // Warps and stages that fill about 192 KB.  With enough arithmetic per byte more warps are worth more than a second stage
  // for each: what one waits for, the others compute over.  0.5 GiB of cache, 82 us at the copy rate: E4M3 of width 64
  // eight warps 165 us, twelve 136; F32 of width 128 six warps of two stages 119, twelve of one 102; F32 of width 256 three of
  // two 268, six of one 178 (each before the weights' range below and the cut TF32 terms: 143, 100 and 174 now).  BF16 and
  // F16 of width 64 and 128 take 93 to 97 with eight, E4M3 of width 128 120 with eight and 109 with twelve.
  static constexpr int WARPS = TILE <= 8192 ? (DTYPE == STB_E4M3 && ROW <= 128 ? 12 : 8) : (DTYPE == STB_F32 && ROW == 512 ? 12 : 6);
  static constexpr int STAGES = 196608 / (WARPS * TILE) < 6 ? 196608 / (WARPS * TILE) : 6;
  static constexpr int META = 16 + (DTYPE == STB_E4M3 ? TK * 8 : 0);  // per stage: valid mask, scales of keys and values
  static constexpr bool META_SCALES = DTYPE == STB_E4M3;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int RING = WARPS * STAGES * TILE;
  static constexpr int PART = 8 * (WP + 4);       // floats of a partial result: per head max, weight max, sum, -, values
  static constexpr int SMEM = RING + WARPS * STAGES * META + (2 * MAX_BATCH + 4) * 4;
  static_assert(STAGES >= 1 && (STAGES > 1 || !META_SCALES) && SMEM + 1024 <= 232448, "shared memory per block");
  static_assert(STAGES * TILE >= PART * 4, "a warp's last part reuses its ring");
  static_assert((2 + WARPS) * PART <= BLOCK_PIECES, "workspace");
};

__device__ __forceinline__ uint32_t shared_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes of global memory to shared memory; the second form writes zeros instead where `live` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// 2^x, at most 2 steps of Float32 off; results below 2^-126 are 0.
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void load_matrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void load_matrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Transpose of an 8 x 8 matrix of 16-bit elements, two neighbours of row lane / 4 per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// c += a . b, 16 x 8 results; a 16 x 16 (BF16, F16) or 16 x 8 (F32 taken as TF32).
template <int DTYPE>
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DTYPE == STB_F32)
    product_tf32(c, a, b0, b1);
  else if constexpr (DTYPE == STB_BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Three BF16 terms of two values: rounded, rest rounded, rest rounded (rests are exact).
__device__ __forceinline__ void split3_pair(float x, float y, uint32_t (&t)[3]) {
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    t[i] = *reinterpret_cast<const uint32_t *>(&h);
    x -= __uint_as_float(t[i] << 16);
    y -= __uint_as_float(t[i] & 0xffff0000u);
  }
}
// Two F16 terms, the second times `up`.
__device__ __forceinline__ void split2_pair(float x, float y, uint32_t (&t)[2], float up = 1.0f) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn((x - f.x) * up, (y - f.y) * up);
  t[0] = *reinterpret_cast<const uint32_t *>(&h);
  t[1] = *reinterpret_cast<const uint32_t *>(&l);
}

__device__ __forceinline__ uint32_t widen_pair(uint32_t two_bytes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two_bytes, __NV_E4M3);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Shared-memory address of 16-byte chunk `chunk` of row `row`: 128-byte lines whose chunks are XORed with the line, so
// that the same chunk of eight neighbouring rows lies in eight different places of a line (no bank conflict).
template <int ROW>
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, int row, int chunk) {
  if constexpr (ROW >= 128) return base + row * ROW + ((chunk ^ (row & 7)) << 4);
  const int line = row * ROW / 128, at = (row * ROW % 128) / 16 + chunk;
  return base + line * 128 + ((at ^ (line & 7)) << 4);
}

// `total` tiles cut into `parts` stretches whose lengths differ by one at most: where a stretch begins, and whose tile i is.
__device__ __forceinline__ int stretch_start(int k, int total, int parts) {
  return k * (total / parts) + min(k, total % parts);
}
__device__ __forceinline__ int stretch_of(int i, int total, int parts) {
  const int q = total / parts, r = total % parts;
  return i < r * (q + 1) ? i / (q + 1) : r + (i - r * (q + 1)) / q;
}
// The blocks' stretches: the whole line's tiles, or each item's, cut among `blocks` of them.
struct Line {
  int tiles, blocks;
  __device__ __forceinline__ int start(int k) const { return k / blocks * tiles + stretch_start(k % blocks, tiles, blocks); }
  __device__ __forceinline__ int of(int i) const { return i / tiles * blocks + stretch_of(i % tiles, tiles, blocks); }
};

// A place on the line of tiles.
struct Cursor {
  int b, item, tile, tiles, n;  // request, its item (kv head * chunks + chunk), tile of the item, tiles and keys of the request
};

template <int DTYPE, int WP>
__global__ void __launch_bounds__(Shape<DTYPE, WP>::THREADS, 1) paged_attention_kernel(const PagedView c, const AttendArgs a) {
  using S = Shape<DTYPE, WP>;
  constexpr int TK = S::TK, MB = TK / 16;          // keys of a tile, its 16-key results
  constexpr int STEP = DTYPE == STB_F32 ? 8 : 16;  // dimensions of one product
  constexpr int STEPS = WP / STEP, NT = WP / 16;
  constexpr int TERMS = DTYPE == STB_BF16 ? 3 : 2;  // of q and of the weights
  constexpr bool HALF = DTYPE == STB_F16 || DTYPE == STB_E4M3, SCALED = DTYPE == STB_E4M3;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *s_meta = smem + S::RING;
  int *s_start = (int *)(s_meta + S::WARPS * S::STAGES * S::META);  // tiles before request b, of one item each
  int *s_len = s_start + MAX_BATCH + 1;
  __shared__ int s_scan[S::WARPS], s_most[S::WARPS];
  __shared__ int s_part[2 * S::WARPS][4];  // a warp's first and last part: request (or -1), item, whether it starts / ends it

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunks_of = (a.group + 7) / 8, items = c.kv_heads * chunks_of;
  const int row_chunks = c.width * S::ESZ / 16, row_bytes = row_chunks * 16;

  for (int i = threadIdx.x; i < 2 * S::WARPS; i += S::THREADS) s_part[i][0] = -1;
  if (row_chunks < 2 * S::PAIRS) {  // chunks behind a key's row meet zeros of q: they must not hold NaNs (a value's go nowhere)
    const int behind = 2 * S::PAIRS - row_chunks;
    for (int i = threadIdx.x; i < S::WARPS * S::STAGES * TK * behind; i += S::THREADS) {
      const int row = i / behind;
      *(uint4 *)(smem + row / TK * S::TILE + chunk_at<S::ROW>(0, row % TK, row_chunks + i % behind)) = make_uint4(0, 0, 0, 0);
    }
  }

  pdl_wait();
  pdl_trigger();
  // The requests' lengths, the longest of them, and the sum of their tiles so far.
  const int per = (a.batch + S::THREADS - 1) / S::THREADS, b0 = threadIdx.x * per, b1 = min(a.batch, b0 + per);
  int own = 0, longest = 0;
  for (int b = b0; b < b1; b++) {
    const int n = attend_length(c, a, a.first + b);
    s_len[b] = n;
    own += (n + TK - 1) / TK;
    longest = max(longest, n);
  }
  int before = own;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += v;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) {
    s_scan[warp] = before;
    s_most[warp] = longest;
  }
  __syncthreads();
  for (int w = 0; w < S::WARPS; w++) {
    longest = max(longest, s_most[w]);
    if (w < warp) before += s_scan[w];
  }
  // Few short items: one block each, no line, nothing to join between blocks.
  const bool direct = a.batch * items <= (int)gridDim.x && longest <= DIRECT_TILES * TK;
  Cursor load, use;
  int total = 0, grid = 0, block0 = 0, t0, todo;
  Line line = {1, 1};
  if (direct) {
    if ((int)blockIdx.x >= a.batch * items) return;
    load.b = blockIdx.x / items;
    load.item = blockIdx.x % items;
    load.n = s_len[load.b];
    load.tiles = (load.n + TK - 1) / TK;
    if (load.n == 0) {
      for (int h = load.item % chunks_of * 8; h < min(a.group, (load.item % chunks_of + 1) * 8); h++)
        for (int i = threadIdx.x; i < c.width; i += S::THREADS)
          a.y[(a.first + load.b) * a.y_row + (size_t)(load.item / chunks_of * a.group + h) * c.width + i] = 0.0f;
      return;
    }
    const int warps = min(S::WARPS, (load.tiles + 1) / 2);  // two tiles cost less than a join
    t0 = stretch_start(min(warp, warps), load.tiles, warps);
    todo = stretch_start(min(warp + 1, warps), load.tiles, warps) - t0;
    load.tile = t0;
  } else {
    before -= own;
    for (int b = b0; b < b1; b++) {
      s_start[b] = before;
      before += (s_len[b] + TK - 1) / TK;
      if (b == a.batch - 1) s_start[a.batch] = before;
    }
    __syncthreads();
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x)  // zeros for the empty ones
      if (s_len[b] == 0)
        for (int i = threadIdx.x; i < a.heads * c.width; i += S::THREADS) a.y[(a.first + b) * a.y_row + i] = 0.0f;

    total = s_start[a.batch] * items;
    const bool whole = longest <= WHOLE_TILES * TK;  // short items, many of them: none is cut
    const bool rounded = !whole && longest <= (a.batch * items >= (int)gridDim.x * 3 / 2 ? 2 : 1) * ROUND_TILES * TK;  // none is cut between blocks
    grid = min((int)gridDim.x, whole ? total : (total + 2 * S::WARPS - 1) / (2 * S::WARPS));
    line = {total, grid};
    // One request: the same number of blocks for each of its items, if that idles few (no block then joins twice).
    if (a.batch == 1 && grid % items <= grid / 16) {
      grid -= grid % items;
      line = {total / items, grid / items};
    }
    if ((int)blockIdx.x >= grid) return;
    // The place of tile t: the last request that starts at or before it (the empty ones before that share its start).
    auto locate = [&](int t) {
      Cursor k;
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] * items <= t) lo = mid;
        else hi = mid - 1;
      }
      k.b = lo;
      k.tiles = s_start[lo + 1] - s_start[lo];
      k.n = s_len[lo];
      const int in = t - s_start[lo] * items;
      k.item = k.tiles ? in / k.tiles : 0;
      k.tile = k.tiles ? in - k.item * k.tiles : 0;
      return k;
    };
    auto next_item = [&](int t) {  // the first tile from t on that starts an item
      if (t >= total) return t;
      const Cursor k = locate(t);
      return k.tile ? t + k.tiles - k.tile : t;
    };
    int from = line.start(blockIdx.x), to = line.start(blockIdx.x + 1);
#pragma unroll 1
    for (int level = 0; level < 2; level++) {  // the block's stretch, then the warp's
      if (level) {
        const int mine = to - from;
        block0 = from;
        from = block0 + stretch_start(warp, mine, S::WARPS);
        to = block0 + stretch_start(warp + 1, mine, S::WARPS);
      }
      if (level ? whole : rounded) {
        from = next_item(from);
        to = next_item(to);
        if (!level && from == to) return;
      }
    }
    t0 = from;
    todo = to - from;
    load = locate(t0);
  }
  use = load;

  const uint32_t ring = shared_u32(smem) + warp * S::STAGES * S::TILE;
  uint8_t *meta = s_meta + warp * S::STAGES * S::META;
  auto advance = [&](Cursor &k) {
    if (++k.tile < k.tiles || direct) return;
    k.tile = 0;
    if (++k.item < items) return;
    k.item = 0;
    do k.b++;
    while (k.b < a.batch && s_len[k.b] == 0);
    if (k.b < a.batch) {
      k.tiles = s_start[k.b + 1] - s_start[k.b];
      k.n = s_len[k.b];
    }
  };

  // Copies of one tile: lane i looks up key i, then the warp copies whole rows, their addresses by shuffle.  The page of
  // the next tile's key is read one tile ahead, and scale bytes are stored one tile after they are read: neither waits
  // for memory here.
  constexpr int PER = 32 / S::CHUNKS > 0 ? 32 / S::CHUNKS : 1;      // rows of one copy of the warp
  constexpr int TIMES = S::CHUNKS > 32 ? S::CHUNKS / 32 : 1;        // copies of one row
  const int my_key = lane % TK, my_row = TIMES == 1 ? lane / S::CHUNKS : 0, my_chunk = TIMES == 1 ? lane % S::CHUNKS : lane;
  const uint8_t *const from[2] = {(const uint8_t *)c.kv[0] + my_chunk * 16, (const uint8_t *)c.kv[1] + my_chunk * 16};
  const int page_shift = (c.page_size & (c.page_size - 1)) == 0 ? 31 - __clz(c.page_size) : -1;
  auto page_ahead = [&](bool live) {
    const int key = load.tile * TK + my_key;
    if (!live || key >= load.n) return -1;
    return c.tables[(size_t)(a.first + load.b) * c.blocks + (page_shift >= 0 ? key >> page_shift : key / c.page_size)];
  };
  int issued = 0, page = page_ahead(todo > 0);
  int key_scale = 0, value_scale = 0;
  float2 *scales_to = nullptr;
  auto issue = [&](int stage) {
    if (SCALED && scales_to) {
      *scales_to = make_float2(scale_of((uint8_t)key_scale), (float)(value_scale - 127));
      scales_to = nullptr;
    }
    if (issued < todo) {
      const int key = load.tile * TK + my_key, kvh = chunks_of == 1 ? load.item : load.item / chunks_of;
      bool live = key < load.n;
      if (live && (unsigned)page >= (unsigned)c.pages) {
        *c.err = DEV_BAD_INDEX;
        live = false;
      }
      const int slot = page_shift >= 0 ? key & (c.page_size - 1) : key % c.page_size;
      const int at = live ? (page * c.kv_heads + kvh) * c.page_size + slot : 0;
      const uint32_t mask = __ballot_sync(0xffffffffu, live);
      uint8_t *m = meta + stage * S::META;
      if (lane == 0) *(uint32_t *)m = mask;
      if (SCALED) {
        key_scale = live ? c.scale[0][at] : 127;
        value_scale = live ? c.scale[1][at] : 127;
        scales_to = (float2 *)(m + 16) + my_key;
      }
      const uint32_t dst = ring + stage * S::TILE;
      auto copy = [&](auto all) {
#pragma unroll
        for (int r0 = 0; r0 < TK; r0 += PER) {
          const int r = r0 + my_row;
          const size_t off = (size_t)(uint32_t)__shfl_sync(0xffffffffu, at, r) * row_bytes;
#pragma unroll
          for (int side = 0; side < 2; side++)
#pragma unroll
            for (int i = 0; i < TIMES; i++)
              if (S::CHUNKS == 1 || my_chunk + i * 32 < row_chunks) {
                const uint32_t to = chunk_at<S::ROW>(dst + side * TK * S::ROW, r, my_chunk + i * 32);
                if (decltype(all)::value) copy16(to, from[side] + off + i * 512);
                else copy16(to, from[side] + off + i * 512, mask >> r & 1);
              }
        }
      };
      if (mask == 0xffffffffu) copy(std::true_type());
      else copy(std::false_type());
      const int item = load.item, b = load.b;
      advance(load);
      issued++;
      if ((load.item != item || load.b != b) && issued < todo) {  // the next item's q to L1, ahead of its use
        const int chunk = load.item % chunks_of;
        const float *row = a.q + (a.first + load.b) * a.q_row + (size_t)(load.item / chunks_of * a.group + chunk * 8) * c.width;
        for (int i = lane * 32; i < min(8, a.group - chunk * 8) * c.width; i += 1024)
          asm volatile("prefetch.global.L1 [%0];" ::"l"(row + i));
      }
      page = page_ahead(issued < todo);
    }
    copy_commit();
  };

  uint32_t q[STEPS][2 * TERMS];
  float o[NT][4], m1[2], m2[2], sum[2], unscale[2] = {1.0f, 1.0f};
  float base[2], down[2];  // F16 weights are 2^(score - base); `down` takes them to the scale of o, 2^P_SHIFT at m2

  // q of the item at `use` into registers: dimensions of this lane in step s, two pairs (F32: two single ones).
  constexpr int N = DTYPE == STB_F32 ? 2 : 4;
  auto load_query = [&]() {
    const int kvh = use.item / chunks_of, head = (use.item % chunks_of) * 8 + g;
    const bool live = head < a.group;
    const float *row = a.q + (a.first + use.b) * a.q_row + (size_t)(kvh * a.group + head) * c.width;
    auto dim = [&](int s, int i) {
      if (DTYPE == STB_F32) return s * 8 + t + 4 * i;
      if (SCALED) return s * 16 + 4 * t + i;
      return s * 16 + 2 * t + (i & 1) + 8 * (i >> 1);
    };
#pragma unroll
    for (int s = 0; s < STEPS; s++)
#pragma unroll
      for (int i = 0; i < N; i++) q[s][i] = __float_as_uint(live && dim(s, i) < c.width ? row[dim(s, i)] : 0.0f);
  };
  // Its operand terms, scaled by log2(e) / sqrt(width), and a fresh state.
  auto start_item = [&]() {
    float up = 1.0f;
    if (HALF) {  // the head's largest magnitude to 2^12
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(__uint_as_float(q[s][i])));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * a.scale_log2;
      int e = 0;
      if (top > 0.0f && top <= 3.402823466e38f) e = min(126, 12 - ((int)(__float_as_uint(top) >> 23) - 127));
      up = scale_of((uint8_t)(127 + e));
      const float down = scale_of((uint8_t)(127 - e));
      unscale[0] = __shfl_sync(0xffffffffu, down, 8 * t);
      unscale[1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
    }
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = __uint_as_float(q[s][i]) * a.scale_log2 * up;
      if constexpr (DTYPE == STB_F32) {  // hi, hi, lo, lo
        split_tf32(x[0], q[s][0], q[s][2]);
        split_tf32(x[1], q[s][1], q[s][3]);
      } else if constexpr (DTYPE == STB_BF16) {  // pairs of the first, second and third terms
        uint32_t u[3], v[3];
        split3_pair(x[0], x[1], u);
        split3_pair(x[2], x[3], v);
#pragma unroll
        for (int k = 0; k < 3; k++) {
          q[s][2 * k] = u[k];
          q[s][2 * k + 1] = v[k];
        }
      } else {
        uint32_t u[2], v[2];
        split2_pair(x[0], x[1], u);
        split2_pair(x[2], x[3], v);
        q[s][0] = u[0];
        q[s][1] = v[0];
        q[s][2] = u[1];
        q[s][3] = v[1];
      }
    }
#pragma unroll
    for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    m1[0] = m1[1] = m2[0] = m2[1] = -INFINITY;
    sum[0] = sum[1] = 0.0f;
    base[0] = base[1] = -1e30f;
    down[0] = down[1] = 1.0f;
  };

  // o[i][j + 2 k]: head 2 t + j at this dimension (E4M3 values come in pairs of neighbouring dimensions).
  auto dim_of = [&](int i, int k) { return SCALED ? i * 16 + 2 * g + k : i * 16 + g + 8 * k; };

  // What takes the weights' scale from a result; E4M3's own can pass Float32's range at either end: its root, applied twice.
  auto back = [](float shift) { return SCALED ? exp2f(0.5f * (shift - P_SHIFT)) : (HALF ? exp2f(-P_SHIFT) : 1.0f); };

  // The result of an item's tiles that this warp has seen: all of them to y; a part to the block's pieces (a first
  // part, while the ring is in use) or over the warp's own ring (a last part).
  float *const block_pieces = a.pieces + (size_t)blockIdx.x * BLOCK_PIECES;
  float *const my_ring = (float *)(smem + warp * S::STAGES * S::TILE);
  auto finish = [&](bool starts, bool ends) {
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], off);
    const bool whole = starts && ends;
    float *part = ends ? block_pieces + (2 + warp) * S::PART : my_ring;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int in_chunk = 2 * t + j, head = (use.item % chunks_of) * 8 + in_chunk;
      float *to = part + in_chunk * (WP + 4) + 4, f = 1.0f, f2 = 1.0f;
      int most = WP;
      if (whole) {
        to = a.y + (a.first + use.b) * a.y_row + (size_t)(use.item / chunks_of * a.group + head) * c.width;
        f2 = back(m2[j] - m1[j]);
        f = (SCALED ? f2 : 1.0f) / sum[j];
        most = head < a.group ? c.width : 0;
      } else if (g == 0) {
        *(float4 *)(to - 4) = make_float4(m1[j], m2[j], sum[j], 0.0f);
      }
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int k = 0; k < 2; k++)
          if (dim_of(i, k) < most) to[dim_of(i, k)] = sum[j] != 0.0f ? o[i][j + 2 * k] * f2 * f : 0.0f;
    }
    if (whole) return;
    if (lane == 0) {
      int *p = s_part[2 * warp + (ends ? 0 : 1)];
      p[0] = use.b;
      p[1] = use.item;
      p[2] = starts;
      p[3] = ends;
    }
  };

  // One loop for the first copies (i < 0) and the tiles: every long piece of code stands once, for the sake of the
  // instruction cache -- a short call runs all of it cold.
  bool starts = use.tile == 0;
  int want = 2;  // 2: q of the item at `use` has to be read, 1: it is on its way
  int stage = 0, next = 0;
#pragma unroll 1
  for (int i = todo > 0 ? 1 - S::STAGES : 0; i < todo; i++) {
    if (want == 2) {  // before the copies: these loads would queue behind them
      load_query();
      want = 1;
    }
    if (i >= 0) {
      copy_wait<(S::STAGES > 1 ? S::STAGES - 2 : 0)>();
      __syncwarp();  // every lane's copies of this tile are there, and the tile before it has been read
    }
    issue(next);
    next = next + 1 == S::STAGES ? 0 : next + 1;
    if (i < 0) continue;
    if (S::STAGES == 1) {
      copy_wait<0>();
      __syncwarp();
    }
    if (SCALED && S::STAGES == 2) __syncwarp();  // the tile's scales, stored just now
    if (want == 1) {
      start_item();
      want = 0;
    }
    const uint32_t keys = ring + stage * S::TILE, values = keys + TK * S::ROW;
    const uint8_t *m = meta + stage * S::META;
    const uint32_t mask = *(const uint32_t *)m;

    // scores: keys as rows, heads as columns; an accumulator per term of q and per parity of the step
    constexpr int PRODUCTS = DTYPE == STB_F32 ? 3 : TERMS;
    float acc[MB][PRODUCTS][2][4] = {};
    {
      const int row = (lane & 7) + ((lane >> 3) & 1) * 8, odd = lane >> 4;
#pragma unroll
      for (int s = 0; s < S::PAIRS; s++)
#pragma unroll
        for (int b = 0; b < MB; b++) {
          uint32_t r[4];
          load_matrix4(r, chunk_at<S::ROW>(keys, row + 16 * b, 2 * s + odd));
          if constexpr (SCALED) {  // two steps of 16 dimensions
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const uint32_t x = r[2 * h], y = r[2 * h + 1];
              const uint32_t k[4] = {widen_pair(x & 0xffffu), widen_pair(y & 0xffffu), widen_pair(x >> 16), widen_pair(y >> 16)};
#pragma unroll
              for (int i = 0; i < 2; i++) product<DTYPE>(acc[b][i][h], k, q[2 * s + h][2 * i], q[2 * s + h][2 * i + 1]);
            }
          } else if constexpr (DTYPE == STB_F32) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; i++) cut_tf32(__uint_as_float(r[i]), hi[i], lo[i]);
            product<DTYPE>(acc[b][0][s & 1], hi, q[s][0], q[s][1]);
            product<DTYPE>(acc[b][1][s & 1], hi, q[s][2], q[s][3]);
            product<DTYPE>(acc[b][2][s & 1], lo, q[s][0], q[s][1]);
          } else {
#pragma unroll
            for (int i = 0; i < TERMS; i++) product<DTYPE>(acc[b][i][s & 1], r, q[s][2 * i], q[s][2 * i + 1]);
          }
        }
    }
    float sc[MB][4], sw[SCALED ? MB : 1][4];  // [2 k + j]: key g + 8 k, head 2 t + j
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float2 scale = make_float2(1.0f, 0.0f);
        if (SCALED) scale = ((const float2 *)(m + 16))[16 * b + 8 * k + g];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int i = 2 * k + j;
          float x = acc[b][PRODUCTS - 1][0][i] + acc[b][PRODUCTS - 1][1][i];
#pragma unroll
          for (int n = PRODUCTS - 2; n >= 0; n--) x += acc[b][n][0][i] + acc[b][n][1][i];
          if (HALF) x *= SCALED ? unscale[j] * scale.x : unscale[j];
          sc[b][i] = x;
          if (SCALED) sw[b][i] = x + scale.y;
        }
      }
    if (mask != 0xffffffffu) {
#pragma unroll
      for (int b = 0; b < MB; b++)
#pragma unroll
        for (int k = 0; k < 2; k++)
          if (!(mask >> (16 * b + 8 * k + g) & 1))
            sc[b][2 * k] = sc[b][2 * k + 1] = sw[SCALED ? b : 0][2 * k] = sw[SCALED ? b : 0][2 * k + 1] = -INFINITY;
    }
    // What is rare, by one vote: a score that passed its maximum by far, or (F16 weights) one out of the weights' range.
    auto weighed = [&](int b, int i) -> float & { return SCALED ? sw[SCALED ? b : 0][i] : sc[b][i]; };  // log2 of the weight
    auto is_rare = [&](bool masked_too) {
      bool rare = false;
#pragma unroll
      for (int b = 0; b < MB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (SCALED || !HALF) rare |= sc[b][i] > m1[i & 1] + LAZY;
          if (HALF) {
            rare |= weighed(b, i) > base[i & 1] + P_TOP;
            if (masked_too) rare |= weighed(b, i) < base[i & 1] + P_LOW;
            else rare |= (weighed(b, i) < base[i & 1] + P_LOW) & (weighed(b, i) != -INFINITY);
          }
        }
      return __any_sync(0xffffffffu, rare);  // the same for the whole warp
    };
    bool low = false;
    volatile float later[MB * 4];  // in local memory, which only tiles with low weights touch
    if (is_rare(true)) {  // a masked key looks so at first
      if (!HALF || is_rare(false)) {  // move the heads' maxima, and the weights' base to this tile's
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float t1 = -INFINITY, t2 = -INFINITY, least = INFINITY;  // of this tile
#pragma unroll
          for (int b = 0; b < MB; b++)
#pragma unroll
            for (int i = j; i < 4; i += 2) {
              t1 = fmaxf(t1, sc[b][i]);
              if (HALF) {
                if (SCALED) t2 = fmaxf(t2, sw[b][i]);
                if (weighed(b, i) != -INFINITY) least = fminf(least, weighed(b, i));
              }
            }
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, off));
            if (SCALED) t2 = fmaxf(t2, __shfl_xor_sync(0xffffffffu, t2, off));
            if (HALF) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, off));
          }
          if (!SCALED) t2 = t1;
          const float n1 = fmaxf(m1[j], t1), n2 = SCALED ? fmaxf(m2[j], t2) : n1;
          const float f1 = n1 == m1[j] ? 1.0f : pow2(m1[j] - n1), f2 = n2 == m2[j] ? 1.0f : pow2(m2[j] - n2);
          sum[j] *= f1;
#pragma unroll
          for (int i = 0; i < NT; i++) {
            o[i][j] *= f2;
            o[i][2 + j] *= f2;
          }
          m1[j] = n1;
          m2[j] = n2;
          if (HALF && t2 != -INFINITY) {
            if (t2 > base[j] + P_TOP || least < base[j] + P_LOW) base[j] = fmaxf(t2, n2 - 100.0f) - P_SHIFT;
            down[j] = pow2(base[j] - n2 + P_SHIFT);
          }
        }
        if constexpr (HALF) {
          auto is_low = [&](int b, int i) { return (weighed(b, i) < base[i & 1] + P_LOW) & (weighed(b, i) != -INFINITY); };
          bool some = false;
#pragma unroll
          for (int b = 0; b < MB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) some |= is_low(b, i);
          low = __any_sync(0xffffffffu, some);
          if (low) {
#pragma unroll
            for (int b = 0; b < MB; b++)
#pragma unroll
              for (int i = 0; i < 4; i++) later[b * 4 + i] = is_low(b, i) ? missing(pow2(weighed(b, i) - base[i & 1])) : 0.0f;
          }
        }
      }
    }
    // Weights; a maximum of -inf means that no key has counted yet, and none does here (their scores are -inf).
    float w[MB][4];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float base1 = m1[j] == -INFINITY ? 0.0f : m1[j];
#pragma unroll
      for (int b = 0; b < MB; b++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const float p = pow2(sc[b][2 * k + j] - base1);
          sum[j] += p;
          w[b][2 * k + j] = HALF ? pow2(weighed(b, 2 * k + j) - base[j]) : p;
        }
    }

    // weighted values: dimensions as rows, heads as columns, a fresh result per tile added in Float32
    if constexpr (DTYPE == STB_F32) {
      uint32_t hi[2][2], lo[2][2];  // [8-key half][key 2 t + i] of head g
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int from = (2 * t + i) * 4 + (g >> 1);
          const float x = __shfl_sync(0xffffffffu, w[0][2 * k], from), y = __shfl_sync(0xffffffffu, w[0][2 * k + 1], from);
          split_tf32(g & 1 ? y : x, hi[k][i], lo[k][i]);
        }
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float r[4] = {};
#pragma unroll
        for (int k = 0; k < 2; k++) {
          uint32_t vh[4], vl[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {  // dimension g + 8 (i & 1), key 2 t + (i >> 1): the product's slots t and t + 4
            float v;
            asm volatile("ld.shared.f32 %0, [%1];"
                         : "=f"(v)
                         : "r"(chunk_at<S::ROW>(values, 8 * k + 2 * t + (i >> 1), 4 * n + 2 * (i & 1) + (g >> 2)) + (g & 3) * 4));
            cut_both_tf32(v, vh[i], vl[i]);
          }
          product<DTYPE>(r, vl, hi[k][0], hi[k][1]);
          product<DTYPE>(r, vh, lo[k][0], lo[k][1]);
          product<DTYPE>(r, vh, hi[k][0], hi[k][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) o[n][i] += r[i];
      }
    } else {
      uint32_t p[MB][2][TERMS];  // [8-key half] of each term: keys 2 t, 2 t + 1 of head g
#pragma unroll
      for (int b = 0; b < MB; b++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          if constexpr (DTYPE == STB_BF16) split3_pair(w[b][2 * k], w[b][2 * k + 1], p[b][k]);
          else split2_pair(w[b][2 * k], w[b][2 * k + 1], p[b][k], P_REST);
#pragma unroll
          for (int i = 0; i < TERMS; i++) p[b][k][i] = transpose8(p[b][k][i]);
        }
      const int row = (lane & 7) + (lane >> 4) * 8, odd = (lane >> 3) & 1;
#pragma unroll
      for (int s = 0; s < S::PAIRS; s++) {
        constexpr int PAIR = SCALED ? 2 : 1;  // 16-dimension results of two chunks
        constexpr int SUMS = HALF ? 2 : 1;    // of the first terms, and of the second ones
        uint32_t v[MB][4];
#pragma unroll
        for (int b = 0; b < MB; b++) load_matrix4_trans(v[b], chunk_at<S::ROW>(values, row + 16 * b, 2 * s + odd));
#pragma unroll
        for (int h = 0; h < PAIR; h++) {
          float r[SUMS][4] = {};
#pragma unroll
          for (int b = 0; b < MB; b++) {
            if constexpr (SCALED) {  // bytes (key, dim), (key, dim + 1), (key + 1, dim), (key + 1, dim + 1)
              const uint32_t x = __byte_perm(v[b][h], 0, 0x3120), z = __byte_perm(v[b][2 + h], 0, 0x3120);
              const uint32_t u[4] = {widen_pair(x & 0xffffu), widen_pair(x >> 16), widen_pair(z & 0xffffu), widen_pair(z >> 16)};
#pragma unroll
              for (int i = TERMS - 1; i >= 0; i--) product<DTYPE>(r[i % SUMS], u, p[b][0][i], p[b][1][i]);
            } else {
#pragma unroll
              for (int i = TERMS - 1; i >= 0; i--) product<DTYPE>(r[i % SUMS], v[b], p[b][0][i], p[b][1][i]);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float &to = o[PAIR * s + h][i];
            if (HALF) to = fmaf(r[0][i], down[i & 1], fmaf(r[SUMS - 1][i], down[i & 1] / P_REST, to));
            else to += r[0][i];
          }
        }
      }
    }

    if constexpr (HALF) {
      if (low) {  // would 2^-37 of all values be 2^-22 of some result?
        float widest = 448.0f;
        if (!SCALED) {
          __half2 top = __float2half2_rn(0.0f);
#pragma unroll 1
          for (int n = 0; n < MB * S::PAIRS; n++) {
            uint32_t v[4];
            const int chunk = n / MB * 2 + (lane >> 4);
            load_matrix4(v, chunk_at<S::ROW>(values, n % MB * 16 + (lane & 15), chunk < row_chunks ? chunk : 0));
#pragma unroll
            for (int k = 0; k < 4; k++) top = __hmax2(top, __habs2(*reinterpret_cast<const __half2 *>(&v[k])));
          }
          const float mine = __half2float(__hmax(__low2half(top), __high2half(top)));
          widest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mine)));
        }
        float least[2] = {INFINITY, INFINITY};
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
          for (int k = 0; k < 2; k++)
            if ((SCALED ? i : 2 * i + k) < row_chunks) {
#pragma unroll
              for (int j = 0; j < 2; j++) least[j] = fminf(least[j], fabsf(o[i][j + 2 * k]));
            }
        const bool some = (least[0] < down[0] * widest * (TK * 0x1p-15f)) | (least[1] < down[1] * widest * (TK * 0x1p-15f));
        if (__any_sync(0xffffffffu, some)) {  // what the low weights miss, in Float32, key by key
#pragma unroll 1
          for (int key = 0; key < TK; key++) {
            float x[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const float mine = later[2 * (key >> 3) + j];
              x[j] = __shfl_sync(0xffffffffu, mine, (key & 7) * 4 + t) * down[j];
            }
            if (!__any_sync(0xffffffffu, (x[0] != 0.0f) | (x[1] != 0.0f))) continue;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
              for (int k = 0; k < 2; k++) {
                float v;
                if constexpr (SCALED) {
                  uint32_t u;
                  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(u) : "r"(chunk_at<S::ROW>(values, key, i) + 2 * g + k));
                  v = widen_e4m3x2((uint16_t)u).x;
                } else {
                  uint16_t u;
                  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(chunk_at<S::ROW>(values, key, 2 * i + k) + 2 * g));
                  v = widen1<__half>(u);
                }
                o[i][2 * k] = fmaf(x[0], v, o[i][2 * k]);
                o[i][2 * k + 1] = fmaf(x[1], v, o[i][2 * k + 1]);
              }
          }
        }
      }
    }
    const bool ends = use.tile + 1 == use.tiles;
    if (ends || i + 1 == todo) {
      if (!ends) {  // the part goes over the ring
        copy_wait<0>();
        __syncwarp();
      }
      finish(starts, ends);
      starts = true;
      want = 2;
    }
    advance(use);
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;
  }
  copy_wait<0>();
  __syncthreads();

  // Joins the parts of the items that this block covers in part, a warp per head, without another block barrier.
  constexpr int FAR = MAX_GRID / 32;
  auto write = [&](int b, int item, int h, int d, float4 v, float n1, float n2, float all) {
    const int head = item % chunks_of * 8 + h;
    if (head >= a.group) return;
    float *y = a.y + (a.first + b) * a.y_row + (size_t)(item / chunks_of * a.group + head) * c.width + d;
    const float f2 = back(n2 - n1), f = (SCALED ? f2 : 1.0f) / all;
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (d + i < c.width) y[i] = all != 0.0f ? x[i] * f2 * f : 0.0f;
  };
  auto add = [](float4 &v, const float4 &x, float f) {
    if (f == 0.0f) return;  // a part without a key may hold anything
    v.x = fmaf(x.x, f, v.x);
    v.y = fmaf(x.y, f, v.y);
    v.z = fmaf(x.z, f, v.z);
    v.w = fmaf(x.w, f, v.w);
  };
  auto most = [](float x) {  // over the warp, by the order of the bits
    const int i = __float_as_int(x), key = i ^ (i >> 31 & 0x7fffffff), top = __reduce_max_sync(0xffffffffu, key);
    return __int_as_float(top ^ (top >> 31 & 0x7fffffff));
  };
  auto total_of = [](float x) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    return x;
  };
  constexpr int WIDE = (WP + 127) / 128;  // float4 of a lane
  const int mine_b = lane < 2 * S::WARPS ? s_part[lane][0] : -1, mine_item = lane < 2 * S::WARPS ? s_part[lane][1] : -1;
  // the part of entry `lane`
  const float *const mine_at = lane & 1 ? (const float *)(smem + (lane >> 1) * S::STAGES * S::TILE) : block_pieces + (2 + (lane >> 1)) * S::PART;
  const uint32_t entries = __ballot_sync(0xffffffffu, mine_b >= 0);
  // First, head by head, every item's parts of this block: to y, or to a piece of the block's (an item at either end of its
  // stretch).
  struct Split {
    int b, item, first, c0, c1;
  } splits[2];
  int cut = 0;
  float4 v[WIDE];
#pragma unroll 1
  for (int h = warp; h < 8; h += S::WARPS) {
    const int row = h * (WP + 4);
    float n1, n2, all;
    cut = 0;
#pragma unroll 1
    for (uint32_t left = entries; left;) {
      const int i0 = __ffs(left) - 1;
      const int b = __shfl_sync(0xffffffffu, mine_b, i0), item = __shfl_sync(0xffffffffu, mine_item, i0);
      const uint32_t which = __ballot_sync(0xffffffffu, mine_b == b && mine_item == item);
      left &= ~which;
      const bool has = which >> lane & 1;
      const float4 part = has ? *(const float4 *)(mine_at + row) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      n1 = most(part.z != 0.0f ? part.x : -INFINITY);
      n2 = SCALED ? most(part.z != 0.0f ? part.y : -INFINITY) : n1;
      all = total_of(part.z != 0.0f ? part.z * exp2f(part.x - n1) : 0.0f);
      const float factor = part.z != 0.0f ? exp2f(part.y - n2) : 0.0f;
#pragma unroll
      for (int k = 0; k < WIDE; k++) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (uint32_t m = which; m;) {  // four parts on their way at a time
        float4 x[4][WIDE];
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int i = __ffs(m) - 1;
          m &= m - 1;
          f[j] = __shfl_sync(0xffffffffu, factor, i & 31);
          if (i < 0) f[j] = 0.0f;
          const float *at = i & 1 ? (const float *)(smem + (i >> 1) * S::STAGES * S::TILE) : block_pieces + (2 + (i >> 1)) * S::PART;
#pragma unroll
          for (int k = 0; k < WIDE; k++)
            if (i >= 0 && k * 128 + lane * 4 < WP) x[j][k] = *(const float4 *)(at + row + 4 + k * 128 + lane * 4);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int k = 0; k < WIDE; k++)
            if (k * 128 + lane * 4 < WP) add(v[k], x[j][k], f[j]);
      }
      if (s_part[i0][2] && s_part[31 - __clz(which)][3]) {  // from its start to its end
#pragma unroll
        for (int k = 0; k < WIDE; k++)
          if (k * 128 + lane * 4 < WP) write(b, item, h, k * 128 + lane * 4, v[k], n1, n2, all);
        continue;
      }
      const int tiles = s_start[b + 1] - s_start[b], first = s_start[b] * items + item * tiles;
      float *piece = block_pieces + (block0 >= first ? 0 : 1) * S::PART;
      if (lane == 0) *(float4 *)(piece + row) = make_float4(n1, n2, all, 0.0f);
#pragma unroll
      for (int k = 0; k < WIDE; k++)
        if (k * 128 + lane * 4 < WP) *(float4 *)(piece + row + 4 + k * 128 + lane * 4) = v[k];
      Split &to = splits[cut ? 1 : 0];
      to.b = b;
      to.item = item;
      to.first = first;
      to.c0 = line.of(first);
      to.c1 = line.of(first + tiles - 1);
      cut++;
    }
  }
  if (!cut) return;
  // Then the warp's pieces are announced, each on the counter of its head and of its item's first block; the last block to
  // arrive joins them, in the blocks' order, and clears the counter.
  __syncwarp();
  __threadfence();
  int last = 0;
  if ((lane & 1) < cut && warp + (lane >> 1) * S::WARPS < 8) {
    const Split &of = lane & 1 ? splits[1] : splits[0];
    int *const counter = a.arrived + of.c0 * 8 + warp + (lane >> 1) * S::WARPS;
    last = atomicAdd(counter, 1) == of.c1 - of.c0;
    if (last) *counter = 0;
  }
  __syncwarp();
  __threadfence();
#pragma unroll 1
  for (uint32_t to_join = __ballot_sync(0xffffffffu, last); to_join; to_join &= to_join - 1) {
    const int n = __ffs(to_join) - 1, h = warp + (n >> 1) * S::WARPS, row = h * (WP + 4);
    const Split &of = n & 1 ? splits[1] : splits[0];
    const int count = of.c1 - of.c0 + 1;
    // A lane per piece: where it lies, its maxima and sum.  This code runs once and cold: what counts is that it is short.
    float4 far[FAR];
    int at[FAR];
    float n1 = -INFINITY, n2 = -INFINITY, all = 0.0f;
#pragma unroll
    for (int r = 0; r < FAR; r++) {
      const int k = of.c0 + min(r * 32 + lane, count - 1);
      at[r] = (k * (BLOCK_PIECES / 4) + (line.start(k) >= of.first ? 0 : S::PART / 4)) + row / 4;
      far[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r * 32 < count) {
        if (r * 32 + lane < count) far[r] = __ldcg((const float4 *)a.pieces + at[r]);
        if (far[r].z != 0.0f) {
          n1 = fmaxf(n1, far[r].x);
          n2 = fmaxf(n2, far[r].y);
        }
      }
    }
    n1 = most(n1);
    n2 = SCALED ? most(n2) : n1;
#pragma unroll
    for (int r = 0; r < FAR; r++)
      if (r * 32 < count) {
        if (far[r].z != 0.0f) all += far[r].z * exp2f(far[r].x - n1);
        far[r].w = far[r].z != 0.0f ? exp2f(far[r].y - n2) : 0.0f;
      }
    all = total_of(all);
#pragma unroll
    for (int k = 0; k < WIDE; k++) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    int place = at[0];
    float factor = far[0].w;
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += 8) {  // eight pieces on their way at a time
      if (i0 > 0 && (i0 & 31) == 0) {
#pragma unroll
        for (int r = 1; r < FAR; r++)
          if (i0 == r * 32) place = at[r], factor = far[r].w;
      }
      float4 x[8][WIDE];
#pragma unroll
      for (int j = 0; j < 8; j++) {  // the last piece again behind the last
        const float4 *from = (const float4 *)a.pieces + __shfl_sync(0xffffffffu, place, (i0 + j) & 31) + 1 + lane;
#pragma unroll
        for (int k = 0; k < WIDE; k++)
          if (k * 128 + lane * 4 < WP) x[j][k] = __ldcg(from + k * 32);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float f = __shfl_sync(0xffffffffu, factor, (i0 + j) & 31);
#pragma unroll
        for (int k = 0; k < WIDE; k++)
          if (k * 128 + lane * 4 < WP) add(v[k], x[j][k], f);
      }
    }
#pragma unroll
    for (int k = 0; k < WIDE; k++)
      if (k * 128 + lane * 4 < WP) write(of.b, of.item, h, k * 128 + lane * 4, v[k], n1, n2, all);
  }
}

template <int DTYPE, int WP>
void launch_attention(stb_session *s, const PagedView &c, AttendArgs a, int batch, int at_once) {
  using S = Shape<DTYPE, WP>;
  {
    static std::mutex mu;
    static bool configured[64] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (s->device < 0 || s->device >= 64 || !configured[s->device]) {
      STB_CUDA(cudaFuncSetAttribute(paged_attention_kernel<DTYPE, WP>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
      if (s->device >= 0 && s->device < 64) configured[s->device] = true;
    }
  }
  const int grid = std::min(tc::sm_count(s->device), MAX_GRID);
  for (a.first = 0; a.first < batch; a.first += at_once) {
    a.batch = std::min(at_once, batch - a.first);
    launch_kernel(paged_attention_kernel<DTYPE, WP>, dim3(grid), dim3(S::THREADS), (size_t)S::SMEM, s->stream, true, c, a);
    count_launch(s);
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
    a.batch = batch;
    a.first = 0;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)c.width));
    a.pieces = nullptr;
    a.arrived = nullptr;
    const int esz = cache->dtype == STB_F32 ? 4 : (cache->dtype == STB_E4M3 ? 1 : 2);
    // Requests of one launch whose tiles (16 keys at least) an Int can count, whatever their lengths.
    const int64_t tiles = ((int64_t)c.blocks * c.page_size / 16 + 1) * c.kv_heads * ((a.group + 7) / 8);
    const int at_once = (int)std::min<int64_t>(MAX_BATCH, 0x7fffffff / tiles);
    // The copies move whole 16-byte chunks and address rows of the cache by an Int.
    const bool chunked = c.width <= 256 && c.width * esz % 16 == 0 && cache->keys % 16 == 0 && cache->values % 16 == 0 &&
                         (int64_t)c.pages * c.kv_heads * c.page_size <= 0x7fffffff && at_once > 0;
    if (!chunked) {
      dispatch_paged(cache->dtype, [&](auto t) {
        launch_kernel(paged_attention_any_kernel<decltype(t)::value>, dim3(heads, batch), dim3(256), 0, s->stream, true, c, a);
      });
      count_launch(s);
      return;
    }
    const uint64_t counters = MAX_GRID * 8 * sizeof(int), bytes = counters + (uint64_t)MAX_GRID * BLOCK_PIECES * sizeof(float);
    if (!s->paged_ws) {
      if (capturing(s)) throw Error(STB_ERR_STATE, "a session's first paged attention cannot be captured: make a call before");
      s->paged_ws = session_alloc(s, bytes);
      STB_CUDA(cudaMemsetAsync((void *)s->paged_ws, 0, counters, s->stream));
    }
    a.arrived = (int *)s->paged_ws;
    a.pieces = (float *)(s->paged_ws + counters);
    dispatch_paged(cache->dtype, [&](auto t) {
      constexpr int DT = decltype(t)::value;
      if (c.width <= 64) launch_attention<DT, 64>(s, c, a, batch, at_once);
      else if (c.width <= 96) launch_attention<DT, 96>(s, c, a, batch, at_once);
      else if (c.width <= 128) launch_attention<DT, 128>(s, c, a, batch, at_once);
      else launch_attention<DT, 256>(s, c, a, batch, at_once);
    });
  });
}
