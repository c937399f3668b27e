// Norm and rotation of the query and key heads in one pass (stb_op_qk_norm_rope): each head x of a row at
// position p becomes
//   u_d = x_d / sqrt(mean(x^2) + eps) * w_d,   y_d = u_d cos a - u_{d+half} sin a,  y_{d+half} = u_{d+half} cos a + u_d sin a
// with a = p * theta^(-2 d / width), d < half = width / 2.
//
// What bounds it: 8 bytes per element, read and written once, as long as enough loads are under way while the angles
// are worked out.  A block of 256 threads takes a row at a time (several rows of few heads), all of its heads' loads
// sent before anything else; the sines and cosines of the row, shared by its heads, go to shared memory meanwhile.  All
// arithmetic is in double, as stb_op_rmsnorm's and stb_op_rope's, with one rounding: 5 operations and 3 conversions
// per element, a quarter and a half of what the SM's double and conversion pipes take at the copy rate.
#include <algorithm>
#include <cmath>

#include "gemv.cuh"
#include "tc_common.cuh"

namespace stb {
namespace {

struct NormRope {
  const float *x[2];  // q, k
  float *y[2];
  const float *w[2];
  int64_t x_row[2], y_row[2];
  int heads[2];
  const int *positions;
  int rows, width;
  double eps, rate;  // rate = -2 log2(theta) / width
};

// One warp per (row, head), any alignment.
__global__ void __launch_bounds__(256) qk_norm_rope_any_kernel(const NormRope p) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31, every = p.heads[0] + p.heads[1], half = p.width / 2;
  if (unit >= (int64_t)p.rows * every) return;
  const int row = (int)(unit / every);
  int head = (int)(unit % every);
  const int side = head >= p.heads[0];
  if (side) head -= p.heads[0];
  const int pos = p.positions[row];
  if (pos < 0) return;
  const float *x = p.x[side] + row * p.x_row[side] + (size_t)head * p.width;
  float *y = p.y[side] + row * p.y_row[side] + (size_t)head * p.width;
  const float *w = p.w[side];
  double inv = 1.0;
  if (w) {
    double sq = 0.0;
    for (int d = lane; d < p.width; d += 32) sq = fma((double)x[d], (double)x[d], sq);
    for (int off = 16; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    inv = 1.0 / sqrt(sq / p.width + p.eps);
  }
  for (int d = lane; d < half; d += 32) {
    double sn, cs;
    sincos((double)pos * exp2(p.rate * d), &sn, &cs);
    double a = x[d], b = x[d + half];
    if (w) {
      a = a * inv * (double)w[d];
      b = b * inv * (double)w[d + half];
    }
    y[d] = (float)(a * cs - b * sn);
    y[d + half] = (float)(b * cs + a * sn);
  }
}

constexpr int THREADS = 256, MAX_ROWS = 8;

// Groups of L lanes take a head each, lane i its elements 4 i .. 4 i + 3 and their partners (i < half / 4 <= L); a block takes
// `at_once` rows at a time (one, where U > 1), its group g the heads g, g + GROUPS, .. of them, U sent for at once.
template <int L, int U>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_kernel(const __grid_constant__ NormRope p, int at_once) {
  constexpr int GROUPS = THREADS / L;
  __shared__ double s_rate[L * 4];                  // angle per position over pi
  __shared__ __align__(16) float s_weight[2][L * 8];
  __shared__ double2 s_turn[2][MAX_ROWS][L * 4];    // (cos, sin), this round's and the next one's
  const int every = p.heads[0] + p.heads[1], half = p.width / 2, lane = threadIdx.x % L, group = threadIdx.x / L;
  const bool live = lane * 4 < half;
  const int in_block = U == 1 ? group / every : 0, head0 = U == 1 ? group % every : group;
  for (int d = threadIdx.x; d < half; d += THREADS) s_rate[d] = exp2(p.rate * d) * 0.31830988618379067154;
  for (int i = threadIdx.x; i < 2 * p.width; i += THREADS) {
    const float *w = i < p.width ? p.w[0] : p.w[1];
    s_weight[i < p.width ? 0 : 1][i % p.width] = w ? w[i % p.width] : 1.0f;
  }
  const bool normed = p.w[0] || p.w[1];
  __syncthreads();
  int buffer = 0;
#pragma unroll 1
  for (int64_t r0 = (int64_t)blockIdx.x * at_once; r0 < p.rows; r0 += (int64_t)gridDim.x * at_once, buffer ^= 1) {
    const int64_t row = r0 + in_block;
    const bool mine = in_block < at_once && row < p.rows && p.positions[row] >= 0 && live;
    for (int i = threadIdx.x; i < at_once * half; i += THREADS) {
      const int r = i / half, d = i % half, pos = r0 + r < p.rows ? p.positions[r0 + r] : -1;
      if (pos < 0) continue;
      double sn, cs;
      sincospi((double)pos * s_rate[d], &sn, &cs);
      s_turn[buffer][r][d] = make_double2(cs, sn);
    }
    bool waited = false;
#pragma unroll 1
    for (int h0 = head0; h0 - head0 < (U == 1 ? 1 : every); h0 += U * GROUPS) {
      float4 a[U], b[U];
#pragma unroll
      for (int k = 0; k < U; k++) {
        const int h = h0 + k * GROUPS, side = h >= p.heads[0];
        if (!mine || h >= every) continue;
        const float *x = (side ? p.x[1] + row * p.x_row[1] : p.x[0] + row * p.x_row[0]) + (size_t)(h - (side ? p.heads[0] : 0)) * p.width + lane * 4;
        a[k] = __ldcs((const float4 *)x);
        b[k] = __ldcs((const float4 *)(x + half));
      }
      if (!waited) __syncthreads();
      waited = true;
#pragma unroll
      for (int k = 0; k < U; k++) {
        const int h = h0 + k * GROUPS, side = h >= p.heads[0];
        const bool has = mine && h < every;
        const float u[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, v[4] = {b[k].x, b[k].y, b[k].z, b[k].w};
        double inv = 1.0;
        if (normed) {  // every group of the warp takes part in the shuffles
          double sq = 0.0;
          if (has) {
#pragma unroll
            for (int i = 0; i < 4; i++) sq = fma((double)u[i], (double)u[i], fma((double)v[i], (double)v[i], sq));
          }
#pragma unroll
          for (int off = L / 2; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
          if (side ? p.w[1] != nullptr : p.w[0] != nullptr) inv = rsqrt(sq / p.width + p.eps);
        }
        if (!has) continue;
        const float4 wa = *(const float4 *)&s_weight[side][lane * 4], wb = *(const float4 *)&s_weight[side][lane * 4 + half];
        const float wf[4] = {wa.x, wa.y, wa.z, wa.w}, wg[4] = {wb.x, wb.y, wb.z, wb.w};
        float r[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const double2 turn = s_turn[buffer][in_block][lane * 4 + i];
          const double c = (double)u[i] * (inv * (double)wf[i]), d = (double)v[i] * (inv * (double)wg[i]);
          r[i] = (float)(c * turn.x - d * turn.y);
          s[i] = (float)(d * turn.x + c * turn.y);
        }
        float *y = (side ? p.y[1] + row * p.y_row[1] : p.y[0] + row * p.y_row[0]) + (size_t)(h - (side ? p.heads[0] : 0)) * p.width + lane * 4;
        __stcs((float4 *)y, make_float4(r[0], r[1], r[2], r[3]));
        __stcs((float4 *)(y + half), make_float4(s[0], s[1], s[2], s[3]));
      }
    }
    if (!waited) __syncthreads();
  }
}

template <int L>
void launch_rows(stb_session *s, const NormRope &p) {
  constexpr int GROUPS = THREADS / L;
  const int every = p.heads[0] + p.heads[1];
  const int at_once = every <= GROUPS ? std::min(MAX_ROWS, GROUPS / every) : 1;
  const int64_t rounds = ((int64_t)p.rows + at_once - 1) / at_once;
  auto go = [&](auto u) {
    constexpr int U = decltype(u)::value;
    const int grid = (int)std::min<int64_t>(rounds, (int64_t)tc::sm_count(s->device) * (U <= 2 ? 4 : 3));
    launch_kernel(qk_norm_rope_kernel<L, U>, dim3(grid), dim3(THREADS), 0, s->stream, false, p, at_once);
  };
  const int deep = (every + GROUPS - 1) / GROUPS;
  if (deep == 1) go(std::integral_constant<int, 1>());
  else if (deep == 2) go(std::integral_constant<int, 2>());
  else if (deep == 3 || deep == 6) go(std::integral_constant<int, 3>());
  else go(std::integral_constant<int, 5>());
}

}  // namespace
}  // namespace stb

using namespace stb;

extern "C" int stb_op_qk_norm_rope(stb_session *s, uint64_t q, int64_t q_row, int heads, uint64_t k, int64_t k_row,
                                   int kv_heads, int width, int rows, uint64_t q_weight, uint64_t k_weight,
                                   uint64_t positions, double eps, double theta, uint64_t q_out, int64_t q_out_row,
                                   uint64_t k_out, int64_t k_out_row) {
  return guarded([&] {
    enter(s);
    STB_REQUIRE(rows >= 0 && heads >= 0 && kv_heads >= 0, "negative dimension");
    STB_REQUIRE(width > 0 && width % 2 == 0 && width <= 512, "RoPE requires a positive even width of at most 512");
    STB_REQUIRE(std::isfinite(theta) && theta > 0, "invalid rotary position or theta");
    STB_REQUIRE(std::isfinite(eps) && eps > 0, "invalid RMSNorm epsilon");
    if (!rows || heads + kv_heads == 0) return;
    STB_REQUIRE(std::isfinite(2147483647.0 * std::pow(theta, -2.0 * (width / 2 - 1) / width)), "rotary angle overflow");
    const uint64_t in[2] = {q, k}, out[2] = {q_out, k_out}, weight[2] = {q_weight, k_weight};
    const int64_t in_row[2] = {q_row, k_row}, out_row[2] = {q_out_row, k_out_row};
    const int count[2] = {heads, kv_heads};
    NormRope p;
    for (int i = 0; i < 2; i++) {
      if (count[i]) {
        STB_REQUIRE(in[i] && out[i] && in[i] % 4 == 0 && out[i] % 4 == 0, "norm and rope: null or misaligned Float32 buffer");
        STB_REQUIRE(weight[i] % 4 == 0, "norm and rope: misaligned weight");
        STB_REQUIRE(rows == 1 || (in_row[i] >= (int64_t)count[i] * width && out_row[i] >= (int64_t)count[i] * width),
                    "norm and rope rows overlap");
      }
      p.x[i] = (const float *)in[i];
      p.y[i] = (float *)out[i];
      p.w[i] = (const float *)weight[i];
      p.x_row[i] = in_row[i];
      p.y_row[i] = out_row[i];
      p.heads[i] = count[i];
    }
    STB_REQUIRE(positions && positions % 4 == 0, "null or misaligned positions");
    p.positions = (const int *)positions;
    p.rows = rows;
    p.width = width;
    p.eps = eps;
    p.rate = -2.0 * std::log2(theta) / width;
    // float4 pieces of each half of a head, wherever the rows begin
    bool pieces = width % 8 == 0 && width <= 256;
    for (int i = 0; i < 2; i++)
      if (count[i]) pieces &= in[i] % 16 == 0 && out[i] % 16 == 0 && weight[i] % 16 == 0 && (rows == 1 || (in_row[i] % 4 == 0 && out_row[i] % 4 == 0));
    if (pieces) {
      if (width <= 64) launch_rows<8>(s, p);
      else if (width <= 128) launch_rows<16>(s, p);
      else launch_rows<32>(s, p);
    } else {
      const int64_t blocks = ((int64_t)rows * (heads + kv_heads) + 7) / 8;
      STB_REQUIRE(blocks <= 0x7fffffff, "too many rows");
      launch_kernel(qk_norm_rope_any_kernel, dim3((unsigned)blocks), dim3(256), 0, s->stream, false, p);
    }
    count_launch(s);
  });
}
