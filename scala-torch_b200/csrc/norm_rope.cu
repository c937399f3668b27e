// Norm and rotation of the query and key heads in one pass (stb_op_qk_norm_rope): each head x of a row at
// position p becomes
//   u_d = x_d / sqrt(mean(x^2) + eps) * w_d,   y_d = u_d cos a - u_{d+half} sin a,  y_{d+half} = u_{d+half} cos a + u_d sin a
// with a = p * theta^(-2 d / width), d < half = width / 2: stb_op_rmsnorm and stb_op_rope's arithmetic, in
// double with one rounding at the end.
#include <cmath>

#include "gemv.cuh"

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

// One warp per (row, head).
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const NormRope p) {
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
    const int64_t blocks = ((int64_t)rows * (heads + kv_heads) + 7) / 8;
    STB_REQUIRE(blocks <= 0x7fffffff, "too many rows");
    launch_kernel(qk_norm_rope_kernel, dim3((unsigned)blocks), dim3(256), 0, s->stream, false, p);
    count_launch(s);
  });
}
