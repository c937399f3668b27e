// Norm and rotation of the query and key heads in one pass (stb_op_qk_norm_rope): each head x of a row at
// position p becomes
//   u_d = x_d / sqrt(mean(x^2) + eps) * w_d,   y_d = u_d cos a - u_{d+half} sin a,  y_{d+half} = u_{d+half} cos a + u_d sin a
// with a = p * theta^(-2 d / width), d < half = width / 2.
//
// What bounds it: 8 bytes per element, read and written once, as long as loads stay under way while the angles are worked
// out.  Every warp runs alone over its units, whole rows' heads or parts of a row's: three steps' copies ahead, the sines
// and cosines of the unit's row in shared memory of its own.  Angles, their sines and cosines, the sum of squares and its
// root are in double; what they are multiplied by is in Float32: at most 2 half steps of the result and 4 of each
// rotated product beside it.  8191 rows of 40 heads of 128 take 60 us = 5.6 TB/s, 0.85 of the copy rate.  The rotation in
// double too took 85 us (the conversions of its results are the scarce thing), in pairs of Float32 75.
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
  pdl_wait();
  pdl_trigger();
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

constexpr int THREADS = 128, BLOCKS = 8, STAGES = 4;

// 1 / sqrt(v) of a positive v to 2^-43: the Float32 root and one Newton step where Float32 has v (the others go the long
// way), a fifth of the double function's operations.
__device__ __forceinline__ double inverse_root(double v) {
  if (!(v > 1e-30 && v < 1e30)) return rsqrt(v);
  const double y = rsqrtf((float)v);
  return y * fma(-0.5 * v * y, y, 1.5);
}

__device__ __forceinline__ void copy16_async(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

// A step is up to 32 / L neighbouring query heads, or key heads, of a row, L lanes each, lane i its elements 4 i .. 4 i + 3
// and their partners (i < half / 4 <= L).  A row has q_steps and then k_steps of them, in `parts` units of `per` steps.
template <int L>
__global__ void __launch_bounds__(THREADS, BLOCKS) qk_norm_rope_kernel(const __grid_constant__ NormRope p, int q_steps, int k_steps,
                                                                       int parts, int per, int64_t units) {
  constexpr int HEADS = 32 / L;
  __shared__ double s_rate[L * 4];                 // angle per position over pi
  __shared__ __align__(16) float s_weight[2][L * 8];  // of q, of k
  __shared__ __align__(16) float2 s_turn[THREADS / 32][L * 4];  // (cos, sin) of each warp's row
  __shared__ float4 s_ring[THREADS / 32][STAGES][2][32];  // the steps ahead: a lane reads what it sent for itself
  const int half = p.width / 2, lane = threadIdx.x % L, in_step = threadIdx.x % 32 / L, per_row = q_steps + k_steps;
  const bool live = lane * 4 < half;
  const int warps = gridDim.x * (THREADS / 32), warp = blockIdx.x * (THREADS / 32) + threadIdx.x / 32;
  const int offset = in_step * p.width + lane * 4;  // of this lane in a step's heads

  // A place in a unit: `left` steps of one side's heads, then `rest` steps of the other's.
  struct Cursor {
    float *at;  // this lane's elements of the step
    int64_t unit;
    int row, side, left, rest, room, pos;  // room: heads of the side from the step's first on
  };
  auto enter = [&](Cursor &c, bool out, int step) {  // at the step-th step of c.side in c.row
    const float *base = out ? (c.side ? p.y[1] + c.row * p.y_row[1] : p.y[0] + c.row * p.y_row[0])
                            : (c.side ? p.x[1] + c.row * p.x_row[1] : p.x[0] + c.row * p.x_row[0]);
    c.at = const_cast<float *>(base) + (int64_t)step * HEADS * p.width + offset;
    c.room = (c.side ? p.heads[1] : p.heads[0]) - step * HEADS;
  };
  auto start = [&](Cursor &c, bool out) {  // of unit c.unit
    if (c.unit >= units) return;
    c.row = (int)(c.unit / parts);
    const int step = (int)(c.unit % parts) * per, end = min(per_row, step + per);
    c.pos = p.positions[c.row];
    c.side = step >= q_steps;
    c.left = (c.side ? end : min(end, q_steps)) - step;
    c.rest = end - step - c.left;
    enter(c, out, step - (c.side ? q_steps : 0));
  };
  auto advance = [&](Cursor &c, bool out) {
    c.at += HEADS * p.width;
    c.room -= HEADS;
    if (--c.left > 0) return;
    if (c.rest > 0) {
      c.side = 1;
      c.left = c.rest;
      c.rest = 0;
      enter(c, out, 0);
    } else {
      c.unit += warps;
      start(c, out);
    }
  };
  for (int d = threadIdx.x; d < half; d += THREADS) s_rate[d] = exp2(p.rate * d) * 0.31830988618379067154;
  pdl_wait();
  pdl_trigger();
  Cursor from, to;
  from.unit = to.unit = warp;
  start(from, false);
  start(to, true);
  float4(*const ring)[2][32] = s_ring[threadIdx.x / 32];
  auto send = [&](int stage) {
    if (from.unit < units) {
      if (live && in_step < from.room && from.pos >= 0) {
        copy16_async(&ring[stage][0][threadIdx.x % 32], from.at);
        copy16_async(&ring[stage][1][threadIdx.x % 32], from.at + half);
      }
      advance(from, false);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; i++) send(i);
  for (int i = threadIdx.x; i < 2 * p.width; i += THREADS) {
    const float *w = i < p.width ? p.w[0] : p.w[1];
    s_weight[i < p.width ? 0 : 1][i % p.width] = w ? w[i % p.width] : 1.0f;
  }
  const double mean = 1.0 / p.width;
  __syncthreads();
  float2 *const turn = s_turn[threadIdx.x / 32];  // of row `turned`
  int turned = -1;
  int stage = 0;
#pragma unroll 1
  while (to.unit < units) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    const float4 f = ring[stage][0][threadIdx.x % 32], g = ring[stage][1][threadIdx.x % 32];
    send(stage == 0 ? STAGES - 1 : stage - 1);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (to.pos >= 0) {
      if (turned != to.row) {
        turned = to.row;
        __syncwarp();
        for (int d = threadIdx.x % 32; d < half; d += 32) {
          double sn, cs;
          sincospi((double)to.pos * s_rate[d], &sn, &cs);
          turn[d] = make_float2((float)cs, (float)sn);
        }
        __syncwarp();
      }
      const bool has = live && in_step < to.room;
      float u[4] = {f.x, f.y, f.z, f.w}, v[4] = {g.x, g.y, g.z, g.w};
      if (to.side ? p.w[1] != nullptr : p.w[0] != nullptr) {  // the same for the whole warp
        double sq = 0.0;
        if (has) {
#pragma unroll
          for (int i = 0; i < 4; i++) sq = fma((double)u[i], (double)u[i], fma((double)v[i], (double)v[i], sq));
        }
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
        double root = inverse_root(fma(sq, mean, p.eps));
        float down = 1.0f;
        if (root < 1e-36) {  // Float32 would have it with few bits
          root *= 0x1p64;
          down = 0x1p-64f;
        } else if (root > 1e36) {  // or not at all
          root = fmin(root * 0x1p-64, 0x1p127);
          down = 0x1p64f;
        }
        const float inv = (float)root;
        const float4 wa = *(const float4 *)&s_weight[to.side][lane * 4], wb = *(const float4 *)&s_weight[to.side][lane * 4 + half];
        const float wf[4] = {wa.x, wa.y, wa.z, wa.w}, wg[4] = {wb.x, wb.y, wb.z, wb.w};
        if (down != 1.0f) {
#pragma unroll
          for (int k = 0; k < 4; k++) u[k] *= down, v[k] *= down;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) u[k] = u[k] * inv * wf[k], v[k] = v[k] * inv * wg[k];
      }
      if (has) {
        float r[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float4 t = *(const float4 *)&turn[lane * 4 + i];
          r[i] = fmaf(u[i], t.x, -(v[i] * t.y));
          s[i] = fmaf(v[i], t.x, u[i] * t.y);
          r[i + 1] = fmaf(u[i + 1], t.z, -(v[i + 1] * t.w));
          s[i + 1] = fmaf(v[i + 1], t.z, u[i + 1] * t.w);
        }
        __stcs((float4 *)to.at, make_float4(r[0], r[1], r[2], r[3]));
        __stcs((float4 *)(to.at + half), make_float4(s[0], s[1], s[2], s[3]));
      }
    }
    advance(to, true);
  }
}

template <int L>
void launch_rows(stb_session *s, const NormRope &p) {
  const int heads = 32 / L, q_steps = (p.heads[0] + heads - 1) / heads, k_steps = (p.heads[1] + heads - 1) / heads;
  const int per_row = q_steps + k_steps, most = tc::sm_count(s->device) * BLOCKS;
  // Rows in parts of five steps (60 us for 8191 rows of 40 heads of 128, 64 with parts of ten), of fewer where that leaves warps idle.
  const int64_t warps = (int64_t)most * (THREADS / 32);
  const int per = (int)std::max<int64_t>(1, std::min<int64_t>(5, (int64_t)p.rows * per_row / warps));
  const int parts = (per_row + per - 1) / per;
  const int64_t units = (int64_t)p.rows * parts, blocks = std::min<int64_t>((units + THREADS / 32 - 1) / (THREADS / 32), most);
  launch_kernel(qk_norm_rope_kernel<L>, dim3((unsigned)blocks), dim3(THREADS), 0, s->stream, true, p, q_steps, k_steps, parts, per, units);
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
      launch_kernel(qk_norm_rope_any_kernel, dim3((unsigned)blocks), dim3(256), 0, s->stream, true, p);
    }
    count_launch(s);
  });
}
