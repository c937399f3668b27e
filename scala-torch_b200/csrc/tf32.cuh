// Products of Float32 values on the tensor cores in TF32 terms.
#pragma once

#include "common.cuh"

namespace stb {

// x = hi + lo in two TF32 values (11 significant bits each), in three ways.  All keep what is no number: a NaN or an infinity
// leaves a NaN in hi or lo, so that what it enters becomes NaN.  Float32's arithmetic gives the NaN 0x7fffffff, which the
// half step would carry into the sign: min keeps it below.
__device__ __forceinline__ uint32_t rest_tf32(float rest) {
  return ((uint32_t)min((int)__float_as_uint(rest), 0x7fffefff) + 0x1000u) & 0xffffe000u;
}

// hi rounded to nearest, cut where that would pass the largest TF32 value: |lo| <= 2^-11 |x|, its sign as good as random.
// x - hi - lo is at most 2^-23 |x|.
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
  const uint32_t b = min((uint32_t)min((int)__float_as_uint(x), 0x7f7fefff), 0xff7fefffu);  // positive, then negative tops
  hi = (b + 0x1000u) & 0xffffe000u;
  lo = rest_tf32(x - __uint_as_float(hi));
}

// hi cut, for the operand that streams through: |lo| < 2^-10 |x|, of x's sign; x - hi - lo at most 2^-22 |x|.  The other
// operand's lo is of either sign, which keeps the product of both los (left out) without bias.  Three operations fewer: 0.5
// GiB of F32 cache 105 / 103 / 186 us at widths 64 / 128 / 256, 115 / 114 / 237 with split_tf32.
__device__ __forceinline__ void cut_tf32(float x, uint32_t &hi, uint32_t &lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = rest_tf32(x - __uint_as_float(hi));
}

// Both cut: hi + lo never passes x, so that a mean of Float32's largest values stays finite; x - hi - lo less than 2^-21 |x|,
// on average 2^-24 of x's sign (the values alone this way: 100 / 100 / 174 us).
__device__ __forceinline__ void cut_both_tf32(float x, uint32_t &hi, uint32_t &lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

// c += a . b: 16 x 8 results of a 16 x 8 and an 8 x 8 operand.
__device__ __forceinline__ void product_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace stb
