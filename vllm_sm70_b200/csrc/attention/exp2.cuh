// 2^x of softmax weights: on the multi-function unit, and for pairs on the FMA
// pipe.
#pragma once
#include <cuda_runtime.h>

#include "common/ptx.cuh"

namespace b200 {

// 2^x on the multi-function unit.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x for a pair on the FMA / integer pipes, taking load off the
// multi-function unit: x is clamped to >= -125; adding 1.5 * 2^23 rounds x to
// the nearest integer n (the sum's low mantissa bits hold n: the standard
// magic-constant rounding), f = x - n lies in [-0.5, 0.5]; 2^f comes from a
// degree-3 polynomial fitted for the attention kernels (max relative error 7.5e-5, far
// below the bf16 rounding of P) and 2^n is applied by adding n to the
// exponent field (the construction of N. Schraudolph, "A fast, compact
// approximation of the exponential function", Neural Computation 11(4),
// 1999). p in [0.70, 1.42] and n >= -125 keep the exponent field positive;
// masked scores (-inf) clamp to 2^-125, which P's bf16 keeps as ~2.4e-38.
__device__ __forceinline__ void exp2_fma_pair(float& a, float& b) {
  a = fmaxf(a, -125.f);
  b = fmaxf(b, -125.f);
  const uint64_t xv = f32x2_pack(a, b);
  const uint64_t t = f32x2_add(xv, f32x2_pack(12582912.f, 12582912.f));
  const uint64_t n = f32x2_add(t, f32x2_pack(-12582912.f, -12582912.f));
  const uint64_t f = f32x2_fma(n, f32x2_pack(-1.f, -1.f), xv);
  uint64_t q = f32x2_fma(f, f32x2_pack(0.055171650f, 0.055171650f),
                         f32x2_pack(0.24261114f, 0.24261114f));
  q = f32x2_fma(q, f, f32x2_pack(0.69326097f, 0.69326097f));
  q = f32x2_fma(q, f, f32x2_pack(0.99992806f, 0.99992806f));
  float t0, t1, q0, q1;
  f32x2_unpack(t, t0, t1);
  f32x2_unpack(q, q0, q1);
  a = __int_as_float(__float_as_int(q0) + (__float_as_int(t0) << 23));
  b = __int_as_float(__float_as_int(q1) + (__float_as_int(t1) << 23));
}

}  // namespace b200
