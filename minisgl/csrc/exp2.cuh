// Exponentials and packed fp32 arithmetic of the softmax loops.
#pragma once

#include "common.cuh"

namespace minisgl {

// 2^x on the special-function unit (PTX ex2.approx.ftz: relative error of a
// few ulp, ex2(-inf) = +0).
__device__ __forceinline__ float ex2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed fp32 pairs (sm_100 f32x2 arithmetic: one instruction for two lanes
// of work) for the softmax inner loop.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair of arguments on the FMA pipe, to take part of a softmax's
// exponentials off the special-function unit (which otherwise bounds it).
// Method: x = n + f with n = round(x) (adding and subtracting 1.5 * 2^23
// rounds to the nearest integer and leaves n in the low mantissa bits),
// f in [-1/2, 1/2]; 2^f by a cubic fitted here for minimal relative error
// on [-1/2, 1/2] (Lawson-weighted least squares; max relative error 7.5e-5,
// far below the 2^-8 of the bf16 P it feeds); 2^n added to the exponent
// field as n << 23. Arguments are clamped at -126 so that field stays in
// range: 2^-126 and below all come out as about 1e-38 instead of 0, which
// adds nothing measurable to a softmax whose largest term is at least 1.
__device__ __forceinline__ void exp2_poly_pair(uint64_t x2, float& y0, float& y1) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23
  float x0, x1;
  f2_unpack(x2, x0, x1);
  x2 = f2_pack(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t t = f2_add(x2, f2_pack(kRound, kRound));
  const uint64_t r = f2_add(t, f2_pack(-kRound, -kRound));
  const uint64_t f = f2_fma(r, f2_pack(-1.f, -1.f), x2);
  uint64_t q = f2_fma(f, f2_pack(0.05517132f, 0.05517132f), f2_pack(0.24261054f, 0.24261054f));
  q = f2_fma(q, f, f2_pack(0.69326097f, 0.69326097f));
  q = f2_fma(q, f, f2_pack(0.99992812f, 0.99992812f));
  float q0, q1, t0, t1;
  f2_unpack(q, q0, q1);
  f2_unpack(t, t0, t1);
  y0 = __uint_as_float(__float_as_uint(q0) + (__float_as_uint(t0) << 23));
  y1 = __uint_as_float(__float_as_uint(q1) + (__float_as_uint(t1) << 23));
}

}  // namespace minisgl
