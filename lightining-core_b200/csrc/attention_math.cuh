// Softmax arithmetic shared by the tcgen05 attention kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lcb {

// 2^x with the hardware approximation (MUFU ex2, flush-to-zero): P is rounded to bf16 right
// after, and results below 2^-126 are irrelevant to a softmax weight.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed fp32x2 arithmetic and the 3-input max of sm_100: half the FP instructions per score.
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpk2(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2^x for a pair of scores on the FMA pipes instead of MUFU: x = i + f with i = rint(x) (adding
// and subtracting 1.5 * 2^23), f in [-0.5, 0.5]; 2^f by a degree-3 polynomial whose coefficients
// are a weighted-least-squares minimax fit of 2^f on that interval (relative error 7.5e-5, far
// below the bf16 rounding of P); 2^i is added into the exponent field.  x is clamped at -125 so
// the result stays a normal number (a masked score gives 2^-125 instead of 0).
__device__ __forceinline__ void exp2_poly_pair(float x0, float x1, float& y0, float& y1) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23
  const uint64_t xx = pk2(fmaxf(x0, -125.0f), fmaxf(x1, -125.0f));
  const uint64_t t = add2(xx, pk2(kRound, kRound));
  const uint64_t r = add2(t, pk2(-kRound, -kRound));
  const uint64_t f = fma2(r, pk2(-1.0f, -1.0f), xx);
  uint64_t q = fma2(pk2(0.05517132207751274f, 0.05517132207751274f), f,
                    pk2(0.24261054396629333f, 0.24261054396629333f));
  q = fma2(q, f, pk2(0.6932609677314758f, 0.6932609677314758f));
  q = fma2(q, f, pk2(0.9999281167984009f, 0.9999281167984009f));
  float q0, q1, t0, t1;
  unpk2(q, q0, q1);
  unpk2(t, t0, t1);
  y0 = __uint_as_float(__float_as_uint(q0) + (__float_as_uint(t0) << 23));
  y1 = __uint_as_float(__float_as_uint(q1) + (__float_as_uint(t1) << 23));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// x rounded to tf32 (half a unit added to the magnitude, 13 low bits cleared); x - that is exact in fp32.
__device__ __forceinline__ float tf32_round(float x) {
  uint32_t u = __float_as_uint(x);
  if ((u & 0x7f800000u) != 0x7f800000u) u = (u + 0x1000u) & 0xffffe000u;
  return __uint_as_float(u);
}

}  // namespace lcb
