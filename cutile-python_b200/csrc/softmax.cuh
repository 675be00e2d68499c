// Pieces of the online softmax that the tensor-core attention kernels share.
#pragma once
#include <cuda_runtime.h>

namespace b200k {

// A row keeps a stale maximum while the true one is less than 2^8 above it: the factor cancels
// in O / l, and fp32 sums have the range.
constexpr float kRescaleThreshold = 8.0f;  // log2 units

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The larger one, NaN where either is NaN.
__device__ __forceinline__ float fmax_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Every kFmhaPolyEvery-th pair of scores takes its exp2 on the FMA pipe (a degree-3
// polynomial after splitting off the integer part) instead of the special-function unit,
// which is the busiest pipe of the softmax.  Relative error 7.5e-5, far below the rounding
// of P to 16 bits.  0 disables the polynomial path.
//
// Arguments far below zero: without EXACT_ENDS they give 2^-125, which a row that sees something
// does not notice, and NaN gives the largest number, whose rounding to 16 bits is infinite, so that
// the row is not finite either.  With it the power of two is a factor of its own, so that
// arguments from -127 down (a masked score's -inf) give the bits of 2^-127, a zero: rows that see
// nothing keep a sum of zero, and a masked value no weight.  NaN stays NaN.  One more product per pair
// (4 x 64 drafts over 8192 - 32768 keys 127 us as before); the contiguous attention, whose rows all see
// something, keeps the shorter form (4 x 16 heads of 64, 4096 tokens, bf16: 456 us, 468 with the product).
#ifndef B200K_FMHA_POLY
#define B200K_FMHA_POLY 4
#endif
constexpr int kFmhaPolyEvery = B200K_FMHA_POLY;

template <bool EXACT_ENDS = false>
__device__ __forceinline__ float2 exp2_poly_pair(float2 x) {
  const float2 magic = make_float2(12582912.0f, 12582912.0f);       // 1.5 * 2^23
  const float2 neg_magic = make_float2(-12582912.0f, -12582912.0f);
  constexpr float kLeast = EXACT_ENDS ? -127.0f : -125.0f;
  x.x = fmax_or_nan(x.x, kLeast);
  x.y = fmax_or_nan(x.y, kLeast);
  const float2 t = __fadd2_rn(x, magic);            // integer part lands in the low mantissa bits
  const float2 i = __fadd2_rn(t, neg_magic);
  const float2 f = __fadd2_rn(x, make_float2(-i.x, -i.y));   // in [-0.5, 0.5]
  float2 p = __ffma2_rn(make_float2(0.05517164617776871f, 0.05517164617776871f), f,
                        make_float2(0.2426111251115799f, 0.2426111251115799f));
  p = __ffma2_rn(p, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
  p = __ffma2_rn(p, f, make_float2(0.9999280571937561f, 0.9999280571937561f));
  if constexpr (EXACT_ENDS) {
    const int one = 127 << 23;
    return __fmul2_rn(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + one),
                                     __int_as_float((__float_as_int(t.y) << 23) + one)));
  }
  float2 r;
  r.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23));
  r.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23));
  return r;
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace b200k
