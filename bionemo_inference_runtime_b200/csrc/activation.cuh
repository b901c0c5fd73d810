// Activations of the dense layers and their slopes, for pairs of values in 32 bits.
//
// Functions of the logistic kind cost two special-function operations a value (one exponential, one reciprocal), and that
// unit does 16 a clock and SM: with one reciprocal for a pair, 1 / (p q) times q and p, they cost one and a half.
// The exponent is held below 62, so that the product of two terms stays finite; past it the result is below 2^-62 and
// taken as zero, which also keeps z * sigmoid(z) zero where z is large.  Results agree with the formulas to a few units of
// the last place of 32 bits.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace b200ta {

enum Activation { kActNone = 0, kActRelu, kActSilu, kActGelu, kActGeluTanh, kActSigmoid, kActCount };

#ifdef __CUDACC__

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// sigmoid(z) of two values.  A NaN gives some number between 0 and 1; what is made of it here is multiplied by z or passed
// through keep_nan().
__device__ __forceinline__ void sigmoid2(float z0, float z1, float& s0, float& s1) {
  constexpr float kLog2e = 1.4426950408889634f, kMost = 62.f;
  const float t0 = -kLog2e * z0, t1 = -kLog2e * z1;
  const float p = 1.f + ex2_approx(fminf(t0, kMost)), q = 1.f + ex2_approx(fminf(t1, kMost));
  const float r = rcp_approx(p * q);
  s0 = t0 >= kMost ? 0.f : r * q;
  s1 = t1 >= kMost ? 0.f : r * p;
}
__device__ __forceinline__ float keep_nan(float z, float value) { return z == z ? value : z; }

// a = act(z) and, with kSlope, s = act'(z), for two values.
template <int kAct, bool kSlope>
__device__ __forceinline__ void activate2(float z0, float z1, float& a0, float& a1, float& s0, float& s1) {
  if constexpr (kAct == kActNone) {
    a0 = z0, a1 = z1;
    if (kSlope) s0 = 1.f, s1 = 1.f;
  } else if constexpr (kAct == kActRelu) {
    a0 = z0 < 0.f ? 0.f : z0, a1 = z1 < 0.f ? 0.f : z1;  // a NaN stays
    if (kSlope) s0 = z0 > 0.f ? 1.f : 0.f, s1 = z1 > 0.f ? 1.f : 0.f;
  } else if constexpr (kAct == kActSigmoid) {
    sigmoid2(z0, z1, a0, a1);
    a0 = keep_nan(z0, a0), a1 = keep_nan(z1, a1);
    if (kSlope) s0 = a0 * (1.f - a0), s1 = a1 * (1.f - a1);
  } else if constexpr (kAct == kActSilu) {
    float p0, p1;
    sigmoid2(z0, z1, p0, p1);
    a0 = z0 * p0, a1 = z1 * p1;
    if (kSlope) s0 = fmaf(a0, 1.f - p0, p0), s1 = fmaf(a1, 1.f - p1, p1);
  } else if constexpr (kAct == kActGelu) {
    constexpr float kRsqrt2 = 0.70710678118654752f, kDensity = 0.39894228040143268f, kHalfLog2e = 0.72134752044448170f;
    const float p0 = fmaf(0.5f, erff(z0 * kRsqrt2), 0.5f), p1 = fmaf(0.5f, erff(z1 * kRsqrt2), 0.5f);
    a0 = z0 * p0, a1 = z1 * p1;
    if (kSlope) {
      // past 13 the density is below 2^-121; held there, z times it is zero for every larger z
      const float c0 = fminf(fmaxf(z0, -13.f), 13.f), c1 = fminf(fmaxf(z1, -13.f), 13.f);
      s0 = keep_nan(z0, fmaf(c0, kDensity * ex2_approx(-kHalfLog2e * c0 * c0), p0));
      s1 = keep_nan(z1, fmaf(c1, kDensity * ex2_approx(-kHalfLog2e * c1 * c1), p1));
    }
  } else {
    // 0.5 (1 + tanh u) = sigmoid(2 u), u = c (z + k z^3)
    constexpr float kTwoC = 1.5957691216057308f, kK = 0.044715f;
    float p0, p1;
    sigmoid2(z0 * fmaf(kTwoC * kK * z0, z0, kTwoC), z1 * fmaf(kTwoC * kK * z1, z1, kTwoC), p0, p1);
    a0 = z0 * p0, a1 = z1 * p1;
    if (kSlope) {
      // beyond 10 the slope is 0 or 1: p (1 - p) is zero there, and its factor is kept finite
      const float c0 = fminf(fmaxf(z0, -10.f), 10.f), c1 = fminf(fmaxf(z1, -10.f), 10.f);
      s0 = keep_nan(z0, fmaf(c0 * fmaf(3.f * kTwoC * kK * c0, c0, kTwoC), p0 * (1.f - p0), p0));
      s1 = keep_nan(z1, fmaf(c1 * fmaf(3.f * kTwoC * kK * c1, c1, kTwoC), p1 * (1.f - p1), p1));
    }
  }
}

// ---- 16-bit pairs -------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (sizeof(T) == 2 && !__is_same(T, __half))
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (__is_same(T, __half))
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else
    return make_float2(bf16_lo(v), bf16_hi(v));
}

#endif  // __CUDACC__
}  // namespace b200ta
