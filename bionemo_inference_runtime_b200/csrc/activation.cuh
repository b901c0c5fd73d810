// Activations of the dense layers and their slopes, for pairs of values in 32 bits.
//
// Functions of the logistic kind cost two special-function operations a value (one exponential, one reciprocal), and that
// unit does 16 a clock and SM: with one reciprocal for a pair, 1 / (p q) times q and p, they cost one and a half.  The
// exponent is held below 62, so that the product of two terms stays finite, and what multiplies a sigmoid that small is held
// above -44: the products are below 2^-56 where the formulas give zero.  NaN stays in its own value (the exponent's bound
// drops it, the other factor keeps it).  Sums and products are made in packed pairs, which halves their issue slots.
// Results agree with the formulas to a few units of the last place of 32 bits; gelu's probability p(z) does in absolute terms
// only (see normal2).
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace b200ta {

enum Activation { kActNone = 0, kActRelu, kActSilu, kActGelu, kActGeluTanh, kActSigmoid, kActCount };

#ifdef __CUDACC__

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // the larger one, NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float keep_nan(float z, float value) { return z == z ? value : z; }
struct F2 {
  uint64_t v;
  F2() = default;
  __device__ __forceinline__ F2(float a, float b) : v(pack_f32x2(a, b)) {}
  __device__ __forceinline__ explicit F2(float a) : v(pack_f32x2(a, a)) {}
  __device__ __forceinline__ explicit F2(uint64_t x) : v(x) {}
  __device__ __forceinline__ void to(float& a, float& b) const { unpack_f32x2(v, a, b); }
};
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { return F2(mul_f32x2(a.v, b.v)); }
__device__ __forceinline__ F2 operator+(F2 a, F2 b) { return F2(add_f32x2(a.v, b.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { return F2(fma_f32x2(a.v, b.v, c.v)); }

// sigmoid(z) of two values; a NaN gives a number between 0 and 1.
__device__ __forceinline__ F2 sigmoid2(F2 z) {
  constexpr float kLog2e = 1.4426950408889634f, kMost = 62.f;
  float t0, t1, p, q;
  (z * F2(-kLog2e)).to(t0, t1);
  (F2(ex2_approx(fminf(t0, kMost)), ex2_approx(fminf(t1, kMost))) + F2(1.f)).to(p, q);
  const float r = rcp_approx(p * q);
  return F2(r * q, r * p);
}
__device__ __forceinline__ F2 held(float z0, float z1) { return F2(max_nan(z0, -44.f), max_nan(z1, -44.f)); }

// The normal distribution's p(z) = (1 + erf(z / sqrt 2)) / 2 and its density for two values: the rational approximation 7.1.26 of
// Abramowitz and Stegun's handbook, erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2) with t = 1 / (1 + 0.3275911 x), whose error is below
// 1.5e-7 (and falls with exp(-x^2)): one exponential, which is the density's, and a reciprocal for the pair.  (With erff() a
// kernel of 15 million values took 41 us, with this 33.)  For p that is 7.5e-8 beside its roundings.  Below zero, where p itself
// becomes small, its relative error grows: 3e-6 at z = -2, 6e-5 at -3, 5e-4 at -4 (where 1 + erf in 32 bits has 6e-4), 4e-3 at -6
// (where that has lost every bit); half a spacing of fp16 is 5e-4, of bf16 4e-3.  A NaN gives some number; z times it is NaN.
__device__ __forceinline__ void normal2(float z0, float z1, F2& p, F2& density) {
  constexpr float kP = 0.3275911f * 0.70710678118654752f, kHalfLog2e = 0.72134752044448170f, kDensity = 0.39894228040143268f;
  // a factor 1 / 2 is part of the coefficients
  constexpr float kA1 = 0.5f * 0.254829592f, kA2 = -0.5f * 0.284496736f, kA3 = 0.5f * 1.421413741f, kA4 = -0.5f * 1.453152027f,
                  kA5 = 0.5f * 1.061405429f;
  const float x0 = fminf(fabsf(z0), 14.f), x1 = fminf(fabsf(z1), 14.f);  // (the exponential is zero there)
  const F2 x(x0, x1);
  float q0, q1, e0, e1, h0, h1;
  fma2(x, F2(kP), F2(1.f)).to(q0, q1);
  const float r = rcp_approx(q0 * q1);
  const F2 t(r * q1, r * q0);
  (x * x * F2(-kHalfLog2e)).to(e0, e1);
  const F2 e(ex2_approx(e0), ex2_approx(e1));
  const F2 poly = fma2(t, fma2(t, fma2(t, fma2(t, F2(kA5), F2(kA4)), F2(kA3)), F2(kA2)), F2(kA1));
  (poly * t * e).to(h0, h1);  // p(-|z|)
  p = F2(z0 < 0.f ? h0 : 1.f - h0, z1 < 0.f ? h1 : 1.f - h1);
  density = e * F2(kDensity);
}

// a = act(z) and, with kSlope, s = act'(z), for two values.
template <int kAct, bool kSlope>
__device__ __forceinline__ void activate2(float z0, float z1, float& a0, float& a1, float& s0, float& s1) {
  if constexpr (kAct == kActNone) {
    a0 = z0, a1 = z1;
    if (kSlope) s0 = 1.f, s1 = 1.f;
  } else if constexpr (kAct == kActRelu) {
    a0 = max_nan(z0, 0.f), a1 = max_nan(z1, 0.f);
    if (kSlope) s0 = z0 > 0.f ? 1.f : 0.f, s1 = z1 > 0.f ? 1.f : 0.f;
  } else if constexpr (kAct == kActSigmoid) {
    const F2 p = sigmoid2(F2(z0, z1));
    p.to(a0, a1);
    a0 = keep_nan(z0, a0), a1 = keep_nan(z1, a1);
    if (kSlope) s0 = fmaf(-a0, a0, a0), s1 = fmaf(-a1, a1, a1);
  } else if constexpr (kAct == kActSilu) {
    const F2 p = sigmoid2(F2(z0, z1)), a = held(z0, z1) * p;
    a.to(a0, a1);
    if (kSlope) fma2(a, fma2(p, F2(-1.f), F2(1.f)), p).to(s0, s1);
  } else if constexpr (kAct == kActGelu) {
    F2 p, density;
    normal2(z0, z1, p, density);
    (F2(z0, z1) * p).to(a0, a1);
    if (kSlope) {
      // held where the density is zero, so that z times it stays finite
      fma2(F2(fminf(fmaxf(z0, -14.f), 14.f), fminf(fmaxf(z1, -14.f), 14.f)), density, p).to(s0, s1);
      s0 = keep_nan(z0, s0), s1 = keep_nan(z1, s1);
    }
  } else {
    // 0.5 (1 + tanh u) = sigmoid(2 u), u = c (z + k z^3)
    constexpr float kTwoC = 1.5957691216057308f, kK = 0.044715f;
    const F2 z(z0, z1), p = sigmoid2(z * fma2(z * F2(kTwoC * kK), z, F2(kTwoC)));
    (held(z0, z1) * p).to(a0, a1);
    if (kSlope) {
      // beyond 10 the slope is 0 or 1: p (1 - p) is zero there, and its factor is kept finite
      const F2 c(fminf(fmaxf(z0, -10.f), 10.f), fminf(fmaxf(z1, -10.f), 10.f));
      fma2(c * fma2(c * F2(3.f * kTwoC * kK), c, F2(kTwoC)), fma2(p * F2(-1.f), p, p), p).to(s0, s1);
      s0 = keep_nan(z0, s0), s1 = keep_nan(z1, s1);
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
