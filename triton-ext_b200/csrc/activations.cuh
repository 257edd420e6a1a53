// Activations of the feed-forward operators and their derivatives, in fp32, two values at a time.
//
//   relu       max(x, 0)
//   gelu       x Phi(x), Phi(x) = erfc(-x / sqrt 2) / 2
//   gelu_tanh  x sigma(2 u), u = sqrt(2/pi) (x + 0.044715 x^3)   (= x (1 + tanh u) / 2 without its cancellation)
//   silu       x sigma(x)
//
// sigma(x) = 1 / (1 + 2^(-x log2 e)) on the two approximate instructions: a few 1e-7 relative for |x| < 10 and 1e-6 at 20,
// far below the half step of the bf16 / fp16 results (2^-9, 2^-12 of the value) these are rounded to; fp32 slopes of
// these two are made without them (act_slope_f32).  Values below 2^-126 become 0.
//
// erfc(z), z >= 0, is t exp(-z^2 + P(t)) with t = 1 / (1 + z / 2) and the Chebyshev fit P of Press et al., Numerical Recipes,
// section 6.2 (relative error below 1.2e-7 everywhere), so the negative tail of gelu keeps its relative accuracy.
//
// What bounds them is instructions, so products and sums work on pairs (fma.rn.f32x2): with single operations and the
// library's exponential, division and erfc the epilogue's backward pass on 4000 x 28672 took 260 us (gelu 366 us) where
// the memory takes 105.
#pragma once
#include <cstdint>
#include "b2x.h"

namespace b2x {

constexpr float kGeluA = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;
constexpr float kSqrtHalf = 0.7071067811865476f;
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp_approx(float x) { return exp2_approx(x * kLog2E); }
__device__ __forceinline__ float sigma_fast(float x) { return rcp_approx(1.0f + exp2_approx(x * -kLog2E)); }

// A pair of fp32 values in one register pair.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Pair pair(float a) { return pair(a, a); }
__device__ __forceinline__ void unpair(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair exp2_pair(Pair x) {
  float a, b;
  unpair(x, a, b);
  return pair(exp2_approx(a), exp2_approx(b));
}
__device__ __forceinline__ Pair rcp_pair(Pair x) {
  float a, b;
  unpair(x, a, b);
  return pair(rcp_approx(a), rcp_approx(b));
}
// 1 / (1 + 2^x): sigma of -x / log2 e
__device__ __forceinline__ Pair sigma2(Pair x) { return rcp_pair(add2(pair(1.0f), exp2_pair(x))); }

// -2 u log2 e for gelu_tanh, from x and x^2
__device__ __forceinline__ Pair gelu_tanh_arg(Pair x, Pair x2) {
  constexpr float k = -2.0f * kGeluA * kLog2E;
  return mul2(x, fma2(pair(k * kGeluB), x2, pair(k)));
}

// Phi(x) = erfc(-x / sqrt 2) / 2, the normal distribution.
__device__ __forceinline__ Pair normal_cdf(Pair x) {
  float a, b;
  unpair(x, a, b);
  const Pair z = pair(fabsf(a) * kSqrtHalf, fabsf(b) * kSqrtHalf);
  const Pair t = rcp_pair(fma2(z, pair(0.5f), pair(1.0f)));
  Pair q = fma2(t, pair(0.17087277f), pair(-0.82215223f));
  q = fma2(t, q, pair(1.48851587f));
  q = fma2(t, q, pair(-1.13520398f));
  q = fma2(t, q, pair(0.27886807f));
  q = fma2(t, q, pair(-0.18628806f));
  q = fma2(t, q, pair(0.09678418f));
  q = fma2(t, q, pair(0.37409196f));
  q = fma2(t, q, pair(1.00002368f));
  q = fma2(t, q, pair(-1.26551223f));
  const Pair e = exp2_pair(mul2(fma2(z, mul2(z, pair(-1.0f)), q), pair(kLog2E)));
  float c, d;
  unpair(mul2(mul2(t, pair(0.5f)), e), c, d);  // erfc(|x| / sqrt 2) / 2
  return pair(a > 0.0f ? 1.0f - c : c, b > 0.0f ? 1.0f - d : d);
}

template <int ACT>
__device__ __forceinline__ Pair act_fwd(Pair x) {
  if constexpr (ACT == B2X_ACT_RELU) {
    float a, b;
    unpair(x, a, b);
    return pair(a < 0.0f ? 0.0f : a, b < 0.0f ? 0.0f : b);  // NaN stays NaN
  }
  if constexpr (ACT == B2X_ACT_GELU) return mul2(x, normal_cdf(x));
  if constexpr (ACT == B2X_ACT_GELU_TANH) return mul2(x, sigma2(gelu_tanh_arg(x, mul2(x, x))));
  if constexpr (ACT == B2X_ACT_SILU) return mul2(x, sigma2(mul2(x, pair(-kLog2E))));
  return x;
}

template <int ACT>
__device__ __forceinline__ Pair act_slope(Pair x) {
  if constexpr (ACT == B2X_ACT_RELU) {
    float a, b;
    unpair(x, a, b);  // 0 at 0; NaN stays NaN
    return pair(a > 0.0f ? 1.0f : (a <= 0.0f ? 0.0f : a), b > 0.0f ? 1.0f : (b <= 0.0f ? 0.0f : b));
  }
  if constexpr (ACT == B2X_ACT_GELU) {  // Phi(x) + x exp(-x^2 / 2) / sqrt(2 pi)
    const Pair e = exp2_pair(mul2(mul2(x, pair(-0.5f * kLog2E)), x));
    return fma2(mul2(x, pair(0.5f * kGeluA)), e, normal_cdf(x));
  }
  if constexpr (ACT == B2X_ACT_GELU_TANH) {
    // s + x s (1 - s) 2 u': where s is 0 or 1 the product s (1 - s) has to come first, since x (1 - s) 2 u' overflows from
    // |x| of 1e13 on, and x^2 is held below 1e30 to keep 2 u' finite.  NaN and infinities go through the factor x.
    float a, b;
    unpair(mul2(x, x), a, b);
    const Pair x2 = pair(fminf(a, 1e30f), fminf(b, 1e30f)), s = sigma2(gelu_tanh_arg(x, x2));
    const Pair du = fma2(pair(6.0f * kGeluA * kGeluB), x2, pair(2.0f * kGeluA));
    return fma2(mul2(x, mul2(s, fma2(s, pair(-1.0f), pair(1.0f)))), du, s);
  }
  if constexpr (ACT == B2X_ACT_SILU) {  // s (1 + x (1 - s))
    const Pair s = sigma2(mul2(x, pair(-kLog2E)));
    return mul2(s, fma2(x, fma2(s, pair(-1.0f), pair(1.0f)), pair(1.0f)));
  }
  return pair(1.0f);
}

// The slopes of gelu_tanh and silu for fp32 results, to 16 x 2^-24 of their largest value: the library's exponential and a
// true division, and sigma(-x) made beside sigma(x) instead of 1 - sigma(x), which leaves x (1 - sigma(x)) few digits.
// (gelu's is within 12 x 2^-24 as it is; with the library's erfc 4000 x 28672 took 287 us instead of 221.)
template <int ACT>
__device__ __forceinline__ float act_slope_f32(float x) {
  const float x2 = fminf(x * x, 1e30f);
  const float y = ACT == B2X_ACT_SILU ? x : x * fmaf(2.0f * kGeluA * kGeluB, x2, 2.0f * kGeluA);
  const float e = expf(-fabsf(y)), r = __fdiv_rn(1.0f, 1.0f + e);
  const float p = y < 0.0f ? e * r : r, q = y < 0.0f ? r : e * r;  // sigma(y), sigma(-y)
  if constexpr (ACT == B2X_ACT_SILU) return p * fmaf(x, q, 1.0f);
  return fmaf(x * (p * q), fmaf(6.0f * kGeluA * kGeluB, x2, 2.0f * kGeluA), p);
}

template <int ACT, int N>
__device__ __forceinline__ void act_each(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) unpair(act_fwd<ACT>(pair(v[i], v[i + 1])), v[i], v[i + 1]);
}
// Values with the activation chosen at run time (uniform over the grid).
template <int N>
__device__ __forceinline__ void act_all(int act, float (&v)[N]) {
  switch (act) {
    case B2X_ACT_RELU: act_each<B2X_ACT_RELU>(v); break;
    case B2X_ACT_GELU: act_each<B2X_ACT_GELU>(v); break;
    case B2X_ACT_GELU_TANH: act_each<B2X_ACT_GELU_TANH>(v); break;
    case B2X_ACT_SILU: act_each<B2X_ACT_SILU>(v); break;
    default: break;
  }
}

// 16-bit and fp32 values as stored.
__device__ __forceinline__ float load_f32(const void* p, int64_t i, int type) {
  if (type == B2X_F32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t u = reinterpret_cast<const uint16_t*>(p)[i];
  return type == B2X_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

}  // namespace b2x
