// Activations of the feed-forward operators and their derivatives, in fp32.
//
//   relu       max(x, 0)
//   gelu       x Phi(x) = x erfc(-x / sqrt 2) / 2   (erfc, not 1 + erf: no cancellation in the negative tail)
//   gelu_tanh  x sigma(2 u), u = sqrt(2/pi) (x + 0.044715 x^3)   (= x (1 + tanh u) / 2, again without cancellation)
//   silu       x sigma(x)
//
// sigma uses the fast exponential and division: a few 1e-7 relative for |x| < 10 and 1e-6 at 20, far below the
// half step of the bf16 / fp16 results (2^-9, 2^-12 of the value) these are rounded to.
#pragma once
#include <cstdint>
#include "b2x.h"

namespace b2x {

constexpr float kGeluA = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;
constexpr float kSqrtHalf = 0.7071067811865476f;

__device__ __forceinline__ float sigma_fast(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

template <int ACT>
__device__ __forceinline__ float act_fwd(float x) {
  if constexpr (ACT == B2X_ACT_RELU) return x < 0.0f ? 0.0f : x;  // NaN stays NaN
  if constexpr (ACT == B2X_ACT_GELU) return 0.5f * x * erfcf(-x * kSqrtHalf);
  if constexpr (ACT == B2X_ACT_GELU_TANH) return x * sigma_fast(2.0f * kGeluA * (x + kGeluB * x * x * x));
  if constexpr (ACT == B2X_ACT_SILU) return x * sigma_fast(x);
  return x;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float x) {
  if constexpr (ACT == B2X_ACT_RELU) return x > 0.0f ? 1.0f : (x <= 0.0f ? 0.0f : x);  // 0 at 0; NaN stays NaN
  if constexpr (ACT == B2X_ACT_GELU)
    return 0.5f * erfcf(-x * kSqrtHalf) + x * __expf(-0.5f * x * x) * (0.5f * kGeluA);
  if constexpr (ACT == B2X_ACT_GELU_TANH) {
    const float p = sigma_fast(2.0f * kGeluA * (x + kGeluB * x * x * x));
    return p + x * p * (1.0f - p) * (2.0f * kGeluA * (1.0f + 3.0f * kGeluB * x * x));
  }
  if constexpr (ACT == B2X_ACT_SILU) {
    const float p = sigma_fast(x);
    return p + x * p * (1.0f - p);
  }
  return 1.0f;
}

// Values with the activation chosen at run time (uniform over the grid).
template <int N>
__device__ __forceinline__ void act_all(int act, float (&v)[N]) {
  switch (act) {
    case B2X_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_fwd<B2X_ACT_RELU>(v[i]);
      break;
    case B2X_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_fwd<B2X_ACT_GELU>(v[i]);
      break;
    case B2X_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_fwd<B2X_ACT_GELU_TANH>(v[i]);
      break;
    case B2X_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_fwd<B2X_ACT_SILU>(v[i]);
      break;
    default:
      break;
  }
}

// 16-bit and fp32 values as stored.
__device__ __forceinline__ float load_f32(const void* p, int64_t i, int type) {
  if (type == B2X_F32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t u = reinterpret_cast<const uint16_t*>(p)[i];
  return type == B2X_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

}  // namespace b2x
