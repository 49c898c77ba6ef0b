// Activations of the feed-forward operators and their slopes, in fp32.
//
//   relu max(z, 0); silu z s(z); gelu z Phi(z); gelu_tanh z s(2c (z + 0.044715 z^3)), which
//   is the tanh form 0.5 z (1 + tanh(c (z + ..))), c = sqrt(2 / pi); sigmoid s(z).
//
// s is the logistic function.  Everything is written so that small values keep
// their relative precision: Phi by erfc (1 + erf cancels for z < 0), 1 - s(z) as
// s(-z) in the slopes.  The fast exponential and division err by about 2^-21 of
// the value where the 16-bit outputs round by 2^-9 or 2^-12.
#pragma once
#include <stdint.h>

#include "b200_ffn.h"

namespace b200 {

constexpr float kRoot2OverPi = 0.7978845608028654f;

__device__ __forceinline__ float logistic(float z) {
  return __fdividef(1.0f, 1.0f + __expf(-z));
}

// s(z) and 1 - s(z) = s(-z), neither by cancellation.
__device__ __forceinline__ void logistic_both(float z, float* s, float* rest) {
  const float e = __expf(-fabsf(z));
  const float big = __fdividef(1.0f, 1.0f + e), small = e * big;
  *s = z < 0.0f ? small : big;
  *rest = z < 0.0f ? big : small;
}

__device__ __forceinline__ float normal_cdf(float z) {
  return 0.5f * erfcf(z * -0.70710678118654752f);
}

__device__ __forceinline__ float tanh_argument(float z) {
  return 2.0f * kRoot2OverPi * (z + 0.044715f * z * z * z);
}

// v = act(v); `act` is the same for a whole launch.
template <int kN>
__device__ __forceinline__ void activate(int act, float (&v)[kN]) {
  switch (act) {
    case B200_ACT_RELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // (NaN stays)
      break;
    case B200_ACT_SILU:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] *= logistic(v[i]);
      break;
    case B200_ACT_GELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] *= normal_cdf(v[i]);
      break;
    case B200_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] *= logistic(tanh_argument(v[i]));
      break;
    case B200_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = logistic(v[i]);
      break;
    default:
      break;
  }
}

// a = act(z), slope = act'(z).
template <int kN>
__device__ __forceinline__ void activate_slope(int act, const float (&z)[kN], float (&a)[kN],
                                               float (&slope)[kN]) {
  switch (act) {
    case B200_ACT_RELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        a[i] = z[i] < 0.0f ? 0.0f : z[i];
        slope[i] = z[i] > 0.0f ? 1.0f : 0.0f;
      }
      break;
    case B200_ACT_SILU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        float s, r;
        logistic_both(z[i], &s, &r);
        a[i] = z[i] * s;
        slope[i] = s + a[i] * r;
      }
      break;
    case B200_ACT_GELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float p = normal_cdf(z[i]);
        a[i] = z[i] * p;
        slope[i] = p + z[i] * (0.39894228040143268f * __expf(-0.5f * z[i] * z[i]));
      }
      break;
    case B200_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        float s, r;
        logistic_both(tanh_argument(z[i]), &s, &r);
        a[i] = z[i] * s;
        slope[i] = s + a[i] * r * (2.0f * kRoot2OverPi * (1.0f + 0.134145f * z[i] * z[i]));
      }
      break;
    case B200_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        float r;
        logistic_both(z[i], &a[i], &r);
        slope[i] = a[i] * r;
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        a[i] = z[i];
        slope[i] = 1.0f;
      }
      break;
  }
}

}  // namespace b200
