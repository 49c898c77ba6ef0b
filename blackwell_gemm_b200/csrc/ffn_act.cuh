// Activations of the feed-forward operators and their slopes, in fp32.
//
//   relu max(z, 0); silu z s(z); gelu z Phi(z); gelu_tanh z s(2c (z + 0.044715 z^3)), which
//   is the tanh form 0.5 z (1 + tanh(c (z + ..))), c = sqrt(2 / pi); sigmoid s(z).
//
// s is the logistic function, Phi the normal distribution's.  Everything keeps its
// relative precision where it is small: Phi(-x) as a value of its own (1 + erf cancels),
// 1 - s(z) as s(-z) in the slopes.  An exponential and a reciprocal a value, both of the
// special function unit: off by about 2^-22 (1 + the exponent) of the value, where the
// 16-bit outputs round by 2^-8 or 2^-11.
//
// Which activation is a template argument, chosen by with_act once per tile: a branch per
// four values took 200 cycles each (8191 x 8192 x 2048 with silu: 227 us, 183 without).
#pragma once
#include <stdint.h>

#include "b200_ffn.h"

namespace b200 {

template <int kValue>
struct ActCode {
  static constexpr int value = kValue;
};

template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case B200_ACT_RELU: f(ActCode<B200_ACT_RELU>()); break;
    case B200_ACT_SILU: f(ActCode<B200_ACT_SILU>()); break;
    case B200_ACT_GELU: f(ActCode<B200_ACT_GELU>()); break;
    case B200_ACT_GELU_TANH: f(ActCode<B200_ACT_GELU_TANH>()); break;
    case B200_ACT_SIGMOID: f(ActCode<B200_ACT_SIGMOID>()); break;
    default: f(ActCode<B200_ACT_NONE>()); break;
  }
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kRoot2OverPi = 0.7978845608028654f;

// (results below 2^-126 become zero)
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float logistic(float z) {
  return fast_rcp(1.0f + fast_exp2(z * -kLog2E));
}

// s(z) and 1 - s(z) = s(-z), neither by cancellation.
__device__ __forceinline__ void logistic_both(float z, float* s, float* rest) {
  const float e = fast_exp2(fabsf(z) * -kLog2E);
  const float big = fast_rcp(1.0f + e), small = e * big;
  *s = z < 0.0f ? small : big;
  *rest = z < 0.0f ? big : small;
}

// Phi(z), and exp(-z^2 / 2) on the way: Phi(-x) exp(x^2 / 2) is smooth in t =
// 1 / (1 + 0.36 x) over [0, inf); t times a polynomial of degree 6, fitted to it with
// equal relative errors (Lawson's weights), is off by 9e-7 of the value at most.
__device__ __forceinline__ float normal_cdf(float z, float* bell) {
  const float t = fast_rcp(fmaf(0.36f, fabsf(z), 1.0f));
  float p = 0.0470560668f;
  p = fmaf(p, t, -0.179763946f);
  p = fmaf(p, t, 0.180953029f);
  p = fmaf(p, t, 0.0265499685f);
  p = fmaf(p, t, 0.139719047f);
  p = fmaf(p, t, 0.141772489f);
  p = fmaf(p, t, 0.143713043f);
  *bell = fast_exp2(z * z * (-0.5f * kLog2E));
  const float tail = p * t * *bell;
  return z < 0.0f ? tail : 1.0f - tail;
}

__device__ __forceinline__ float tanh_argument(float z) {
  return 2.0f * kRoot2OverPi * z * fmaf(0.044715f * z, z, 1.0f);
}

// v = act(v)
template <int kAct, int kN>
__device__ __forceinline__ void activate(float (&v)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    if constexpr (kAct == B200_ACT_RELU) {
      v[i] = v[i] < 0.0f ? 0.0f : v[i];  // (NaN stays)
    } else if constexpr (kAct == B200_ACT_SILU) {
      v[i] *= logistic(v[i]);
    } else if constexpr (kAct == B200_ACT_GELU) {
      float bell;
      v[i] *= normal_cdf(v[i], &bell);
    } else if constexpr (kAct == B200_ACT_GELU_TANH) {
      v[i] *= logistic(tanh_argument(v[i]));
    } else if constexpr (kAct == B200_ACT_SIGMOID) {
      v[i] = logistic(v[i]);
    }
  }
}

// a = act(z), slope = act'(z).
template <int kAct, int kN>
__device__ __forceinline__ void activate_slope(const float (&z)[kN], float (&a)[kN],
                                               float (&slope)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    if constexpr (kAct == B200_ACT_RELU) {
      a[i] = z[i] < 0.0f ? 0.0f : z[i];
      slope[i] = z[i] > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (kAct == B200_ACT_SILU) {
      float s, r;
      logistic_both(z[i], &s, &r);
      a[i] = z[i] * s;
      slope[i] = fmaf(a[i], r, s);
    } else if constexpr (kAct == B200_ACT_GELU) {
      float bell;
      const float p = normal_cdf(z[i], &bell);
      a[i] = z[i] * p;
      slope[i] = fmaf(z[i] * 0.39894228040143268f, bell, p);
    } else if constexpr (kAct == B200_ACT_GELU_TANH) {
      float s, r;
      logistic_both(tanh_argument(z[i]), &s, &r);
      a[i] = z[i] * s;
      slope[i] = fmaf(a[i] * r, 2.0f * kRoot2OverPi * fmaf(0.134145f * z[i], z[i], 1.0f), s);
    } else if constexpr (kAct == B200_ACT_SIGMOID) {
      float r;
      logistic_both(z[i], &a[i], &r);
      slope[i] = a[i] * r;
    } else {
      a[i] = z[i];
      slope[i] = 1.0f;
    }
  }
}

}  // namespace b200
