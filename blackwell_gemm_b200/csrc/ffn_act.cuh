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
// four values took 200 cycles each (8191 rows x 8192 x 2048 with bias and gelu_tanh 227 us,
// 183 so).
#pragma once
#include <stdint.h>

#include "b200_ffn.h"
#include "sm100_ptx.cuh"

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

// s(z) and 1 - s(z) = s(-z), neither by cancellation.
__device__ __forceinline__ void logistic_both(float z, float* s, float* rest) {
  const float e = fast_exp2(fabsf(z) * -kLog2E);
  const float big = fast_rcp(1.0f + e), small = e * big;
  *s = z < 0.0f ? small : big;
  *rest = z < 0.0f ? big : small;
}

// Phi(z), and exp(-z^2 / 2) on the way: Phi(-x) exp(x^2 / 2) is smooth in t =
// 1 / (1 + 0.36 x); t times a polynomial of degree 6, fitted to it with equal relative
// errors (Lawson's weights), is off by 9e-7 of the value at most up to x = 14.  (From 13.2
// on the exponential is below 2^-126 and taken for zero.)
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

// The same for two values at a time, where instructions are what is short (the products'
// epilogues).
__device__ __forceinline__ F32x2 both(float v) { return pair_of(v, v); }
__device__ __forceinline__ F32x2 exp2_pair(F32x2 x) {
  float a, b;
  halves_of(x, a, b);
  return pair_of(fast_exp2(a), fast_exp2(b));
}
__device__ __forceinline__ F32x2 rcp_pair(F32x2 x) {
  float a, b;
  halves_of(x, a, b);
  return pair_of(fast_rcp(a), fast_rcp(b));
}
// s(-z / log2(e))
__device__ __forceinline__ F32x2 logistic_pair(F32x2 exponent) {
  return rcp_pair(add2(exp2_pair(exponent), both(1.0f)));
}
__device__ __forceinline__ F32x2 normal_cdf_pair(F32x2 z) {
  float a, b, t0, t1;
  halves_of(z, a, b);
  const F32x2 t = rcp_pair(fma2(pair_of(fabsf(a), fabsf(b)), both(0.36f), both(1.0f)));
  F32x2 p = fma2(both(0.0470560668f), t, both(-0.179763946f));
  p = fma2(p, t, both(0.180953029f));
  p = fma2(p, t, both(0.0265499685f));
  p = fma2(p, t, both(0.139719047f));
  p = fma2(p, t, both(0.141772489f));
  p = fma2(p, t, both(0.143713043f));
  const F32x2 bell = exp2_pair(mul2(mul2(z, z), both(-0.5f * kLog2E)));
  halves_of(mul2(mul2(p, t), bell), t0, t1);
  return pair_of(a < 0.0f ? t0 : 1.0f - t0, b < 0.0f ? t1 : 1.0f - t1);
}

// v = act(v); kN even, or 1.
template <int kAct, int kN>
__device__ __forceinline__ void activate(float (&v)[kN]) {
  if constexpr (kAct == B200_ACT_NONE) return;
  if constexpr (kN == 1) {
    float two[2] = {v[0], v[0]};
    activate<kAct>(two);
    v[0] = two[0];
  } else {
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      if constexpr (kAct == B200_ACT_RELU) {
        v[i] = v[i] < 0.0f ? 0.0f : v[i];  // (NaN stays)
        v[i + 1] = v[i + 1] < 0.0f ? 0.0f : v[i + 1];
      } else {
        const F32x2 z = pair_of(v[i], v[i + 1]);
        F32x2 r;
        if constexpr (kAct == B200_ACT_SILU) {
          r = mul2(z, logistic_pair(mul2(z, both(-kLog2E))));
        } else if constexpr (kAct == B200_ACT_GELU) {
          r = mul2(z, normal_cdf_pair(z));
        } else if constexpr (kAct == B200_ACT_GELU_TANH) {
          constexpr float kScale = -2.0f * kRoot2OverPi * kLog2E;
          const F32x2 y = mul2(z, fma2(mul2(z, both(0.044715f * kScale)), z, both(kScale)));
          r = mul2(z, logistic_pair(y));
        } else {
          r = logistic_pair(mul2(z, both(-kLog2E)));
        }
        halves_of(r, v[i], v[i + 1]);
      }
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
      // (held at 200, |z| = 67: s r is zero from there on, and stays a factor of something finite)
      const float q = fminf(0.044715f * z[i] * z[i], 200.0f), y = 2.0f * kRoot2OverPi * z[i];
      float s, r;
      logistic_both(fmaf(y, q, y), &s, &r);
      a[i] = z[i] * s;
      slope[i] = fmaf(a[i] * r, fmaf(6.0f * kRoot2OverPi, q, 2.0f * kRoot2OverPi), s);
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

// d act'(z).  relu lets through or not: what comes back to a unit that it shuts is zero
// whatever arrives, where inf * 0 would be NaN.
template <int kAct>
__device__ __forceinline__ float times_slope(float d, float slope) {
  if constexpr (kAct == B200_ACT_RELU) return slope > 0.0f ? d : 0.0f;
  return d * slope;
}

}  // namespace b200
