// Activations of the expert layers in f32, and their derivatives.
//
// Relative errors in units of 2^-23, which results of 16 bits (2^-11 at best) do not show: silu 5
// above 0 and 4 + 0.62 |v| below (58 at -87: the exp's argument is rounded first); gelu 5.4e-6 of
// its fit and 9 + 0.56 v^2 units below 0 (1.8e-5 at -13). silu is 0 below -87.3 and gelu below
// -13.2, where they are less than 1.1e-36. act(0) is 0 for each.
#pragma once

#include <cuda_runtime.h>

#include "lgbm_b200.h"

namespace lgbm_b200 {
namespace experts {

// e^v and 1 / v, one instruction of the special function unit each (the exp's argument is scaled
// first), results below 2^-126 as 0. What calls for subnormals in expf and in a division took four
// times as many instructions, and an epilogue has two of these for every output.
__device__ __forceinline__ float exp_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.44269504f));
  return r;
}
__device__ __forceinline__ float inverse_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// The larger and the smaller of two numbers; NaN stays NaN.
__device__ __forceinline__ float not_below(float v, float least) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(least));
  return r;
}
__device__ __forceinline__ float not_above(float v, float most) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(most));
  return r;
}
constexpr float kLargest = 3.402823466e38f;

// value(v), and both: the value a and the slope d of what was saved. A product beyond f16's range
// is saved as an infinity, so at infinities both() gives its limits: d 1 and a infinite above, d
// and a 0 below.
template <int ACT>
struct Act;

template <>
struct Act<LGBM_B200_ACT_NONE> {
  static __device__ __forceinline__ float value(float v) { return v; }
  static __device__ __forceinline__ void both(float v, float& a, float& d) {
    a = v;
    d = 1.0f;
  }
};

// NaN stays NaN; the slope at 0 is 0.
template <>
struct Act<LGBM_B200_ACT_RELU> {
  static __device__ __forceinline__ float value(float v) { return v < 0.0f ? 0.0f : v; }
  static __device__ __forceinline__ void both(float v, float& a, float& d) {
    a = value(v);
    d = v > 0.0f ? 1.0f : v <= 0.0f ? 0.0f : v;
  }
};

// v s(v), s = 1 / (1 + e^-v): 0 where s is below 2^-126.
template <>
struct Act<LGBM_B200_ACT_SILU> {
  static __device__ __forceinline__ float value(float v) {
    return v * inverse_fast(1.0f + exp_fast(-v));
  }
  static __device__ __forceinline__ void both(float v, float& a, float& d) {
    const float s = inverse_fast(1.0f + exp_fast(-v)), lo = not_below(v, -kLargest);
    a = lo * s;
    d = s * fmaf(not_above(lo, kLargest), 1.0f - s, 1.0f);
  }
};

// v P(v), P the distribution function of the normal law. With t = 1 / (1 + q |v|) (Hastings'
// form, 1955) the tail 1 - P(|v|) = e^(-v^2 / 2) (a1 t + .. + a6 t^6): coefficients fitted for the
// smallest largest relative error on |v| <= 17, 5.4e-6. 1 + erf(v) would leave nothing of P at
// v < -5, and erfcf takes twice the instructions.
template <>
struct Act<LGBM_B200_ACT_GELU> {
  static __device__ __forceinline__ float tail(float v, float e) {
    const float t = inverse_fast(fmaf(0.311f, fabsf(v), 1.0f));
    float s = fmaf(-0.0731476133f, t, 0.175886592f);
    s = fmaf(s, t, 0.0198684974f);
    s = fmaf(s, t, 0.13196364f);
    s = fmaf(s, t, 0.121193485f);
    s = fmaf(s, t, 0.124232849f);
    return s * t * e;
  }
  static __device__ __forceinline__ float value(float v) {
    const float p = tail(v, exp_fast(-0.5f * v * v));
    return v * (v < 0.0f ? p : 1.0f - p);
  }
  static __device__ __forceinline__ void both(float v, float& a, float& d) {
    const float e = exp_fast(-0.5f * v * v), q = tail(v, e), p = v < 0.0f ? q : 1.0f - q;
    const float lo = not_below(v, -kLargest);
    a = lo * p;
    d = fmaf(not_above(lo, kLargest) * 0.39894228f, e, p);  // 1 / sqrt(2 pi)
  }
};

template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
  if (act == LGBM_B200_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Act<LGBM_B200_ACT_SILU>::value(v[i]);
  } else if (act == LGBM_B200_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Act<LGBM_B200_ACT_GELU>::value(v[i]);
  } else if (act == LGBM_B200_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Act<LGBM_B200_ACT_RELU>::value(v[i]);
  }
}

// Values a and slopes d.
template <int N>
__device__ __forceinline__ void activate_both(int act, const float (&v)[N], float (&a)[N],
                                              float (&d)[N]) {
  if (act == LGBM_B200_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) Act<LGBM_B200_ACT_SILU>::both(v[i], a[i], d[i]);
  } else if (act == LGBM_B200_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) Act<LGBM_B200_ACT_GELU>::both(v[i], a[i], d[i]);
  } else if (act == LGBM_B200_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) Act<LGBM_B200_ACT_RELU>::both(v[i], a[i], d[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) Act<LGBM_B200_ACT_NONE>::both(v[i], a[i], d[i]);
  }
}

}  // namespace experts
}  // namespace lgbm_b200
