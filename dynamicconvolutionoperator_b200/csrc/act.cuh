// Activations of the channel-last operators and their derivatives, FP32.
//   relu       max(z, 0)
//   silu       z / (1 + e^-z)
//   gelu       z * Phi(z), Phi the normal distribution function (erf form)
//   gelu_tanh  z/2 * (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3)))
// kFast (16-bit data) takes the hardware's approximate exponential and
// division: a relative error of about 2^-21, far below the rounding to 16
// bits; FP32 data takes the full-precision functions.
#pragma once

#include "common.cuh"

namespace ddpm {

__host__ inline bool act_known(int act) { return act >= DDPM_ACT_NONE && act <= DDPM_ACT_GELU_TANH; }

template <bool kFast> __device__ __forceinline__ float exp_f(float v) {
  if constexpr (kFast) return __expf(v);
  else return expf(v);
}
template <bool kFast> __device__ __forceinline__ float div_f(float a, float b) {
  // __fdividef returns 0 for divisors above 2^126, which is also the limit of
  // the quotients formed here (1 / (1 + e^-z))
  if constexpr (kFast) return __fdividef(a, b);
  else return a / b;
}

template <bool kFast, int A> __device__ __forceinline__ float act_value(float z) {
  if constexpr (A == DDPM_ACT_RELU) {
    return z < 0.f ? 0.f : z;  // keeps a NaN
  } else if constexpr (A == DDPM_ACT_SILU) {
    // e^-z overflows to infinity for z < -88: the quotient is then -0
    return div_f<kFast>(z, 1.f + exp_f<kFast>(-z));
  } else if constexpr (A == DDPM_ACT_GELU) {
    // erfc keeps the relative precision of the tail below zero
    return 0.5f * z * erfcf(-0.70710678118654752f * z);
  } else if constexpr (A == DDPM_ACT_GELU_TANH) {
    const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
    // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
    return div_f<kFast>(z, 1.f + exp_f<kFast>(-2.f * u));
  } else {
    return z;
  }
}

template <bool kFast, int A> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (A == DDPM_ACT_RELU) {
    return z > 0.f ? 1.f : 0.f;
  } else if constexpr (A == DDPM_ACT_SILU) {
    const float s = div_f<kFast>(1.f, 1.f + exp_f<kFast>(-z));
    return s * (1.f + z * (1.f - s));
  } else if constexpr (A == DDPM_ACT_GELU) {
    return 0.5f * erfcf(-0.70710678118654752f * z) +
           z * 0.39894228040143268f * exp_f<kFast>(-0.5f * z * z);
  } else if constexpr (A == DDPM_ACT_GELU_TANH) {
    const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
    const float s = div_f<kFast>(1.f, 1.f + exp_f<kFast>(-2.f * u));
    const float du = 0.79788456080286536f * (1.f + 0.134145f * z * z);
    return s + 2.f * z * s * (1.f - s) * du;
  } else {
    return 1.f;
  }
}

// v[i] = act(v[i]) and s[i] = act'(v[i]) for n values, the choice made once.
template <bool kFast, int n> __device__ __forceinline__ void act_values(int act, float (&v)[n]) {
#define DDPM_ACT_CASE(A)                                        \
  case A:                                                       \
    _Pragma("unroll") for (int i = 0; i < n; ++i) v[i] = act_value<kFast, A>(v[i]); \
    break;
  switch (act) {
    DDPM_ACT_CASE(DDPM_ACT_RELU)
    DDPM_ACT_CASE(DDPM_ACT_SILU)
    DDPM_ACT_CASE(DDPM_ACT_GELU)
    DDPM_ACT_CASE(DDPM_ACT_GELU_TANH)
    default: break;
  }
#undef DDPM_ACT_CASE
}
template <bool kFast, int n> __device__ __forceinline__ void act_slopes(int act, float (&v)[n]) {
#define DDPM_ACT_CASE(A)                                        \
  case A:                                                       \
    _Pragma("unroll") for (int i = 0; i < n; ++i) v[i] = act_slope<kFast, A>(v[i]); \
    break;
  switch (act) {
    DDPM_ACT_CASE(DDPM_ACT_RELU)
    DDPM_ACT_CASE(DDPM_ACT_SILU)
    DDPM_ACT_CASE(DDPM_ACT_GELU)
    DDPM_ACT_CASE(DDPM_ACT_GELU_TANH)
    default:
      _Pragma("unroll") for (int i = 0; i < n; ++i) v[i] = 1.f;
  }
#undef DDPM_ACT_CASE
}

}  // namespace ddpm
