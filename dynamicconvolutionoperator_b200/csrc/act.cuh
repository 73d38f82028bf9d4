// Activations of the channel-last operators and their derivatives, FP32.
//   relu       max(z, 0)
//   silu       z / (1 + e^-z)
//   gelu       z * Phi(z), Phi the normal distribution function (erf form)
//   gelu_tanh  z/2 * (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3)))
// kFast (16-bit data) takes the hardware's approximate exponential and
// reciprocal and a fitted Phi, with errors far below the rounding to 16 bits.
// FP32 data takes the full-precision functions.
#pragma once

#include "common.cuh"

namespace ddpm {

// Two floats rounded to the 16-bit type and packed, `a` in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// 16 bytes as floats, and back.
template <typename T> __device__ __forceinline__ void unpack16(uint4 u, float* v) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
  } else {
    const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y), c = unpack2<T>(u.z), d = unpack2<T>(u.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
}
template <typename T> __device__ __forceinline__ uint4 pack16(const float* v) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
  else
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                      pack2<T>(v[6], v[7]));
}

__host__ inline bool act_known(int act) { return act >= DDPM_ACT_NONE && act <= DDPM_ACT_GELU_TANH; }

// 1 / (1 + 2^t) by the hardware's exponential and reciprocal (2^-22 each); an
// overflow of 2^t gives 0.
__device__ __forceinline__ float logistic2(float t) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;

// Phi(z) = 1 / (1 + e^-s(z)) with s(z) = log(Phi(z) / Phi(-z)) = z p(z^2). p is a
// polynomial of degree 7 over z^2 <= 25 (constant beyond), fitted here for the
// least maximum of Phi's relative error below zero, 1.6e-5; |z Phi(z)| is off
// by at most 2.8e-6. A 16-bit value's half step is 2.4e-4 or more of it. The
// coefficients hold the factor -log2(e).
__device__ __forceinline__ float normal_cdf(float z) {
  const float u = fminf(z * z, 25.f);
  float q = fmaf(u, 7.628720572e-11f, -8.903303872e-09f);
  q = fmaf(u, q, 4.363843402e-07f);
  q = fmaf(u, q, -1.140831500e-05f);
  q = fmaf(u, q, 1.531346206e-04f);
  q = fmaf(u, q, 1.431668934e-04f);
  q = fmaf(u, q, -1.049632579e-01f);
  q = fmaf(u, q, -2.302116394e+00f);
  return logistic2(z * q);
}

// Factors of the forms that are z / (1 + e^-s(z)).
template <bool kFast, int A> __device__ __forceinline__ float act_gate(float z) {
  if constexpr (A == DDPM_ACT_SILU) {
    if constexpr (kFast) return logistic2(-kLog2e * z);
    else return 1.f / (1.f + expf(-z));
  } else if constexpr (A == DDPM_ACT_GELU) {
    if constexpr (kFast) return normal_cdf(z);
    // erfc keeps the relative precision of the tail below zero
    else return 0.5f * erfcf(-0.70710678118654752f * z);
  } else {  // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
    const float u2 = z * fmaf(0.07135481627f, z * z, 1.59576912161f);
    if constexpr (kFast) return logistic2(-kLog2e * u2);
    else return 1.f / (1.f + expf(-u2));
  }
}

template <bool kFast, int A> __device__ __forceinline__ float act_value(float z) {
  if constexpr (A == DDPM_ACT_NONE) return z;
  else if constexpr (A == DDPM_ACT_RELU) return z < 0.f ? 0.f : z;  // keeps a NaN
  else return z * act_gate<kFast, A>(z);
}

template <bool kFast, int A> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (A == DDPM_ACT_NONE) {
    return 1.f;
  } else if constexpr (A == DDPM_ACT_RELU) {
    return z > 0.f ? 1.f : 0.f;
  } else {
    const float g = act_gate<kFast, A>(z);
    if constexpr (A == DDPM_ACT_SILU) {
      return g * fmaf(z, 1.f - g, 1.f);
    } else if constexpr (A == DDPM_ACT_GELU) {
      const float x = -0.5f * z * z;
      return fmaf(z * 0.39894228040143268f, kFast ? __expf(x) : expf(x), g);
    } else {
      const float du2 = fmaf(0.21406444881f, z * z, 1.59576912161f);
      return fmaf(z * g, (1.f - g) * du2, g);
    }
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
