// Activations of the channel-last operators and their derivatives, FP32.
//   relu       max(z, 0)
//   silu       z / (1 + e^-z)
//   gelu       z * Phi(z), Phi the normal distribution function (erf form)
//   gelu_tanh  z/2 * (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3)))
// kFast (16-bit data) takes the hardware's approximate exponential and
// reciprocal and a fitted Phi, with errors far below the rounding to 16 bits (of
// gelu: 1.7e-5 of the value, over the whole range). FP32 data takes the
// full-precision functions.
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

// Two FP32 values in a register pair: one instruction does both.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__host__ inline bool act_known(int act) { return act >= DDPM_ACT_NONE && act <= DDPM_ACT_GELU_TANH; }

// 1 / (1 + 2^t) by the hardware's exponential and reciprocal (2^-22 each); an
// overflow of 2^t gives 0.
__device__ __forceinline__ float exp2_fast(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float rcp_fast(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}
__device__ __forceinline__ F2 logistic2(F2 t) {
  const float2 u = split(t);
  const float2 d = split(f2(exp2_fast(u.x), exp2_fast(u.y)) + f2(1.f));
  return f2(rcp_fast(d.x), rcp_fast(d.y));
}

constexpr float kLog2e = 1.4426950408889634f;

// -Phi(-|z|), and e = e^(-z^2 / 2). Phi(-t) = e G(t), where G falls slowly (as
// 1 / t far out): a polynomial of degree 5 in 1 / (1 + 0.36 t), fitted here for the
// least maximum of its relative error over 0 <= t <= 13.3, 1.1e-5; with the FP32
// roundings 1.7e-5. So Phi keeps its digits down to -13.2, where bf16 has its least
// values of z Phi(z) (a fit of log(Phi(z) / Phi(-z)) over z^2 <= 25 was 13 times off at
// -6); beyond, the exponential gives 0. The coefficients hold the factor -1.
__device__ __forceinline__ F2 normal_tail(F2 z, F2& e) {
  const float2 x = split(z * z * f2(-0.5f * kLog2e)), u = split(z);
  e = f2(exp2_fast(x.x), exp2_fast(x.y));
  const float2 d = split(fma2(f2(fabsf(u.x), fabsf(u.y)), f2(0.36f), f2(1.f)));
  const F2 k = f2(rcp_fast(d.x), rcp_fast(d.y));
  F2 g = fma2(k, f2(9.919366325e-02f), f2(-2.561782224e-01f));
  g = fma2(k, g, f2(-3.334195208e-02f));
  g = fma2(k, g, f2(-1.695141690e-01f));
  g = fma2(k, g, f2(-1.399494276e-01f));
  g = fma2(k, g, f2(-2.050534351e-04f));
  return e * g;
}

// Factors of the forms that are z / (1 + e^-s(z)): Phi and its like. (16-bit gelu
// goes by normal_tail.)
template <int A> __device__ __forceinline__ float act_gate(float z) {  // FP32 data
  if constexpr (A == DDPM_ACT_SILU) return 1.f / (1.f + expf(-z));
  // erfc keeps the relative precision of the tail below zero
  else if constexpr (A == DDPM_ACT_GELU) return 0.5f * erfcf(-0.70710678118654752f * z);
  // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
  else return 1.f / (1.f + expf(-z * fmaf(0.07135481627f, z * z, 1.59576912161f)));
}
template <int A> __device__ __forceinline__ F2 act_gate(F2 z) {  // 16-bit data
  if constexpr (A == DDPM_ACT_SILU) return logistic2(z * f2(-kLog2e));
  else return logistic2(z * fma2(z * z, f2(-kLog2e * 0.07135481627f), f2(-kLog2e * 1.59576912161f)));
}

template <bool kFast, int A> __device__ __forceinline__ F2 act_value(F2 z) {
  if constexpr (A == DDPM_ACT_NONE) {
    return z;
  } else {
    const float2 u = split(z);
    if constexpr (A == DDPM_ACT_RELU)
      return f2(u.x < 0.f ? 0.f : u.x, u.y < 0.f ? 0.f : u.y);  // keeps a NaN
    else if constexpr (kFast && A == DDPM_ACT_GELU) {
      // max(z, 0) - |z| Phi(-|z|); 14 in place of |z| keeps infinity times 0 out above
      F2 e;
      const F2 tail = normal_tail(z, e);
      return fma2(f2(fmaxf(-u.x, fminf(u.x, 14.f)), fmaxf(-u.y, fminf(u.y, 14.f))), tail,
                  f2(fmaxf(u.x, 0.f), fmaxf(u.y, 0.f)));
    } else if constexpr (kFast)
      return z * act_gate<A>(z);
    else
      return z * f2(act_gate<A>(u.x), act_gate<A>(u.y));
  }
}

template <bool kFast, int A> __device__ __forceinline__ F2 act_slope(F2 z) {
  if constexpr (A == DDPM_ACT_NONE) {
    return f2(1.f);
  } else {
    const float2 u = split(z);
    if constexpr (A == DDPM_ACT_RELU) {
      return f2(u.x > 0.f ? 1.f : 0.f, u.y > 0.f ? 1.f : 0.f);
    } else {
      if constexpr (kFast && A == DDPM_ACT_GELU) {
        F2 e;
        const float2 tail = split(normal_tail(z, e));
        const F2 g = f2(u.x < 0.f ? -tail.x : 1.f + tail.x, u.y < 0.f ? -tail.y : 1.f + tail.y);
        return fma2(z * f2(0.39894228040143268f), e, g);
      } else {
        F2 g;
        if constexpr (kFast) g = act_gate<A>(z);
        else g = f2(act_gate<A>(u.x), act_gate<A>(u.y));
        const F2 rest = fma2(g, f2(-1.f), f2(1.f));
        if constexpr (A == DDPM_ACT_SILU) {
          return g * fma2(z, rest, f2(1.f));
        } else if constexpr (A == DDPM_ACT_GELU) {
          const F2 e = f2(expf(-0.5f * u.x * u.x), expf(-0.5f * u.y * u.y));
          return fma2(z * f2(0.39894228040143268f), e, g);
        } else {
          // beyond |z| = 100 one of g and 1 - g is 0: a z^2 past FP32 must not meet it
          const float2 sq = split(z * z);
          const F2 du = fma2(f2(fminf(sq.x, 1e4f), fminf(sq.y, 1e4f)), f2(0.21406444881f),
                             f2(1.59576912161f));
          return fma2(z * g, rest * du, g);
        }
      }
    }
  }
}

// v[i] = act(v[i]), and v[i] = act'(v[i]), for n (even) values, the choice made
// once.
template <bool kFast, int n> __device__ __forceinline__ void act_values(int act, float (&v)[n]) {
#define DDPM_ACT_CASE(A)                                        \
  case A:                                                       \
    _Pragma("unroll") for (int i = 0; i < n; i += 2) {                               \
      const float2 r = split(act_value<kFast, A>(f2(v[i], v[i + 1])));                       \
      v[i] = r.x;                                                                            \
      v[i + 1] = r.y;                                                                        \
    }                                                                                        \
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
    _Pragma("unroll") for (int i = 0; i < n; i += 2) {                               \
      const float2 r = split(act_slope<kFast, A>(f2(v[i], v[i + 1])));                       \
      v[i] = r.x;                                                                            \
      v[i + 1] = r.y;                                                                        \
    }                                                                                        \
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
