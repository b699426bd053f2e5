// Activations of the feed-forward operators and their derivatives, in fp32, and the
// two 16-bit element types that the operators take.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/felix_c.h"

namespace felix_ffn {

// 1 / d. The approximate reciprocal is within 1 ulp and, other than __fdividef, holds
// for every d: a large one gives a subnormal, infinity gives zero.
__device__ __forceinline__ float reciprocal(float d) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

// 2^x, to 2 ulp.
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 1 / (1 + e^-z). The exponent's rounding becomes an error of e^-z that grows with z: the
// result is within (7 + 1.25 max(-z, 0.4)) 2^-24 relative (half a step of the 16-bit values
// made of it is 2^-11 or 2^-8). Past z = -88.7 e^-z is infinite, which gives 0.
__device__ __forceinline__ float logistic(float z) {
  return reciprocal(1.f + exp2_approx(-1.44269504f * z));
}

// sqrt(8 / pi) (z + 0.044715 z^3): gelu_tanh is z logistic(that).
__device__ __forceinline__ float gelu_inner(float z) {
  return z * fmaf(0.0713548163f, z * z, 1.59576912f);
}

// The normal distribution function, and e^(-z^2 / 2). With s = |z| / sqrt 2 and
// t = 1 / (1 + s / 2) (the variable of the fit of erfc in Press et al., Numerical Recipes, 6.2),
// erfc(s) e^(s^2) / (2 t) is smooth in t on (0, 1]; the polynomial is its minimax fit of
// degree 6 for s up to 10 (where e^(-s^2) is 0), to 1.5e-6 relative, so that small values for
// negative z keep their leading bits too: the whole is within 2e-6 for z > -5 and, as the
// exponent's rounding grows with z^2, 7e-6 near -13, far below half a step of 16 bits.
__device__ __forceinline__ float normal_area(float z, float& e) {
  e = exp2_approx(-0.721347520f * z * z);
  const float t = reciprocal(fmaf(0.353553391f, fabsf(z), 1.f));
  float c = fmaf(0.04410203546f, t, -0.17836862803f);
  c = fmaf(c, t, 0.19461159408f);
  c = fmaf(c, t, 0.01894582063f);
  c = fmaf(c, t, 0.14075168967f);
  c = fmaf(c, t, 0.13879109917f);
  c = fmaf(c, t, 0.14116570354f);
  const float tail = c * t * e;
  return z < 0.f ? tail : 1.f - tail;
}

// act(z). What is not a number stays one.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == FELIX_ACT_RELU) {
    return z < 0.f ? 0.f : z;
  } else if constexpr (ACT == FELIX_ACT_GELU) {
    float e;
    return z * normal_area(z, e);
  } else if constexpr (ACT == FELIX_ACT_GELU_TANH) {
    return z * logistic(gelu_inner(z));
  } else if constexpr (ACT == FELIX_ACT_SILU) {
    return z * logistic(z);
  } else if constexpr (ACT == FELIX_ACT_SIGMOID) {
    return logistic(z);
  } else {
    return z;
  }
}

// act(z) and act'(z). The derivative of relu is 0 at 0. 1 - p stands for the logistic of
// -z where it is added to something that is larger; sigmoid's derivative is a product of
// both and takes them without cancellation.
template <int ACT>
__device__ __forceinline__ void activate_both(float z, float& a, float& d) {
  if constexpr (ACT == FELIX_ACT_RELU) {
    a = z < 0.f ? 0.f : z;
    d = z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  } else if constexpr (ACT == FELIX_ACT_GELU) {
    float e;
    const float area = normal_area(z, e);
    a = z * area;
    d = fmaf(z * 0.398942280f, e, area);
  } else if constexpr (ACT == FELIX_ACT_GELU_TANH) {
    const float p = logistic(gelu_inner(z));
    a = z * p;
    // (z^2 bounded: where 1 - p is 0 the product is)
    d = fmaf(a * (1.f - p), fmaf(0.214064449f, fminf(z * z, 1e6f), 1.59576912f), p);
  } else if constexpr (ACT == FELIX_ACT_SILU) {
    const float p = logistic(z);
    a = z * p;
    d = fmaf(a, 1.f - p, p);
  } else if constexpr (ACT == FELIX_ACT_SIGMOID) {
    const float t = exp2_approx(-1.44269504f * fabsf(z)), r = reciprocal(1.f + t);
    a = z < 0.f ? t * r : r;
    d = t * r * r;
  } else {
    a = z;
    d = 1.f;
  }
}

// Calls f with the activation as a compile-time constant (f.template operator()<ACT>()).
template <class F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case FELIX_ACT_RELU: return f.template operator()<FELIX_ACT_RELU>();
    case FELIX_ACT_GELU: return f.template operator()<FELIX_ACT_GELU>();
    case FELIX_ACT_GELU_TANH: return f.template operator()<FELIX_ACT_GELU_TANH>();
    case FELIX_ACT_SILU: return f.template operator()<FELIX_ACT_SILU>();
    case FELIX_ACT_SIGMOID: return f.template operator()<FELIX_ACT_SIGMOID>();
    default: return f.template operator()<FELIX_ACT_NONE>();
  }
}

// ------------------------------------------------------------------ 16-bit types
template <class T>
struct Pair;
template <>
struct Pair<__half> {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ float to_float(uint16_t v) {
    return __half2float(__ushort_as_half(v));
  }
  static __device__ __forceinline__ uint16_t of_float(float v) {
    return __half_as_ushort(__float2half_rn(v));
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return {__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)};
  }
  static __device__ __forceinline__ float to_float(uint16_t v) {
    return __uint_as_float(uint32_t(v) << 16);
  }
  static __device__ __forceinline__ uint16_t of_float(float v) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
};

}  // namespace felix_ffn
