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

// p = 1 / (1 + e^-z) and q = 1 - p without cancellation, from e^-|z| in (0, 1].
__device__ __forceinline__ void logistic(float z, float& p, float& q) {
  const float t = __expf(-fabsf(z)), r = reciprocal(1.f + t), tr = t * r;
  p = z < 0.f ? tr : r;
  q = z < 0.f ? r : tr;
}

// sqrt(8 / pi) (z + 0.044715 z^3): gelu_tanh is z p(that).
__device__ __forceinline__ float gelu_inner(float z) {
  return z * fmaf(0.0713548163f, z * z, 1.59576912f);
}

// act(z). What is not a number stays one.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == FELIX_ACT_RELU) {
    return z < 0.f ? 0.f : z;
  } else if constexpr (ACT == FELIX_ACT_GELU) {
    return 0.5f * z * erfcf(-0.707106781f * z);
  } else if constexpr (ACT == FELIX_ACT_GELU_TANH) {
    float p, q;
    logistic(gelu_inner(z), p, q);
    return z * p;
  } else if constexpr (ACT == FELIX_ACT_SILU) {
    float p, q;
    logistic(z, p, q);
    return z * p;
  } else if constexpr (ACT == FELIX_ACT_SIGMOID) {
    float p, q;
    logistic(z, p, q);
    return p;
  } else {
    return z;
  }
}

// act(z) and act'(z). The derivative of relu is 0 at 0.
template <int ACT>
__device__ __forceinline__ void activate_both(float z, float& a, float& d) {
  if constexpr (ACT == FELIX_ACT_RELU) {
    a = z < 0.f ? 0.f : z;
    d = z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  } else if constexpr (ACT == FELIX_ACT_GELU) {
    const float area = 0.5f * erfcf(-0.707106781f * z);
    a = z * area;
    d = fmaf(z * 0.398942280f, __expf(-0.5f * z * z), area);
  } else if constexpr (ACT == FELIX_ACT_GELU_TANH) {
    float p, q;
    logistic(gelu_inner(z), p, q);
    a = z * p;
    d = fmaf(a * q, fmaf(0.214064449f, z * z, 1.59576912f), p);
  } else if constexpr (ACT == FELIX_ACT_SILU) {
    float p, q;
    logistic(z, p, q);
    a = z * p;
    d = fmaf(a, q, p);
  } else if constexpr (ACT == FELIX_ACT_SIGMOID) {
    float q;
    logistic(z, a, q);
    d = a * q;
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
