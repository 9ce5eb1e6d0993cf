// Activations of the feed-forward operators and their slopes, in FP32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/j1.h"
#include "ptx.cuh"

namespace j1rt {

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
  static __device__ __forceinline__ void store(void* p, long long i, float v) {
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __half2float(static_cast<const __half*>(p)[i]);
  }
  static __device__ __forceinline__ void store(void* p, long long i, float v) {
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
};

// Minimum and maximum that keep a NaN (fminf / fmaxf drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float recip_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + exp(-x)): relative error about 1e-6 on both tails (exp(-x) may overflow: 1 / inf = 0).
__device__ __forceinline__ float sigmoid(float x) {
  return recip_approx(1.f + exp2_approx(-1.4426950408889634f * x));
}
// The normal distribution function Phi(h) and density phi(h) from one exponential:
// erf(x) = 1 - t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) exp(-x^2), t = 1 / (1 + p x), x >= 0,
// absolute error below 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26).
__device__ __forceinline__ void normal(float h, float& cdf, float& pdf) {
  const float x = fabsf(h) * 0.70710678118654752f;
  const float t = recip_approx(fmaf(0.3275911f, x, 1.f));
  const float e = exp2_approx(-1.4426950408889634f * x * x);
  float s = fmaf(t, 1.061405429f, -1.453152027f);
  s = fmaf(t, s, 1.421413741f);
  s = fmaf(t, s, -0.284496736f);
  s = fmaf(t, s, 0.254829592f);
  s = 0.5f * s * t * e;  // Phi(-|h|)
  cdf = h < 0.f ? s : 1.f - s;
  pdf = 0.3989422804014327f * e;
}

constexpr float kTanhScale2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)

// act(p). The negative tails go to 0 also where p itself overflows to -inf; NaN stays NaN.
template <int ACT>
__device__ __forceinline__ float act_value(float p) {
  if constexpr (ACT == J1_ACT_RELU) return p < 0.f ? 0.f : p;
  if constexpr (ACT == J1_ACT_GELU) {
    float cdf, pdf;
    const float h = max_nan(p, -40.f);
    normal(h, cdf, pdf);
    return h * cdf;
  }
  if constexpr (ACT == J1_ACT_GELU_TANH) {  // 0.5 (1 + tanh z) = sigmoid(2 z)
    const float h = max_nan(p, -40.f);
    return h * sigmoid(kTanhScale2 * fmaf(0.044715f * h * h, h, h));
  }
  if constexpr (ACT == J1_ACT_SILU) {
    const float h = max_nan(p, -200.f);
    return h * sigmoid(h);
  }
  return p;
}

// act of two values. GELU: erf(x) = x P(x^2) / Q(x^2) for |x| <= 4 with P of degree 6 and Q of
// degree 4 in x^2 (the Eigen / XLA single-precision rational, within 1.2e-7 of erf), evaluated
// on pairs with packed FP32 arithmetic: no exponential, a reciprocal per value, and half the
// instructions. x = p / sqrt(2) is folded into the coefficients. Below the clamp the product
// uses the clamped p, so a far negative p gives 0 (to 4e-7) and not p times an error.
template <int ACT>
__device__ __forceinline__ void act_pair(float& a, float& b) {
  if constexpr (ACT == J1_ACT_GELU) {
    constexpr float kClamp = 5.656854f;  // 4 sqrt(2)
    const float la = max_nan(a, -kClamp), lb = max_nan(b, -kClamp);
    const uint64_t x = f2pack(fminf(la, kClamp), fminf(lb, kClamp));
    const uint64_t t = mul2(x, x);
    auto c2 = [](float c) { return f2pack(c, c); };
    uint64_t p = c2(-3.01199018e-12f);
    p = fma2(p, t, c2(6.1223987e-10f));
    p = fma2(p, t, c2(-9.28530142e-08f));
    p = fma2(p, t, c2(-5.03151205e-06f));
    p = fma2(p, t, c2(-0.00012992922f));
    p = fma2(p, t, c2(-0.00104460877f));
    p = fma2(p, t, c2(-0.011381614f));
    uint64_t q = c2(-9.10379526e-07f);
    q = fma2(q, t, c2(-2.6671758e-05f));
    q = fma2(q, t, c2(-0.000420706754f));
    q = fma2(q, t, c2(-0.00368666439f));
    q = fma2(q, t, c2(-0.01426474f));
    float q0, q1;
    f2unpack(q, q0, q1);
    const uint64_t erf = mul2(mul2(x, p), f2pack(recip_approx(q0), recip_approx(q1)));
    const uint64_t h = mul2(f2pack(la, lb), c2(0.5f));
    f2unpack(fma2(h, erf, h), a, b);
  } else {
    a = act_value<ACT>(a);
    b = act_value<ACT>(b);
  }
}

// act'(p) and act(p). The slopes are constant to FP32 beyond |p| = 40; clamping there keeps
// 0 * inf out of them.
template <int ACT>
__device__ __forceinline__ void act_slope(float p, float& slope, float& value) {
  const float h = min_nan(max_nan(p, -40.f), 40.f);
  if constexpr (ACT == J1_ACT_RELU) {
    slope = p > 0.f ? 1.f : 0.f;
    value = p < 0.f ? 0.f : p;
  } else if constexpr (ACT == J1_ACT_GELU) {
    float cdf, pdf;
    normal(h, cdf, pdf);
    slope = fmaf(h, pdf, cdf);
    value = max_nan(p, -40.f) * cdf;
  } else if constexpr (ACT == J1_ACT_GELU_TANH) {
    const float h2 = h * h;
    const float s = sigmoid(kTanhScale2 * fmaf(0.044715f * h2, h, h));
    slope = fmaf(h * (s * (1.f - s)), kTanhScale2 * fmaf(3.f * 0.044715f, h2, 1.f), s);
    value = max_nan(p, -40.f) * s;
  } else if constexpr (ACT == J1_ACT_SILU) {
    const float s = sigmoid(h);
    slope = fmaf(h * s, 1.f - s, s);
    value = max_nan(p, -40.f) * s;
  } else {
    slope = 1.f;
    value = p;
  }
}

}  // namespace j1rt
