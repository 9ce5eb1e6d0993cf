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
  // Rounded towards zero (a NaN may become an infinity); the smallest step.
  static __device__ __forceinline__ float cut(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
  static constexpr float kStep = 0x1p-133f;
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
  static __device__ __forceinline__ float cut(float v) { return __half2float(__float2half_rz(v)); }
  static constexpr float kStep = 0x1p-24f;
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
// Every activation here but ReLU is p times a logistic function of an odd polynomial of p, and all
// are evaluated that way, with one exponential and one reciprocal per value (the exponential may
// overflow on the far side: 1 / inf = 0):
//   silu       p / (1 + 2^(-p log2 e))
//   gelu_tanh  0.5 (1 + tanh z) = 1 / (1 + 2^(-2 z log2 e)),  z = sqrt(2/pi) (p + 0.044715 p^3)
//   gelu       Phi(p) = 1 / (1 + 2^(-p R(p^2))): R(p^2) = log2(Phi / (1 - Phi)) / p is smooth and even; a
//              polynomial of degree 6 in p^2, fitted here by reweighted least squares on |p| <= 6 to the
//              smallest maximal error of Phi, is within 3e-8 of Phi (5e-8 in FP32 arithmetic), and its
//              leading coefficient keeps it growing beyond.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTanhA = -2.302208198144325f;                // -2 sqrt(2 / pi) log2(e)
constexpr float kTanhB = -2.302208198144325f * 0.044715f;
__host__ __device__ constexpr float gelu_coef(int k) {  // minus the coefficient of p^(2 k) in R
  return k == 0   ? -2.3022093772888184f
         : k == 1 ? -0.10483512282371521f
         : k == 2 ? 9.404900629306212e-05f
         : k == 3 ? 1.5958001313265413e-04f
         : k == 4 ? -1.1439842637628317e-05f
         : k == 5 ? 3.8163187809914234e-07f
                  : -5.06724973092787e-09f;
}

// act of a pair of values (packed FP32 arithmetic around the exponentials and reciprocals).
template <int ACT>
__device__ __forceinline__ uint64_t act_pair(uint64_t p) {
  if constexpr (ACT == J1_ACT_NONE) return p;
  float a, b;
  if constexpr (ACT == J1_ACT_RELU) {
    f2unpack(p, a, b);
    return f2pack(a < 0.f ? 0.f : a, b < 0.f ? 0.f : b);  // keeps NaN
  }
  auto c2 = [](float c) { return f2pack(c, c); };
  uint64_t x;
  if constexpr (ACT == J1_ACT_GELU) {
    const uint64_t t = mul2(p, p);
    x = c2(gelu_coef(6));
#pragma unroll
    for (int k = 5; k >= 0; --k) x = fma2(x, t, c2(gelu_coef(k)));
    x = mul2(x, p);
  } else if constexpr (ACT == J1_ACT_GELU_TANH) {
    x = mul2(p, fma2(mul2(p, p), c2(kTanhB), c2(kTanhA)));
  } else {
    x = mul2(p, c2(-kLog2e));
  }
  f2unpack(x, a, b);
  f2unpack(add2(f2pack(exp2_approx(a), exp2_approx(b)), c2(1.f)), a, b);
  return mul2(p, f2pack(recip_approx(a), recip_approx(b)));
}

// act'(p) and act(p) of a pair. With s the logistic function and x(p) its argument, act = p s and
// act' = s + p s (1 - s) x'(p); for gelu p s (1 - s) x' is p phi(p), taken from the density itself.
// The tanh form's slope is constant to FP32 beyond |p| = 40; clamping there keeps 0 * inf out of it.
template <int ACT>
__device__ __forceinline__ void act_slope(uint64_t p, uint64_t& slope, uint64_t& value) {
  auto c2 = [](float c) { return f2pack(c, c); };
  float a, b;
  if constexpr (ACT == J1_ACT_NONE) {
    slope = c2(1.f);
    value = p;
  } else if constexpr (ACT == J1_ACT_RELU) {
    f2unpack(p, a, b);
    slope = f2pack(a > 0.f ? 1.f : 0.f, b > 0.f ? 1.f : 0.f);
    value = f2pack(a < 0.f ? 0.f : a, b < 0.f ? 0.f : b);
  } else {
    uint64_t h = p, x;
    if constexpr (ACT == J1_ACT_GELU_TANH) {
      f2unpack(p, a, b);
      h = f2pack(min_nan(max_nan(a, -40.f), 40.f), min_nan(max_nan(b, -40.f), 40.f));
    }
    const uint64_t t = mul2(h, h);
    if constexpr (ACT == J1_ACT_GELU) {
      x = c2(gelu_coef(6));
#pragma unroll
      for (int k = 5; k >= 0; --k) x = fma2(x, t, c2(gelu_coef(k)));
      x = mul2(x, h);
    } else if constexpr (ACT == J1_ACT_GELU_TANH) {
      x = mul2(h, fma2(t, c2(kTanhB), c2(kTanhA)));
    } else {
      x = mul2(h, c2(-kLog2e));
    }
    f2unpack(x, a, b);
    f2unpack(add2(f2pack(exp2_approx(a), exp2_approx(b)), c2(1.f)), a, b);
    const uint64_t s = f2pack(recip_approx(a), recip_approx(b));
    value = mul2(p, s);
    if constexpr (ACT == J1_ACT_GELU) {
      f2unpack(mul2(t, c2(-0.5f * kLog2e)), a, b);
      slope = fma2(mul2(h, c2(0.3989422804014327f)), f2pack(exp2_approx(a), exp2_approx(b)), s);
    } else {
      const uint64_t rest = fma2(s, c2(-1.f), c2(1.f));  // 1 - s
      if constexpr (ACT == J1_ACT_GELU_TANH)
        slope = fma2(mul2(mul2(h, s), rest), fma2(t, c2(3.f * 0.044715f * 1.5957691216057308f), c2(1.5957691216057308f)), s);
      else
        slope = fma2(mul2(h, s), rest, s);
    }
  }
}

}  // namespace j1rt
