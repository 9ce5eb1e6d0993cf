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
// Activations but ReLU are p times a factor s between 0 and 1, with one exponential and one reciprocal per value
// (an exponential may overflow on the far side: 1 / inf = 0):
//   silu       s = 1 / (1 + 2^(-p log2 e))
//   gelu_tanh  s = 0.5 (1 + tanh z) = 1 / (1 + 2^(-2 z log2 e)),  z = sqrt(2/pi) (p + 0.044715 p^3)
//   gelu       s = Phi(p) = 1 - Phi(-p);  Phi(-q) = e^(-q^2 / 2) u Q(u) for q >= 0, u = 1 / (3.3125 + q): the
//              factor before u Q(u) has the tail's fall, and what is left is smooth in u. Q, of degree 7, is
//              fitted here to the smallest maximal error relative to Phi(-q), 1.3e-7 up to q = 14 (a linear
//              program over 1500 points, coefficients rounded one after the other); 5e-7 in FP32 arithmetic up to
//              q = 2, beyond it what the rounding of q^2 / 2 in the exponent makes, 8e-6 at q = 13.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTanhA = -2.302208198144325f;                // -2 sqrt(2 / pi) log2(e)
constexpr float kTanhB = -2.302208198144325f * 0.044715f;
__host__ __device__ constexpr float gelu_coef(int k) {  // of u^k in Q
  return k == 0   ? 0.3987848460674286f
         : k == 1 ? 1.3320972919464111f
         : k == 2 ? 3.6793785095214844f
         : k == 3 ? 15.142889976501465f
         : k == 4 ? -19.1063175201416f
         : k == 5 ? 262.7478332519531f
         : k == 6 ? -682.2756958007812f
                  : 523.8531494140625f;
}

// Phi of a pair of values, and e^(-p^2 / 2).
__device__ __forceinline__ uint64_t normal_cdf(uint64_t p, uint64_t& density) {
  auto c2 = [](float c) { return f2pack(c, c); };
  float p0, p1, a, b, d, e;
  f2unpack(p, p0, p1);
  f2unpack(mul2(mul2(p, p), c2(-0.5f * kLog2e)), a, b);
  density = f2pack(exp2_approx(a), exp2_approx(b));
  const uint64_t u = f2pack(recip_approx(fabsf(p0) + 3.3125f), recip_approx(fabsf(p1) + 3.3125f));
  uint64_t x = c2(gelu_coef(7));
#pragma unroll
  for (int k = 6; k >= 0; --k) x = fma2(x, u, c2(gelu_coef(k)));
  x = mul2(mul2(x, u), density);
  f2unpack(x, a, b);
  f2unpack(fma2(x, c2(-1.f), c2(1.f)), d, e);
  return f2pack(p0 < 0.f ? a : d, p1 < 0.f ? b : e);
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
    return mul2(p, normal_cdf(p, x));
  } else if constexpr (ACT == J1_ACT_GELU_TANH) {
    x = mul2(p, fma2(mul2(p, p), c2(kTanhB), c2(kTanhA)));
  } else {
    x = mul2(p, c2(-kLog2e));
  }
  f2unpack(x, a, b);
  f2unpack(add2(f2pack(exp2_approx(a), exp2_approx(b)), c2(1.f)), a, b);
  return mul2(p, f2pack(recip_approx(a), recip_approx(b)));
}

// act'(p) and act(p) of a pair. gelu: s + p phi(p). The others, with s the logistic function and x(p) its
// argument: act = p s and act' = s + p s (1 - s) x'(p).
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
  } else if constexpr (ACT == J1_ACT_GELU) {
    uint64_t density;
    const uint64_t s = normal_cdf(p, density);
    value = mul2(p, s);
    slope = fma2(mul2(p, c2(0.3989422804014327f)), density, s);
  } else {
    uint64_t h = p, x;
    if constexpr (ACT == J1_ACT_GELU_TANH) {
      f2unpack(p, a, b);
      h = f2pack(min_nan(max_nan(a, -40.f), 40.f), min_nan(max_nan(b, -40.f), 40.f));
    }
    const uint64_t t = mul2(h, h);
    if constexpr (ACT == J1_ACT_GELU_TANH) {
      x = mul2(h, fma2(t, c2(kTanhB), c2(kTanhA)));
    } else {
      x = mul2(h, c2(-kLog2e));
    }
    f2unpack(x, a, b);
    f2unpack(add2(f2pack(exp2_approx(a), exp2_approx(b)), c2(1.f)), a, b);
    const uint64_t s = f2pack(recip_approx(a), recip_approx(b));
    value = mul2(p, s);
    const uint64_t rest = fma2(s, c2(-1.f), c2(1.f));  // 1 - s
    if constexpr (ACT == J1_ACT_GELU_TANH)
      slope = fma2(mul2(mul2(h, s), rest), fma2(t, c2(3.f * 0.044715f * 1.5957691216057308f), c2(1.5957691216057308f)), s);
    else
      slope = fma2(mul2(h, s), rest, s);
  }
}

}  // namespace j1rt
