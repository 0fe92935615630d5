// Arithmetic on two neighbouring channels at a time: packed fp32 instructions, and
// functions by the inputs' type.
#pragma once

#include "common.cuh"

namespace la {

__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 load_two(const __nv_bfloat16 *p) {
  const uint32_t w = *(const uint32_t *)p;
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 load_two(const float *p) { return *(const float2 *)p; }

// Whether any of some bf16 values are below a negative bound: as unsigned numbers floats
// below zero are the larger the lower they are, above all others.
struct Least {
  uint32_t v = 0;
  __device__ __forceinline__ void take(const __nv_bfloat16 *p, const __nv_bfloat16 *q) {
    v = __vimax3_u16x2(v, *(const uint32_t *)p, *(const uint32_t *)q);
  }
  __device__ __forceinline__ bool below(float bound) const {
    return max(v & 0xFFFF, v >> 16) > __float_as_uint(bound) >> 16;
  }
};

// Channels c and c + 1 of a row of n (the second may be beyond it); `pair`: the
// row's pairs are aligned.
__device__ __forceinline__ void store_two(__nv_bfloat16 *p, float2 v, bool pair, bool second) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
  if (pair) {
    *(__nv_bfloat162 *)p = b;
  } else {
    p[0] = b.x;
    if (second) p[1] = b.y;
  }
}
__device__ __forceinline__ void store_two(float *p, float2 v, bool pair, bool second) {
  if (pair) {
    *(float2 *)p = v;
  } else {
    p[0] = v.x;
    if (second) p[1] = v.y;
  }
}

// Functions by the inputs' type.  The special-function unit's reciprocal is within
// an ulp, its roots and exponentials within 2^-22: for bf16 inputs, which are 2^-9
// apart, that is far below what they carry.  fp32 ones take the library's
// exponential, which is as near for large arguments too.
template <typename T> struct Fn;
template <> struct Fn<__nv_bfloat16> {
  static __device__ __forceinline__ float exp(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
  }
  static __device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
  static __device__ __forceinline__ float rsqrt(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
};
template <> struct Fn<float> {
  static __device__ __forceinline__ float exp(float x) { return expf(x); }
  static __device__ __forceinline__ float rcp(float x) { return Fn<__nv_bfloat16>::rcp(x); }
  static __device__ __forceinline__ float rsqrt(float x) { return rsqrtf(x); }
};

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 min_nan(float2 a, float b) {
  return make_float2(min_nan(a.x, b), min_nan(a.y, b));
}
template <typename T> __device__ __forceinline__ float2 rcp_two(float2 x) {
  return make_float2(Fn<T>::rcp(x.x), Fn<T>::rcp(x.y));
}
template <typename T> __device__ __forceinline__ float2 rsqrt_two(float2 x) {
  return make_float2(Fn<T>::rsqrt(x.x), Fn<T>::rsqrt(x.y));
}
// exp(-x)
template <typename T> __device__ __forceinline__ float2 exp_minus(float2 x) {
  if constexpr (sizeof(T) == 2) {
    const float2 t = __fmul2_rn(x, two(-1.4426950408889634f));
    float2 y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(t.y));
    return y;
  } else {
    return make_float2(expf(-x.x), expf(-x.y));
  }
}

// 1 / (1 + exp(-z)); an infinite exponential gives 0.
template <typename T> __device__ __forceinline__ float2 sigmoid_two(float2 z) {
  return rcp_two<T>(__fadd2_rn(exp_minus<T>(z), two(1.f)));
}

}  // namespace la
