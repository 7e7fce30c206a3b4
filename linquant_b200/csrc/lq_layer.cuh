// Helpers of the operators around the recurrence (convolution, scan, product, norms): vectors of any activation type as
// fp32, the activation functions, and the order-independent row maximum.
#pragma once
#include <type_traits>

#include "lq_common.cuh"

namespace lq {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else return Act<T>::from(x);
}

// VEC consecutive values on a VEC * sizeof(T) boundary (16 bytes at most in one access)
template <typename T, int VEC>
struct alignas(VEC * sizeof(T) > 16 ? 16 : VEC * sizeof(T)) Pack {
  T v[VEC];
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
    if constexpr (VEC == 8 && sizeof(T) == 2) {
      Act<T>::unpack8(*reinterpret_cast<const uint4*>(this), x);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = to_f32(v[i]);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[VEC]) {
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
      uint32_t* w = reinterpret_cast<uint32_t*>(this);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) w[i] = Act<T>::pack2(x[2 * i], x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = from_f32<T>(x[i]);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = from_f32<T>(0.f);
  }
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) { return *reinterpret_cast<const Pack<T, VEC>*>(p); }
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& v) { *reinterpret_cast<Pack<T, VEC>*>(p) = v; }

constexpr float kLog2e = 1.4426950408889634f;
// 2^x, one hardware exponential; results below 2^-126 are zero
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// x / (1 + e^-x); e^-x = inf gives -0
__device__ __forceinline__ float silu(float x) { return x * rcp(1.0f + ex2(-kLog2e * x)); }

// log(1 + e^x) = max(x, 0) + log1p(w), w = e^-|x| in (0, 1]; log1p(w) = 2 atanh(s), s = w / (2 + w) <= 1/3: accurate where the
// result is small, where log(1 + w) would lose w's low bits, and without a branch. atanh(s) / s is a polynomial in s^2 fitted at
// Chebyshev nodes of [0, 1/9] (degree 4: within 8e-9 with these fp32 coefficients).
template <bool EXACT = true>
__device__ __forceinline__ float softplus(float x) {
  const float a = -fabsf(x), e = a * kLog2e;
  float w = ex2(e);
  if constexpr (EXACT) {  // what e lost to rounding, with the part of log2(e) that a float does not hold: w is dt's relative error where x is negative
    const float low = fmaf(a, kLog2e, -e) + a * 1.92596299e-8f;
    w = w > 0.0f ? fmaf(w, low * 0.6931471805599453f, w) : w;
  }
  const float s = w * rcp(2.0f + w), q = s * s;
  float t = 0.14087328631750926f;
  t = fmaf(t, q, 0.13980709417397671f);
  t = fmaf(t, q, 0.20012426861730928f);
  t = fmaf(t, q, 0.33333157967540694f);
  t = fmaf(t, q, 1.0000000039388743f);
  return fmaxf(x, 0.0f) + 2.0f * s * t;  // NaN stays: e and w are NaN
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float clamp_nan(float x, float lo, float hi) {  // NaN stays
  float y;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(max_nan(x, lo)), "f"(hi));
  return y;
}
// Row scale and its inverse. Rows whose largest value is below 1.3e-36 (zeros among them) have codes 0.
__device__ __forceinline__ float row_scale(float amax, float& inv) {
  const float scale = __fdiv_rn(amax, 127.0f);
  inv = scale < 1e-38f ? 0.0f : __fdiv_rn(1.0f, scale);
  return scale;
}
// The code rule for a row whose scale is its own: |x inv| exceeds 127 by roundings at most, so nothing has to be clamped
__device__ __forceinline__ int row_code(float x, float inv) {
  const float y = __fmul_rn(x, inv);
  return __float2int_rz(__fadd_rn(y, copysignf(0.5f, y)));
}

// ---- host side
template <typename F>
static inline int with_dtype(int dtype, const char* what, F&& f) {
  switch (dtype) {
    case LQ_F16: return f(__half());
    case LQ_BF16: return f(__nv_bfloat16());
    case LQ_F32: return f(float());
  }
  return fail(LQ_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
}
static inline int dtype_bytes(int dtype) { return dtype == LQ_F32 ? 4 : 2; }
// Extents leave room in an int for the tile that holds an axis' end and the tiles requested ahead of it
static inline bool fits(int extent) { return extent <= 0x7fffffff - (1 << 13); }
// largest power of two (16 at most) that divides every address and byte pitch it is shown
struct Alignment {
  uintptr_t bits = 16;
  Alignment& at(const void* p) { bits |= reinterpret_cast<uintptr_t>(p); return *this; }
  Alignment& pitch(long long elements, int size) { bits |= (uintptr_t)(elements * size); return *this; }
  int bytes() const { return (int)(bits & (~bits + 1)); }
};

}  // namespace lq
