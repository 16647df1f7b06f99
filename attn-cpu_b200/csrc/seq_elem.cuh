// seq_elem.cuh -- element types of packed rows and pages: reading and writing
// single values and 4-element groups as floats.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kernels.h"

namespace attnb {

template <int T>
struct Elem;
template <>
struct Elem<kF32> {
  using type = float;
};
template <>
struct Elem<kBF16> {
  using type = __nv_bfloat16;
};
template <>
struct Elem<kF16> {
  using type = __half;
};
template <>
struct Elem<kE4M3> {
  using type = __nv_fp8_e4m3;
};
template <>
struct Elem<kI8> {
  using type = int8_t;
};
template <int T>
using elem_t = typename Elem<T>::type;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_fp8_e4m3 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_float(int8_t x) { return static_cast<float>(x); }

// One rounding to nearest even.
__device__ __forceinline__ void from_float(float x, float& y) { y = x; }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float x, __half& y) { y = __float2half_rn(x); }

// Four values from an address aligned to four elements.
template <class E>
__device__ __forceinline__ void load4(const E* p, float (&x)[4]) {
  struct alignas(4 * sizeof(E)) Four {
    E e[4];
  };
  Four f;
  if constexpr (sizeof(E) == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    f = *reinterpret_cast<const Four*>(&v);
  } else if constexpr (sizeof(E) == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    f = *reinterpret_cast<const Four*>(&v);
  } else {
    const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(p));
    f = *reinterpret_cast<const Four*>(&v);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_float(f.e[i]);
}

// Calls f with the type as a compile-time constant.
template <class F>
inline bool with_value_type(int type, F&& f) {
  switch (type) {
    case kF32: f(std::integral_constant<int, kF32>{}); return true;
    case kBF16: f(std::integral_constant<int, kBF16>{}); return true;
    case kF16: f(std::integral_constant<int, kF16>{}); return true;
    default: return false;
  }
}

}  // namespace attnb
