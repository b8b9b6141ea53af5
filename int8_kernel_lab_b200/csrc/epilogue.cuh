// epilogue.cuh - element types and activations shared by the products
// (matmul.cu) and the group norm (group_norm.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "int8conv.h"

namespace i8c {

inline int dtype_bytes(int dtype) {
  switch (dtype) {
    case INT8CONV_BF16:
    case INT8CONV_FP16:
      return 2;
    case INT8CONV_INT8:
      return 1;
    default:
      return 4;
  }
}

// Activations in fp32.  __expf and __fdividef instead of the full-range forms:
// relative error below 2^-19 where |v| < 10 (the exponent's argument is rounded
// once, 14.4 * 2^-24, the rest adds 2^-21), and beyond that the value itself is
// v, or below 5e-4 in magnitude.  Large negative v: exp overflows to infinity
// and the quotient is 0.
template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == INT8CONV_ACT_RELU) return v < 0.f ? 0.f : v;  // NaN stays NaN
  if constexpr (ACT == INT8CONV_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  if constexpr (ACT == INT8CONV_ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
    const float u2 = v * (1.5957691216057308f + 0.071354816272600249f * v * v);
    return __fdividef(v, 1.f + __expf(-u2));
  }
  if constexpr (ACT == INT8CONV_ACT_SILU) return __fdividef(v, 1.f + __expf(-v));
  return v;
}

// Round half to even, saturate, NaN -> 0 (an integer conversion of NaN is 0).
__device__ __forceinline__ int32_t to_int8(float v) {
  int32_t r;
  asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack_fp16(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack_int8(float a, float b, float c, float d) {
  return (to_int8(a) & 0xff) | ((to_int8(b) & 0xff) << 8) | ((to_int8(c) & 0xff) << 16) |
         ((to_int8(d) & 0xff) << 24);
}

// Types by their int8conv_dtype.
template <int DT>
struct Elem;
template <>
struct Elem<INT8CONV_BF16> {
  using type = __nv_bfloat16;
  static __device__ __forceinline__ float load(type v) { return __bfloat162float(v); }
  static __device__ __forceinline__ type store(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<INT8CONV_FP16> {
  using type = __half;
  static __device__ __forceinline__ float load(type v) { return __half2float(v); }
  static __device__ __forceinline__ type store(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<INT8CONV_FP32> {
  using type = float;
  static __device__ __forceinline__ float load(type v) { return v; }
  static __device__ __forceinline__ type store(float v) { return v; }
};
template <>
struct Elem<INT8CONV_INT8> {
  using type = int8_t;
  static __device__ __forceinline__ type store(float v) { return static_cast<int8_t>(to_int8(v)); }
};
template <>
struct Elem<INT8CONV_INT32> {
  using type = int32_t;
  static __device__ __forceinline__ float load(type v) { return static_cast<float>(v); }
};

}  // namespace i8c
