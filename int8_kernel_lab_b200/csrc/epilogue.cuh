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

// ---- two fp32 operations in one instruction (sm_100) -------------------------
// Each half rounds like the scalar operation.
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The hardware's 2^x and 1/x, two units in the last place, denormals as zeros.
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Activations in fp32, two values at a time: the products and sums as pairs.
//   silu       v / (1 + 2^(-v log2 e))
//   gelu_tanh  (1 + tanh u) / 2 = 1 / (1 + exp(-2u)): v / (1 + 2^(-v (p + q v^2)))
//   gelu       v Phi(v) with Phi from the complementary error function of
//              Abramowitz and Stegun 7.1.26: for z = |v| / sqrt 2, t = 1 / (1 + p z),
//              erfc(z) = t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) exp(-z^2) + e, |e| <= 1.5e-7;
//              Phi = erfc / 2 below zero, 1 - erfc / 2 above.
// Errors stay below 2^-19 |v|: the exponent's argument is rounded at most
// three times (|v| < 10: 14.4 * 3 * 2^-24, times a quotient below one), the
// exponential and the quotient add 2^-22 each.  Large negative v: the power
// overflows to infinity, its reciprocal is 0, the result -0; NaN stays NaN.
template <int ACT>
__device__ __forceinline__ void activate2(float &a, float &b) {
  if constexpr (ACT == INT8CONV_ACT_RELU) {
    a = a < 0.f ? 0.f : a;
    b = b < 0.f ? 0.f : b;
  } else if constexpr (ACT == INT8CONV_ACT_SILU || ACT == INT8CONV_ACT_GELU_TANH) {
    const uint64_t v = f2_pack(a, b);
    uint64_t x;
    if constexpr (ACT == INT8CONV_ACT_SILU) {
      x = f2_mul(v, f2_pack(-1.4426950408889634f, -1.4426950408889634f));
    } else {
      // 2 sqrt(2 / pi) log2 e, and 0.044715 times it
      const uint64_t p = f2_pack(-2.3022081985f, -2.3022081985f);
      const uint64_t q = f2_pack(-0.1029432396f, -0.1029432396f);
      x = f2_mul(v, f2_fma(f2_mul(v, v), q, p));
    }
    float e0, e1;
    f2_unpack(x, e0, e1);
    x = f2_add(f2_pack(exp2_approx(e0), exp2_approx(e1)), f2_pack(1.f, 1.f));
    f2_unpack(x, e0, e1);
    f2_unpack(f2_mul(v, f2_pack(rcp_approx(e0), rcp_approx(e1))), a, b);
  } else if constexpr (ACT == INT8CONV_ACT_GELU) {
    const uint64_t z = f2_mul(f2_pack(fabsf(a), fabsf(b)),
                              f2_pack(0.70710678118654752f, 0.70710678118654752f));
    float e0, e1;
    f2_unpack(f2_fma(z, f2_pack(0.3275911f, 0.3275911f), f2_pack(1.f, 1.f)), e0, e1);
    const uint64_t t = f2_pack(rcp_approx(e0), rcp_approx(e1));
    // The coefficients are halved: half of erfc.
    uint64_t h = f2_pack(0.5307027145f, 0.5307027145f);
    h = f2_fma(h, t, f2_pack(-0.7265760135f, -0.7265760135f));
    h = f2_fma(h, t, f2_pack(0.7107068705f, 0.7107068705f));
    h = f2_fma(h, t, f2_pack(-0.142248368f, -0.142248368f));
    h = f2_fma(h, t, f2_pack(0.127414796f, 0.127414796f));
    f2_unpack(f2_mul(f2_mul(z, z), f2_pack(-1.4426950408889634f, -1.4426950408889634f)), e0, e1);
    h = f2_mul(f2_mul(h, t), f2_pack(exp2_approx(e0), exp2_approx(e1)));
    f2_unpack(h, e0, e1);
    a *= a < 0.f ? e0 : 1.f - e0;
    b *= b < 0.f ? e1 : 1.f - e1;
  }
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  float unused = 0.f;
  activate2<ACT>(v, unused);
  return v;
}

// Round half to even, saturate, NaN -> 0.  Conversions to integers run at an
// eighth of the rate of additions, so the integer comes from adding 1.5 * 2^23:
// it is the low byte of the sum.
__device__ __forceinline__ uint32_t int8_bits(float v) {
  v = v != v ? 0.f : fminf(fmaxf(v, -128.f), 127.f);
  return __float_as_uint(v + 12582912.f);
}
__device__ __forceinline__ int8_t to_int8(float v) { return static_cast<int8_t>(int8_bits(v) & 0xff); }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack_fp16(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack_int8(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(int8_bits(a), int8_bits(b), 0x0040),
                     __byte_perm(int8_bits(c), int8_bits(d), 0x0040), 0x5410);
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
  static __device__ __forceinline__ type store(float v) { return to_int8(v); }
};
template <>
struct Elem<INT8CONV_INT32> {
  using type = int32_t;
  static __device__ __forceinline__ float load(type v) { return static_cast<float>(v); }
};

}  // namespace i8c
