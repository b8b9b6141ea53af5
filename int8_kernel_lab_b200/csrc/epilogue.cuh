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

__device__ __forceinline__ uint64_t f2_neg(uint64_t a) {
  float lo, hi;
  f2_unpack(a, lo, hi);
  return f2_pack(-lo, -hi);
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
//   gelu       v Phi(v): with z = |v| / sqrt 2, Phi = erfc(z) / 2 below zero and
//              1 - erfc(z) / 2 above; erfc(z) / 2 = exp(-z^2) t P(t), t = 1 / (1 + 0.33 z).
//              P is the polynomial of degree 7 whose largest relative error over
//              0 <= z <= 9.5 is least (8.2e-8; fitted to exp(z^2) erfc(z) by
//              least squares with Lawson's weights).
// FULL, for fp32 results: silu with the rest of its exponent, gelu for |v| <= 1 as
// v / 2 + v^2 R(v^2), R the polynomial of degree 4 fitted to (Phi(v) - 1/2) / v in
// the same way (2.9e-8 of the result); gelu_tanh is as near as fp32 allows anyway.
//
// Largest errors relative to the result, in u = 2^-24 (each exponential has
// 4 u, each reciprocal 2 u, each product or sum 1 u; an exponent x rounded k
// times adds 0.69 k |x| u to 2^x), measured over 4 million values, beside
// those of torch's fp32 forms:
//                         v >= -0.5   -2..-0.5   -6..-2
//   silu                     4.0         4.0       8.3
//   silu, FULL               3.5         4.0       4.0
//   gelu_tanh                3.6         7.5      54        (exponents to 36, three roundings)
//   gelu                    10.4         9.6      32       (exponents to 26, two roundings)
//   gelu, FULL               2.2         9.6      32
//   silu, torch              3.1         3.1       3.4
//   gelu_tanh, torch         2.9        18        all of it
//   gelu, torch              2.7        20        all of it
// Large negative v: the power overflows to infinity, its reciprocal is 0, the
// result -0; NaN stays NaN.
template <int ACT, bool FULL = false>
__device__ __forceinline__ void activate2(float &a, float &b) {
  if constexpr (ACT == INT8CONV_ACT_RELU) {
    a = a < 0.f ? 0.f : a;
    b = b < 0.f ? 0.f : b;
  } else if constexpr (ACT == INT8CONV_ACT_SILU && FULL) {
    // The power of the rounded exponent x, times 1 - ln 2 (what x lacks): d from
    // the rounding of the product, v * 1.9e-8 from that of log2 e.
    const uint64_t v = f2_pack(fminf(a, 100.f), fminf(b, 100.f));
    const uint64_t x = f2_mul(v, f2_pack(-1.44269502f, -1.44269502f));
    const uint64_t d = f2_fma(v, f2_pack(1.44269502f, 1.44269502f), x);
    const uint64_t t = f2_fma(v, f2_pack(1.92596299e-8f, 1.92596299e-8f), d);
    float e0, e1;
    f2_unpack(x, e0, e1);
    const uint64_t e = f2_pack(fminf(exp2_approx(e0), 3e38f), fminf(exp2_approx(e1), 3e38f));
    const uint64_t s = f2_fma(f2_mul(e, t), f2_pack(-0.69314718f, -0.69314718f), e);
    f2_unpack(f2_add(s, f2_pack(1.f, 1.f)), e0, e1);
    a *= rcp_approx(e0);
    b *= rcp_approx(e1);
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
    // 1 + 0.33 z
    float e0, e1;
    f2_unpack(f2_fma(f2_pack(fabsf(a), fabsf(b)), f2_pack(0.23334524f, 0.23334524f),
                     f2_pack(1.f, 1.f)),
              e0, e1);
    const uint64_t t = f2_pack(rcp_approx(e0), rcp_approx(e1));
    uint64_t h = f2_pack(-0.0679643707f, -0.0679643707f);
    h = f2_fma(h, t, f2_pack(0.231343964f, 0.231343964f));
    h = f2_fma(h, t, f2_pack(-0.177719227f, -0.177719227f));
    h = f2_fma(h, t, f2_pack(0.206270591f, 0.206270591f));
    h = f2_fma(h, t, f2_pack(0.0225054312f, 0.0225054312f));
    h = f2_fma(h, t, f2_pack(0.100961884f, 0.100961884f));
    h = f2_fma(h, t, f2_pack(0.0914186293f, 0.0914186293f));
    h = f2_fma(h, t, f2_pack(0.0931830583f, 0.0931830583f));
    // 2^(-v^2 log2 e / 2)
    const uint64_t v = f2_pack(a, b);
    f2_unpack(f2_mul(f2_mul(v, v), f2_pack(-0.72134752044448170f, -0.72134752044448170f)), e0, e1);
    h = f2_mul(f2_mul(h, t), f2_pack(exp2_approx(e0), exp2_approx(e1)));
    f2_unpack(h, e0, e1);
    if constexpr (FULL) {
      const uint64_t w = f2_mul(v, v);
      uint64_t r = f2_pack(9.15124104e-5f, 9.15124104e-5f);
      r = f2_fma(r, w, f2_pack(-0.00116311492f, -0.00116311492f));
      r = f2_fma(r, w, f2_pack(0.00996239664f, 0.00996239664f));
      r = f2_fma(r, w, f2_pack(-0.0664881962f, -0.0664881962f));
      r = f2_fma(r, w, f2_pack(0.398942153f, 0.398942153f));
      r = f2_fma(r, w, f2_mul(v, f2_pack(0.5f, 0.5f)));
      float n0, n1;
      f2_unpack(r, n0, n1);
      a = fabsf(a) <= 1.f ? n0 : a * (a < 0.f ? e0 : 1.f - e0);
      b = fabsf(b) <= 1.f ? n1 : b * (b < 0.f ? e1 : 1.f - e1);
    } else {
      a *= a < 0.f ? e0 : 1.f - e0;
      b *= b < 0.f ? e1 : 1.f - e1;
    }
  }
}

template <int ACT, bool FULL = false>
__device__ __forceinline__ float activate(float v) {
  float unused = 0.f;
  activate2<ACT, FULL>(v, unused);
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
