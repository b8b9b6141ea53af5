// quantize_rows.cu - rows of floats to int8 with one scale each:
//   scale[i] = max_k |x[r,k]| / 127,  q[i,k] = round_half_even(x[r,k] / scale[i])
// with r = index[i] (the gather of an expert dispatch) or r = i.
//
// One pass over memory: a row's vectors of 8 stay in registers between the
// maximum and the division (rows past kHold vectors a thread are read again,
// from L2).  1 to 16 warps share a row, by its length.  The maximum is taken
// over the bits of |x|, which order as unsigned integers with infinities and
// then NaN on top, so one reduction also tells that a row is not finite.
//
// An IEEE division is some ten instructions, and with one for each element the
// kernel was bound by them (16384 x 8192 bf16: 158 us, 2.5 TB/s).  Instead the
// quotient is a product with the rounded reciprocal, off by at most 3 half
// steps (3 * 2^-24 * 127 = 2.3e-5): where it lies further than that from the
// middle between two integers, both round alike; the few vectors with an
// element nearer than 4e-5 are divided.  Now 89 us, 4.5 TB/s; what is left is
// the latency from index to row to maximum, which 1536 threads an SM hide in
// part.
#include <cuda_runtime.h>

#include "epilogue.cuh"
#include "launch.h"
#include "sm100.cuh"

namespace i8c {

namespace {

constexpr int kHold = 4;          // vectors a thread keeps in registers, as they lie in memory
constexpr int kMaxRowWarps = 16;

struct QuantizeArgs {
  const void *x;
  const int32_t *index;
  int8_t *q;
  float *scale;
  int64_t m, k, rows, ldx, ldq;
  int32_t vec_x, vec_q;
};

// Eight elements as they lie in memory.
template <int DT>
struct Raw8 {
  using T = typename Elem<DT>::type;
  static constexpr int kWords = static_cast<int>(sizeof(T)) / 2;
  uint4 w[kWords];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = make_uint4(0, 0, 0, 0);
  }
  // From column k0 on; zeros past the row.
  __device__ __forceinline__ void load(const T *row, int64_t k0, int64_t k, bool vec) {
    if (vec && k0 + 8 <= k) {
#pragma unroll
      for (int j = 0; j < kWords; ++j) w[j] = __ldg(reinterpret_cast<const uint4 *>(row + k0) + j);
    } else {
      clear();
      // Word by word, with constant indices: the vector stays in registers.
      uint32_t *u = reinterpret_cast<uint32_t *>(w);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k0 + j < k) u[j] = reinterpret_cast<const uint32_t *>(row + k0)[j];
      } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(row + k0);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k0 + j < k) u[j >> 1] |= static_cast<uint32_t>(h[j]) << (16 * (j & 1));
      }
    }
  }
  __device__ __forceinline__ float get(int j) const {
    return Elem<DT>::load(reinterpret_cast<const T *>(w)[j]);
  }
  // Elements j and j + 1 (j even) as an fp32 pair.
  __device__ __forceinline__ uint64_t pair(int j) const {
    if constexpr (DT == INT8CONV_BF16) {
      const uint32_t u = reinterpret_cast<const uint32_t *>(w)[j >> 1];
      return f2_pack(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    } else {
      return f2_pack(get(j), get(j + 1));
    }
  }
  // The larger of `top` and the bits of every |x|; 16-bit types two at a time,
  // each half on its own.
  __device__ __forceinline__ uint32_t max_bits(uint32_t top) const {
    const uint32_t *u = reinterpret_cast<const uint32_t *>(w);
#pragma unroll
    for (int j = 0; j < 4 * kWords; ++j)
      top = sizeof(T) == 4 ? max(top, u[j] & 0x7fffffffu) : __vmaxu2(top, u[j] & 0x7fff7fffu);
    return top;
  }
  // The bits of max_bits() as those of one fp32 value (infinite and NaN stay so).
  static __device__ __forceinline__ uint32_t to_fp32_bits(uint32_t top) {
    if constexpr (sizeof(T) == 4) return top;
    const uint16_t h = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    return __float_as_uint(Elem<DT>::load(*reinterpret_cast<const T *>(&h)));
  }
};

// CTAs that an SM should hold at one time: rows on their way hide the latency of
// index, row and reduction.  fp32 rows take twice the registers.
template <int DT, int WARPS>
constexpr int block_count() {
  return (DT == INT8CONV_FP32 ? 1024 : 1536) / (WARPS < 4 ? 128 : 32 * WARPS);
}

template <int DT, int WARPS>
__global__ void __launch_bounds__(WARPS < 4 ? 128 : 32 * WARPS, block_count<DT, WARPS>())
    quantize_kernel(const QuantizeArgs a) {
  using T = typename Elem<DT>::type;
  constexpr int kThreads = WARPS < 4 ? 128 : 32 * WARPS;
  constexpr int kRowThreads = 32 * WARPS;
  constexpr int kRows = kThreads / kRowThreads;
  __shared__ uint32_t maxima[kThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const int t = threadIdx.x % kRowThreads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kRowThreads;
  int64_t r = -1;
  if (i < a.m) r = a.index != nullptr ? __ldg(a.index + i) : i;
  const bool valid = r >= 0 && r < a.rows;
  const T *row = static_cast<const T *>(a.x) + (valid ? r : 0) * a.ldx;
  const bool vec = a.vec_x != 0;
  Raw8<DT> held[kHold];
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < kHold; ++h) {
    const int64_t k0 = static_cast<int64_t>(h * kRowThreads + t) * 8;
    if (valid && k0 < a.k)
      held[h].load(row, k0, a.k, vec);
    else
      held[h].clear();
  }
#pragma unroll
  for (int h = 0; h < kHold; ++h) top = held[h].max_bits(top);
  if (valid) {
    for (int64_t k0 = static_cast<int64_t>(kHold * kRowThreads + t) * 8; k0 < a.k;
         k0 += kRowThreads * 8) {
      Raw8<DT> f;
      f.load(row, k0, a.k, vec);
      top = f.max_bits(top);
    }
  }
  top = Raw8<DT>::to_fp32_bits(top);
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (WARPS > 1) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) maxima[warp] = top;
    __syncthreads();
    const int w0 = warp / WARPS * WARPS;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = maxima[w0 + w] > top ? maxima[w0 + w] : top;
  }
  if (i >= a.m) return;
  const bool finite = top < 0x7f800000u;
  const float scale = __fdiv_rn(__uint_as_float(top), 127.f);
  const bool zero = !valid || !finite || scale == 0.f;
  if (t == 0) a.scale[i] = finite ? scale : __uint_as_float(0x7fffffffu);
  int8_t *q = a.q + i * a.ldq;
  // Scales below 2^-100 (their reciprocals leave fp32's range) are divided by.
  const bool divide = scale < 7.8886090522101181e-31f;
  const float inv = zero ? 0.f : __frcp_rn(scale);
  auto put = [&](int64_t k0, const Raw8<DT> &f) {
    // Adding 1.5 * 2^23 rounds to an integer, half to even, whose low byte is
    // the sum's.
    const uint64_t inv2 = f2_pack(inv, inv);
    const uint64_t magic = f2_pack(12582912.f, 12582912.f);
    const uint64_t minus = f2_pack(-12582912.f, -12582912.f);
    const uint64_t negate = f2_pack(-1.f, -1.f);
    uint32_t w[2];
    float near = 0.f;   // largest distance from an integer
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const uint64_t p = f2_mul(f.pair(4 * h + j), inv2);
        const uint64_t s = f2_add(p, magic);
        float lo, hi;
        f2_unpack(f2_fma(f2_add(s, minus), negate, p), lo, hi);
        near = fmaxf(near, fmaxf(fabsf(lo), fabsf(hi)));
        f2_unpack(s, lo, hi);
        b[j] = __float_as_uint(lo);
        b[j + 1] = __float_as_uint(hi);
      }
      w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    if (zero) {
      w[0] = w[1] = 0;
    } else if (divide || near > 0.49996f) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // |x / scale| passes 127 only where the scale is a denormal.
          v[j] = fminf(fmaxf(__fdiv_rn(f.get(4 * h + j), scale), -127.f), 127.f);
        }
        w[h] = pack_int8(v[0], v[1], v[2], v[3]);
      }
    }
    if (a.vec_q != 0 && k0 + 8 <= a.k) {
      *reinterpret_cast<uint2 *>(q + k0) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < a.k) q[k0 + j] = static_cast<int8_t>(w[j >> 2] >> (8 * (j & 3)));
    }
  };
#pragma unroll
  for (int h = 0; h < kHold; ++h) {
    const int64_t k0 = static_cast<int64_t>(h * kRowThreads + t) * 8;
    if (k0 < a.k) put(k0, held[h]);
  }
  for (int64_t k0 = static_cast<int64_t>(kHold * kRowThreads + t) * 8; k0 < a.k;
       k0 += kRowThreads * 8) {
    Raw8<DT> f;
    if (valid)
      f.load(row, k0, a.k, vec);
    else
      f.clear();
    put(k0, f);
  }
}

template <int DT>
const void *quantize_kernel_for(int warps) {
  switch (warps) {
    case 1:
      return reinterpret_cast<const void *>(&quantize_kernel<DT, 1>);
    case 2:
      return reinterpret_cast<const void *>(&quantize_kernel<DT, 2>);
    case 4:
      return reinterpret_cast<const void *>(&quantize_kernel<DT, 4>);
    case 8:
      return reinterpret_cast<const void *>(&quantize_kernel<DT, 8>);
    default:
      return reinterpret_cast<const void *>(&quantize_kernel<DT, kMaxRowWarps>);
  }
}

}  // namespace

int8conv_status launch_quantize_rows_impl(int64_t m, int64_t k, int x_dtype, const void *x,
                                          int64_t rows, int64_t ldx, const int32_t *index,
                                          int8_t *q, int64_t ldq, float *scale,
                                          cudaStream_t stream) {
  QuantizeArgs a{};
  a.x = x;
  a.index = index;
  a.q = q;
  a.scale = scale;
  a.m = m;
  a.k = k;
  a.rows = rows;
  a.ldx = ldx;
  a.ldq = ldq;
  a.vec_x = (ldx * dtype_bytes(x_dtype)) % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  a.vec_q = ldq % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  // The fewest warps that keep the whole row in registers.
  int warps = 1;
  while (warps < kMaxRowWarps && static_cast<int64_t>(warps) * 32 * kHold * 8 < k) warps *= 2;
  const int threads = warps < 4 ? 128 : 32 * warps;
  const int per_block = threads / (32 * warps);
  LaunchPlan plan;
  plan.func = x_dtype == INT8CONV_BF16   ? quantize_kernel_for<INT8CONV_BF16>(warps)
              : x_dtype == INT8CONV_FP16 ? quantize_kernel_for<INT8CONV_FP16>(warps)
                                         : quantize_kernel_for<INT8CONV_FP32>(warps);
  plan.grid = dim3(static_cast<unsigned>((m + per_block - 1) / per_block));
  plan.block = dim3(static_cast<unsigned>(threads));
  plan_args(plan, a);
  return launch_plan(plan, stream);
}

}  // namespace i8c
