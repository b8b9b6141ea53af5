// quantize_rows.cu - rows of floats to int8 with one scale each:
//   scale[i] = max_k |x[r,k]| / 127,  q[i,k] = round_half_even(x[r,k] / scale[i])
// with r = index[i] (the gather of an expert dispatch) or r = i.
//
// One pass over memory: a row's vectors of 8 stay in registers between the
// maximum and the division (rows past kHold vectors a thread are read again,
// from L2).  1 to 16 warps share a row, by its length.  The maximum is taken
// over the bits of |x|, which order as unsigned integers with infinities and
// then NaN on top, so one reduction also tells that a row is not finite.
#include <cuda_runtime.h>

#include "epilogue.cuh"
#include "launch.h"
#include "sm100.cuh"

namespace i8c {

namespace {

constexpr int kHold = 4;          // vectors a thread keeps in registers
constexpr int kMaxRowWarps = 16;

struct QuantizeArgs {
  const void *x;
  const int32_t *index;
  int8_t *q;
  float *scale;
  int64_t m, k, rows, ldx, ldq;
  int32_t vec_x, vec_q;
};

// Eight elements from column k0 on, zeros past the row.
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::type *row, int64_t k0, int64_t k,
                                      bool vec, float (&f)[8]) {
  using T = typename Elem<DT>::type;
  if (vec && k0 + 8 <= k) {
    constexpr int kPer = 16 / static_cast<int>(sizeof(T));
#pragma unroll
    for (int j = 0; j < 8 / kPer; ++j) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(row + k0) + j);
      const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int t = 0; t < kPer; ++t) f[j * kPer + t] = Elem<DT>::load(e[t]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = k0 + j < k ? Elem<DT>::load(row[k0 + j]) : 0.f;
  }
}

template <int DT, int WARPS>
__global__ void __launch_bounds__(WARPS < 4 ? 128 : 32 * WARPS)
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
  float held[kHold][8];
  uint32_t top = 0;
  if (valid) {
#pragma unroll
    for (int h = 0; h < kHold; ++h) {
      const int64_t k0 = static_cast<int64_t>(h * kRowThreads + t) * 8;
      if (k0 < a.k) {
        load8<DT>(row, k0, a.k, vec, held[h]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) held[h][j] = 0.f;
      }
    }
#pragma unroll
    for (int h = 0; h < kHold; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t b = __float_as_uint(held[h][j]) & 0x7fffffffu;
        top = b > top ? b : top;
      }
    for (int64_t k0 = static_cast<int64_t>(kHold * kRowThreads + t) * 8; k0 < a.k;
         k0 += kRowThreads * 8) {
      float f[8];
      load8<DT>(row, k0, a.k, vec, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t b = __float_as_uint(f[j]) & 0x7fffffffu;
        top = b > top ? b : top;
      }
    }
  }
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
  auto put = [&](int64_t k0, const float (&f)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // |x / scale| passes 127 only where the scale is a denormal.
        v[j] = zero ? 0.f : fminf(fmaxf(__fdiv_rn(f[4 * h + j], scale), -127.f), 127.f);
      }
      w[h] = pack_int8(v[0], v[1], v[2], v[3]);
    }
    if (a.vec_q != 0 && k0 + 8 <= a.k) {
      *reinterpret_cast<uint2 *>(q + k0) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < a.k) q[k0 + j] = static_cast<int8_t>(w[j >> 2] >> (8 * (j & 3)));
    }
  };
  if (!valid) {
#pragma unroll
    for (int h = 0; h < kHold; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) held[h][j] = 0.f;
  }
#pragma unroll
  for (int h = 0; h < kHold; ++h) {
    const int64_t k0 = static_cast<int64_t>(h * kRowThreads + t) * 8;
    if (k0 < a.k) put(k0, held[h]);
  }
  for (int64_t k0 = static_cast<int64_t>(kHold * kRowThreads + t) * 8; k0 < a.k;
       k0 += kRowThreads * 8) {
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (valid) load8<DT>(row, k0, a.k, vec, f);
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
