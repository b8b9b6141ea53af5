// group_norm.cu - group norm with an activation, channels last:
//   v = x[i,p,c] * scale[c];  y = act((v - mean_g) * rsqrt(var_g + eps) * gamma[c] + beta[c])
//
// The statistics of a group run over all pixels, so x is needed twice.
// Kernel 1 takes a chunk of an image's pixels to one (mean, squared
// deviations) pair per group; kernel 2 joins an image's pairs and writes y,
// reading x again (from L2, where it still is for all but the largest
// tensors).
//
// A thread owns one vector of VEC channels and walks down the pixels: 16-byte
// loads, a warp reads whole lines, and the channel's constants stay in
// registers.  Its sums are taken relative to the first value it saw (no
// cancellation for a large mean), turned into (count, mean, squares) and
// joined pairwise, threads to channels, channels to groups, chunks to images,
// always in the same order: the result does not depend on timing.
#include <cuda_runtime.h>
#include <math.h>

#include "epilogue.cuh"
#include "launch.h"
#include "sm100.cuh"

namespace i8c {

namespace {

constexpr int kThreads = 256;

struct NormArgs {
  const void *x;
  void *y;
  const float *scale, *gamma, *beta;
  float2 *partial;       // [n][chunks][groups] (mean, squared deviations)
  int64_t ldx, ldy;
  int64_t pixels;
  int32_t channels, groups, per_group;
  int32_t chunks;        // chunks of an image in kernel 1
  int64_t chunk_pixels;  // pixels of a chunk (the last may hold fewer)
  int32_t apply_chunks;  // chunks of an image in kernel 2
  int64_t apply_pixels;
  float eps, inv_out_scale;
  int32_t activation;
};

struct Moments {
  float n, mean, sq;
};

__device__ __forceinline__ Moments join(const Moments &a, const Moments &b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
  const float w = b.n / n;
  const float d = b.mean - a.mean;
  return Moments{n, a.mean + d * w, a.sq + b.sq + d * d * a.n * w};
}

__device__ __forceinline__ Moments join_warp(Moments m) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    Moments o;
    o.n = __shfl_down_sync(0xffffffffu, m.n, d);
    o.mean = __shfl_down_sync(0xffffffffu, m.mean, d);
    o.sq = __shfl_down_sync(0xffffffffu, m.sq, d);
    m = join(m, o);
  }
  return m;
}

template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const typename Elem<DT>::type *p, float (&f)[VEC]) {
  using T = typename Elem<DT>::type;
  if constexpr (VEC == 1) {
    f[0] = Elem<DT>::load(*p);
  } else {
    constexpr int kPer = 16 / static_cast<int>(sizeof(T));
#pragma unroll
    for (int j = 0; j < VEC / kPer; ++j) {
      const uint4 raw = reinterpret_cast<const uint4 *>(p)[j];
      const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int t = 0; t < kPer; ++t) f[j * kPer + t] = Elem<DT>::load(e[t]);
    }
  }
}

template <int OUT, int VEC>
__device__ __forceinline__ void store_vec(typename Elem<OUT>::type *p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = Elem<OUT>::store(f[0]);
  } else if constexpr (OUT == INT8CONV_FP32) {
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j)
      reinterpret_cast<float4 *>(p)[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
  } else if constexpr (OUT == INT8CONV_INT8) {
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(pack_int8(f[0], f[1], f[2], f[3]), pack_int8(f[4], f[5], f[6], f[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = OUT == INT8CONV_BF16 ? pack_bf16(f[2 * j], f[2 * j + 1]) : pack_fp16(f[2 * j], f[2 * j + 1]);
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Kernel 1.  Dynamic shared memory: kThreads * VEC (mean, squares) pairs.
template <int DT, int VEC>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(const NormArgs a) {
  extern __shared__ float2 cell[];   // [row of threads][channel of the column tile]
  using T = typename Elem<DT>::type;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t image = blockIdx.x / a.chunks;
  const int chunk = static_cast<int>(blockIdx.x % a.chunks);
  const int64_t begin = chunk * a.chunk_pixels;
  const int64_t end = begin + a.chunk_pixels < a.pixels ? begin + a.chunk_pixels : a.pixels;
  const T *x = static_cast<const T *>(a.x) + image * a.pixels * a.ldx;
  const int cols = a.channels / VEC;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (mean, squares) of every channel of the chunk.
  float2 *channel = cell + kThreads * VEC;   // [channels]
  for (int col0 = 0; col0 < cols; col0 += kThreads) {
    const int width = cols - col0 < kThreads ? cols - col0 : kThreads;
    const int lanes = kThreads / width;      // threads that share a column
    const int col = threadIdx.x % width;
    const int part = threadIdx.x / width;
    if (part < lanes) {
      const int c0 = (col0 + col) * VEC;
      float s[VEC], x0[VEC], s1[VEC], s2[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        s[j] = a.scale != nullptr ? __ldg(a.scale + c0 + j) : 1.f;
        x0[j] = s1[j] = s2[j] = 0.f;
      }
      int64_t p = begin + part;
      float f[VEC];
      if (p < end) {
        load_vec<DT, VEC>(x + p * a.ldx + c0, f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x0[j] = f[j] * s[j];
        p += lanes;
      }
#pragma unroll 4
      for (; p < end; p += lanes) {
        load_vec<DT, VEC>(x + p * a.ldx + c0, f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = fmaf(f[j], s[j], -x0[j]);
          s1[j] += d;
          s2[j] = fmaf(d, d, s2[j]);
        }
      }
      const int64_t count = begin + part < end ? (end - begin - part + lanes - 1) / lanes : 0;
      const float inv = count > 0 ? 1.f / static_cast<float>(count) : 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = s1[j] * inv;
        const float sq = s2[j] - s1[j] * d;
        cell[part * width * VEC + col * VEC + j] = make_float2(x0[j] + d, sq > 0.f || sq != sq ? sq : 0.f);
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width * VEC; c += kThreads) {
      Moments m{0.f, 0.f, 0.f};
      for (int q = 0; q < lanes; ++q) {
        const int64_t count = begin + q < end ? (end - begin - q + lanes - 1) / lanes : 0;
        const float2 e = cell[q * width * VEC + c];
        m = join(m, Moments{static_cast<float>(count), e.x, e.y});
      }
      channel[col0 * VEC + c] = make_float2(m.mean, m.sq);
    }
    __syncthreads();
  }
  const float rows = static_cast<float>(end - begin);
  for (int g = warp; g < a.groups; g += kThreads / 32) {
    Moments m{0.f, 0.f, 0.f};
    for (int c = lane; c < a.per_group; c += 32) {
      const float2 e = channel[g * a.per_group + c];
      m = join(m, Moments{rows, e.x, e.y});
    }
    m = join_warp(m);
    if (lane == 0)
      a.partial[(image * a.chunks + chunk) * a.groups + g] =
          make_float2(m.mean, m.sq);
  }
}

// Rows [begin, end) of one image through the norm; mean[] and rstd[] of its
// groups in shared memory.
template <int DT, int OUT, int VEC, int ACT>
__device__ __forceinline__ void apply_rows(const NormArgs &a, const typename Elem<DT>::type *x,
                                           typename Elem<OUT>::type *y, int64_t begin, int64_t end,
                                           const float *mean, const float *rstd) {
  const int cols = a.channels / VEC;
  for (int col0 = 0; col0 < cols; col0 += kThreads) {
    const int width = cols - col0 < kThreads ? cols - col0 : kThreads;
    const int lanes = kThreads / width;
    const int col = threadIdx.x % width;
    const int part = threadIdx.x / width;
    if (part >= lanes) continue;
    const int c0 = (col0 + col) * VEC;
    float s[VEC], m[VEC], w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int g = (c0 + j) / a.per_group;
      s[j] = a.scale != nullptr ? __ldg(a.scale + c0 + j) : 1.f;
      m[j] = mean[g];
      w[j] = rstd[g] * (a.gamma != nullptr ? __ldg(a.gamma + c0 + j) : 1.f);
      b[j] = a.beta != nullptr ? __ldg(a.beta + c0 + j) : 0.f;
    }
    auto finish = [&](float (&f)[VEC], int64_t p) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        f[j] = activate<ACT>(fmaf(fmaf(f[j], s[j], -m[j]), w[j], b[j]));
        if constexpr (OUT == INT8CONV_INT8) f[j] *= a.inv_out_scale;
      }
      store_vec<OUT, VEC>(y + p * a.ldy + c0, f);
    };
    // Several pixels are read before the first is written: y may be x, so the
    // compiler may not move a load above a store itself.
    constexpr int kBatch = 4;
    int64_t p = begin + part;
    for (; p + (kBatch - 1) * lanes < end; p += kBatch * lanes) {
      float f[kBatch][VEC];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) load_vec<DT, VEC>(x + (p + u * lanes) * a.ldx + c0, f[u]);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) finish(f[u], p + u * lanes);
    }
    for (; p < end; p += lanes) {
      float f[VEC];
      load_vec<DT, VEC>(x + p * a.ldx + c0, f);
      finish(f, p);
    }
  }
}

template <int DT, int OUT, int VEC>
__device__ __forceinline__ void apply_rows_act(const NormArgs &a, const typename Elem<DT>::type *x,
                                               typename Elem<OUT>::type *y, int64_t begin,
                                               int64_t end, const float *mean, const float *rstd) {
  switch (a.activation) {
    case INT8CONV_ACT_RELU:
      apply_rows<DT, OUT, VEC, INT8CONV_ACT_RELU>(a, x, y, begin, end, mean, rstd);
      break;
    case INT8CONV_ACT_GELU:
      apply_rows<DT, OUT, VEC, INT8CONV_ACT_GELU>(a, x, y, begin, end, mean, rstd);
      break;
    case INT8CONV_ACT_GELU_TANH:
      apply_rows<DT, OUT, VEC, INT8CONV_ACT_GELU_TANH>(a, x, y, begin, end, mean, rstd);
      break;
    case INT8CONV_ACT_SILU:
      apply_rows<DT, OUT, VEC, INT8CONV_ACT_SILU>(a, x, y, begin, end, mean, rstd);
      break;
    default:
      apply_rows<DT, OUT, VEC, INT8CONV_ACT_NONE>(a, x, y, begin, end, mean, rstd);
  }
}

// Kernel 2.  Dynamic shared memory: mean[groups], rstd[groups].
template <int DT, int OUT, int VEC>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(const NormArgs a) {
  extern __shared__ float stats[];
  using T = typename Elem<DT>::type;
  using O = typename Elem<OUT>::type;
  float *mean = stats, *rstd = stats + a.groups;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t image = blockIdx.x / a.apply_chunks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < a.groups; g += kThreads / 32) {
    Moments m{0.f, 0.f, 0.f};
    for (int k = lane; k < a.chunks; k += 32) {
      const int64_t begin = k * a.chunk_pixels;
      const int64_t rows = begin + a.chunk_pixels < a.pixels ? a.chunk_pixels : a.pixels - begin;
      const float2 e = a.partial[(image * a.chunks + k) * a.groups + g];
      m = join(m, Moments{static_cast<float>(rows) * a.per_group, e.x, e.y});
    }
    m = join_warp(m);
    if (lane == 0) {
      mean[g] = m.mean;
      rstd[g] = rsqrtf(m.sq / m.n + a.eps);
    }
  }
  __syncthreads();
  const int64_t begin = (blockIdx.x % a.apply_chunks) * a.apply_pixels;
  const int64_t end = begin + a.apply_pixels < a.pixels ? begin + a.apply_pixels : a.pixels;
  const T *x = static_cast<const T *>(a.x) + image * a.pixels * a.ldx;
  O *y = static_cast<O *>(a.y) + image * a.pixels * a.ldy;
  apply_rows_act<DT, OUT, VEC>(a, x, y, begin, end, mean, rstd);
}

template <int DT, int VEC>
const void *apply_for(int out) {
  switch (out) {
    case INT8CONV_BF16:
      return reinterpret_cast<const void *>(&norm_apply_kernel<DT, INT8CONV_BF16, VEC>);
    case INT8CONV_FP16:
      return reinterpret_cast<const void *>(&norm_apply_kernel<DT, INT8CONV_FP16, VEC>);
    case INT8CONV_FP32:
      return reinterpret_cast<const void *>(&norm_apply_kernel<DT, INT8CONV_FP32, VEC>);
    default:
      return reinterpret_cast<const void *>(&norm_apply_kernel<DT, INT8CONV_INT8, VEC>);
  }
}

template <int DT>
void kernels_for(bool vec, int out, const void **stats, const void **apply) {
  *stats = vec ? reinterpret_cast<const void *>(&norm_stats_kernel<DT, 8>)
               : reinterpret_cast<const void *>(&norm_stats_kernel<DT, 1>);
  *apply = vec ? apply_for<DT, 8>(out) : apply_for<DT, 1>(out);
}

// Chunks of an image: enough CTAs for the GPU four times over all images, but
// at least 16 KB of channels x pixels each.
int64_t pick_chunk_pixels(const int8conv_group_norm &d) {
  const int64_t want = (4 * 148 + d.n - 1) / d.n;
  int64_t pixels = (d.pixels + want - 1) / want;
  const int64_t least = (8192 + d.channels - 1) / d.channels;
  return pixels > least ? pixels : least;
}

}  // namespace

int64_t group_norm_blocks(const int8conv_group_norm &d) {
  if (d.n == 0 || d.pixels == 0) return 0;
  const int64_t per = pick_chunk_pixels(d);
  return d.n * ((d.pixels + per - 1) / per);
}

size_t group_norm_workspace(const int8conv_group_norm &d) {
  return static_cast<size_t>(group_norm_blocks(d)) * static_cast<size_t>(d.groups) * sizeof(float2);
}

int8conv_status launch_group_norm_impl(const int8conv_group_norm &d, const void *x, void *y,
                                       void *workspace, cudaStream_t stream) {
  NormArgs a{};
  a.x = x;
  a.y = y;
  a.scale = d.scale;
  a.gamma = d.gamma;
  a.beta = d.beta;
  a.partial = static_cast<float2 *>(workspace);
  a.ldx = d.ldx;
  a.ldy = d.ldy;
  a.pixels = d.pixels;
  a.channels = d.channels;
  a.groups = d.groups;
  a.per_group = d.channels / d.groups;
  a.chunk_pixels = pick_chunk_pixels(d);
  a.chunks = static_cast<int32_t>((d.pixels + a.chunk_pixels - 1) / a.chunk_pixels);
  a.apply_pixels = a.chunk_pixels;
  a.apply_chunks = a.chunks;
  a.eps = d.eps;
  a.inv_out_scale = d.y_dtype == INT8CONV_INT8 ? 1.0f / d.out_scale : 1.0f;
  a.activation = d.activation;
  // Vectors of 8 channels where every row of x and y allows the wide accesses
  // (16 bytes; 8 for int8 rows).
  const int xs = dtype_bytes(d.x_dtype), ys = dtype_bytes(d.y_dtype);
  const int ya = ys == 1 ? 8 : 16;
  const bool vec = d.channels % 8 == 0 && (d.ldx * xs) % 16 == 0 && (d.ldy * ys) % ya == 0 &&
                   (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(y) & (ya - 1)) == 0;
  const void *stats = nullptr, *apply = nullptr;
  switch (d.x_dtype) {
    case INT8CONV_BF16:
      kernels_for<INT8CONV_BF16>(vec, d.y_dtype, &stats, &apply);
      break;
    case INT8CONV_FP16:
      kernels_for<INT8CONV_FP16>(vec, d.y_dtype, &stats, &apply);
      break;
    case INT8CONV_FP32:
      kernels_for<INT8CONV_FP32>(vec, d.y_dtype, &stats, &apply);
      break;
    default:
      kernels_for<INT8CONV_INT32>(vec, d.y_dtype, &stats, &apply);
  }
  LaunchPlan plan;
  plan.func = stats;
  plan.grid = dim3(static_cast<unsigned>(a.chunks * d.n));
  plan.block = dim3(kThreads);
  plan.smem = static_cast<uint32_t>((kThreads * (vec ? 8 : 1) + d.channels) * sizeof(float2));
  if (!ensure_smem_attr(plan.func, static_cast<int>(plan.smem))) return INT8CONV_CUDA_ERROR;
  plan_args(plan, a);
  int8conv_status st = launch_plan(plan, stream);
  if (st != INT8CONV_OK) return st;
  plan.func = apply;
  plan.grid = dim3(static_cast<unsigned>(a.apply_chunks * d.n));
  plan.smem = static_cast<uint32_t>(2 * d.groups * sizeof(float));
  if (!ensure_smem_attr(plan.func, static_cast<int>(plan.smem))) return INT8CONV_CUDA_ERROR;
  return launch_plan(plan, stream);
}

}  // namespace i8c
