// group_norm.cu - group norm with an activation, channels last:
//   v = x[i,p,c] * scale[c];  y = act((v - mean_g) * rsqrt(var_g + eps) * gamma[c] + beta[c])
//
// The statistics of a group run over all pixels of an image, so every value is
// needed twice.  Two forms:
//   one kernel   a thread-block cluster of 1 to 8 CTAs holds an image: each CTA
//                takes a span of pixels, keeps as much of it as fits in shared
//                memory, and the CTAs exchange their groups' partial statistics
//                through distributed shared memory.  What was kept is read once,
//                the rest of x again.
//   two kernels  for few large images, whose clusters would leave SMs idle:
//                statistics of pixel chunks to scratch, then the norm, reading
//                x again (from L2 while it fits there).
//
// A thread owns one vector of 8 channels and walks down the pixels: 16-byte
// loads, a warp reads whole lines.  Sums are taken in fp32 about a shift that
// follows the mean (span_stats), of float inputs with a scale as x * scale -
// shift, so that x may have any size that the scale makes ordinary.  int32 inputs
// are summed as they are (no square of theirs leaves fp32's range), and the scale
// is applied to the channel's mean and squares.  Threads, channels, CTAs and
// chunks are joined as (mean, squared deviations) in a fixed order, so the result
// does not depend on timing.
//
// Measured: 256 images of 3136 x 256 int32 to fp16 317 us, DRAM at 6.4 TB/s with x
// read twice (one CTA holds an image of 3.2 MB, of which it keeps 0.1); 8 of
// 4096 x 320 bf16 to bf16 with silu 18.8 us, two kernels bound by the latency of
// their loads and reductions (and, with silu, by the two special functions of each
// element); one of 196 x 256 int32 6.7 us, where a launch alone takes 2.3.
//
// Two CTAs of 512 threads an SM leave a thread 64 registers, and the vector kernels
// spill some, before and after their loops (bf16 to bf16, bytes stored / loaded a
// thread: one kernel 108 / 92; two kernels 4 / 4 and 140 / 156, of which 12 loads a
// warp were executed over 2 x 65536 x 256).
#include <cuda_runtime.h>
#include <math.h>

#include "epilogue.cuh"
#include "int8conv_rules.h"
#include "launch.h"
#include "sm100.cuh"

namespace i8c {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
// Shared memory of a CTA that leaves room for another on its SM (228 KB, of
// which each CTA takes 1 KB for itself): one loads while the other reduces or
// stores.
constexpr uint32_t kHalfSmem = 113 * 1024;

struct NormArgs {
  const void *x;
  void *y;
  const float *scale, *gamma, *beta;
  float2 *partial;       // two kernels: [n][groups][spans] (mean, squared deviations)
  int64_t ldx, ldy;
  int32_t pixels;
  int32_t channels, groups, per_group;
  int32_t spans;         // spans of an image: CTAs of its cluster, or chunks
  int32_t span_pixels;   // pixels of a span (the last ones may hold fewer, or none)
  int32_t keep;          // vectors each thread keeps in shared memory
  float eps, inv_out_scale;
  int32_t activation;
};

// Shared memory, in this order: kept vectors, the threads' sums, three values
// of each channel, the CTA's group statistics, the image's.
struct NormSmem {
  uint32_t cell_off, channel_off, part_off, stat_off, total;
};

__host__ __device__ inline NormSmem norm_smem(int vec, int raw_bytes, int channels, int groups,
                                              int keep) {
  NormSmem p;
  p.cell_off = static_cast<uint32_t>(keep) * kThreads * vec * raw_bytes;
  p.channel_off = p.cell_off + kThreads * vec * sizeof(float);
  const uint32_t padded = (channels + 3) & ~3u;   // each array starts 16-byte aligned
  p.part_off = p.channel_off + 3 * padded * sizeof(float);
  p.stat_off = p.part_off + groups * sizeof(float2);
  p.total = p.stat_off + groups * sizeof(float2);
  return p;
}

// Three arrays over the channels.  Statistics: the shift, then the mean; sums,
// then squares.  Norm: y = act((x - m) * w + b), m in the input's own units.
struct Channels {
  float *m, *w, *b;
  __device__ __forceinline__ Channels(uint8_t *smem, const NormSmem &plan, int channels) {
    const int padded = (channels + 3) & ~3;
    m = reinterpret_cast<float *>(smem + plan.channel_off);
    w = m + padded;
    b = w + padded;
  }
};

// scale, gamma and beta of one channel.
struct Params {
  float scale, gamma, beta;
  __device__ __forceinline__ Params(const NormArgs &a, int c) {
    const bool in = c < a.channels;
    scale = in && a.scale != nullptr ? __ldg(a.scale + c) : 1.f;
    gamma = in && a.gamma != nullptr ? __ldg(a.gamma + c) : 1.f;
    beta = in && a.beta != nullptr ? __ldg(a.beta + c) : 0.f;
  }
};

// VEC elements as they lie in memory.
template <int DT, int VEC>
struct Raw {
  using T = typename Elem<DT>::type;
  static constexpr int kWords = VEC == 1 ? 1 : VEC * static_cast<int>(sizeof(T)) / 16;
  uint4 w[kWords];   // VEC == 1: the element alone, in w[0].x

  __device__ __forceinline__ void load(const T *p) {
    if constexpr (VEC == 1) {
      *reinterpret_cast<T *>(&w[0].x) = *p;
    } else {
#pragma unroll
      for (int j = 0; j < kWords; ++j) w[j] = reinterpret_cast<const uint4 *>(p)[j];
    }
  }
  __device__ __forceinline__ float get(int j) const {
    return Elem<DT>::load(reinterpret_cast<const T *>(&w[0])[j]);
  }
  // A kept vector, word by word at `slot` + threadIdx.x, so that a warp's
  // accesses are contiguous.  VEC == 8 only.
  __device__ __forceinline__ void keep(uint4 *slot) const {
#pragma unroll
    for (int j = 0; j < kWords; ++j) slot[j * kThreads + threadIdx.x] = w[j];
  }
  __device__ __forceinline__ void kept(const uint4 *slot) {
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = slot[j * kThreads + threadIdx.x];
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
};

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

template <int VEC>
__device__ __forceinline__ void put_vec(float *p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = v[0];
  } else {
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j)
      reinterpret_cast<float4 *>(p)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
}
template <int VEC>
__device__ __forceinline__ void get_vec(const float *p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = *p;
  } else {
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
      const float4 t = reinterpret_cast<const float4 *>(p)[j];
      v[4 * j] = t.x;
      v[4 * j + 1] = t.y;
      v[4 * j + 2] = t.z;
      v[4 * j + 3] = t.w;
    }
  }
}

// How the CTA's threads share a tile of at most kThreads columns (vectors of
// VEC channels): `lanes` threads down each column.
struct Columns {
  int width, lanes, col, part;
  __device__ __forceinline__ Columns(int cols, int col0) {
    width = cols - col0 < kThreads ? cols - col0 : kThreads;
    lanes = kThreads / width;
    col = static_cast<int>(threadIdx.x) % width;
    part = static_cast<int>(threadIdx.x) / width;
  }
};

// Pixels read before the first of them is used.
template <int DT, int VEC>
constexpr int batch() {
  return VEC == 1 ? 8 : (sizeof(typename Elem<DT>::type) == 2 ? 4 : 2);
}

__device__ __forceinline__ int rows_of(const NormArgs &a, int span) {
  const int left = a.pixels - span * a.span_pixels;
  return left <= 0 ? 0 : (left < a.span_pixels ? left : a.span_pixels);
}

// Batches of a run: a thread adds the squares of this many batches before it adds
// the run's sum to the runs' before it.
constexpr int kRun = 16;   // 32, 64 or 128 pixels

// (mean, squared deviations) of every channel over pixels [0, rows) of x, this
// CTA's span, into ch.m and ch.w.  `mine`: the parameters of channel threadIdx.x.
//
// A thread sums d = x - shift and d^2 of its own pixels, the shift its first
// pixel.  Where it has more than 16 (and a batch), the shift moves to the mean so
// far after 8 pixels, 32, twice that up to a run, and every further run, the sums
// with it:
//   e = s1 / n,  s2 <- s2 - e (2 s1 - n e),  s1 <- s1 - n e,  shift <- shift + e
// No step cancels, wherever an outlier lies: the shift is the mean of a part of
// the values, and the squares about the mean of m of n values are at most n / m
// times the squared deviations: up to 24 where that is all (16 and a batch), 8 in
// the first 8, 4 from there to 32, and from then on 2.  The longest chain of
// additions of squares is a run (32 to 128), then the runs.  A thread's squares of
// finished runs lie in its `cell`, which is free until the sums are joined.
// SCALED: each value times its channel's scale.
//
// On small images what is executed once counts by its length (the instructions
// come from L2): the sums move as pairs.
template <int DT, int VEC, bool SCALED>
__device__ __forceinline__ void span_sums(const NormArgs &a, const typename Elem<DT>::type *x,
                                          int rows, uint8_t *area, float *cell,
                                          const Channels &ch, const Params &mine) {
  using T = typename Elem<DT>::type;
  constexpr int kBatch = batch<DT, VEC>();
  constexpr int kPairs = (VEC + 1) / 2;   // one channel alone: the pair's other half is 0
  const int cols = a.channels / VEC;
  uint4 *slot = reinterpret_cast<uint4 *>(area);
  int kept = a.keep;   // full batches go to shared memory until this many vectors lie there
  for (int col0 = 0; col0 < cols; col0 += kThreads) {
    const Columns k(cols, col0);
    const bool active = k.part < k.lanes;
    const int wide = k.width * VEC, c0 = col0 * VEC;
    float *own = cell + k.part * wide + k.col * VEC;   // this thread's place (active threads)
    // The first `more` threads of a column hold one pixel more than the others.
    const int each = rows / k.lanes, more = rows - each * k.lanes;
    const int pixels = active ? each + (k.part < more ? 1 : 0) : 0;
    uint64_t x0[kPairs], s1[kPairs], s2[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) x0[j] = s1[j] = s2[j] = 0;
    auto put = [&](const uint64_t (&v)[kPairs]) {
      float f[2 * kPairs];
#pragma unroll
      for (int j = 0; j < kPairs; ++j) f2_unpack(v[j], f[2 * j], f[2 * j + 1]);
      if constexpr (VEC == 1)
        own[0] = f[0];
      else
        put_vec<VEC>(own, f);
    };
    auto add_own = [&](uint64_t (&v)[kPairs]) {
      float f[2 * kPairs] = {};
      if constexpr (VEC == 1)
        f[0] = own[0];
      else
        get_vec<VEC>(own, f);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[j] = f2_add(v[j], f2_pack(f[2 * j], f[2 * j + 1]));
    };
    if (pixels > 0) {
      [[maybe_unused]] float by[VEC];
      if constexpr (SCALED) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) by[j] = __ldg(a.scale + c0 + k.col * VEC + j);
      }
      const T *at = x + (col0 + k.col) * VEC + k.part * a.ldx;
      const int64_t step = k.lanes * a.ldx;
      auto pair = [&](const Raw<DT, VEC> &r, int j) {
        if constexpr (VEC == 1)
          return f2_pack(r.get(0), 0.f);
        else
          return r.pair(2 * j);
      };
      auto times = [&](int j) {
        if constexpr (!SCALED)
          return f2_pack(1.f, 1.f);
        else if constexpr (VEC == 1)
          return f2_pack(by[0], 0.f);
        else
          return f2_pack(by[2 * j], by[2 * j + 1]);
      };
      auto start = [&](const Raw<DT, VEC> &r) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
          x0[j] = SCALED ? f2_mul(pair(r, j), times(j)) : pair(r, j);
      };
      auto add = [&](const Raw<DT, VEC> &r) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const uint64_t minus = f2_neg(x0[j]);
          const uint64_t d = SCALED ? f2_fma(pair(r, j), times(j), minus) : f2_add(pair(r, j), minus);
          s1[j] = f2_add(s1[j], d);
          s2[j] = f2_fma(d, d, s2[j]);
        }
      };
      // The sums of n pixels move to their mean (to any value near it: the sums
      // are exact about the shift, whatever it is).
      auto center = [&](float n) {
        const float i = rcp_approx(n);
        const uint64_t inv = f2_pack(i, i), minus_n = f2_pack(-n, -n);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const uint64_t to = f2_fma(s1[j], inv, x0[j]);
          const uint64_t e = f2_add(to, f2_neg(x0[j]));
          const uint64_t rest = f2_fma(minus_n, e, s1[j]);
          s2[j] = f2_fma(f2_neg(e), f2_add(s1[j], rest), s2[j]);
          s1[j] = rest;
          x0[j] = to;
        }
      };
      constexpr int kRunPixels = kRun * kBatch;
      int left = pixels;
      int mark = pixels > 16 + kBatch ? pixels - 8 : -1;   // center where `left` is this
#pragma unroll 1
      while (left >= kBatch) {
        Raw<DT, VEC> r[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u, at += step) r[u].load(at);
        if (left == pixels) start(r[0]);
        if constexpr (VEC > 1) {
          if (kept > 0) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u, slot += Raw<DT, VEC>::kWords * kThreads)
              r[u].keep(slot);
            kept -= kBatch;
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) add(r[u]);
        left -= kBatch;
        if (left == mark) {
          const int n = pixels - left;
          if (n > kRunPixels) add_own(s2);
          center(static_cast<float>(n));
          if (n < kRunPixels) {
            mark = pixels - (n == 8 ? 32 : 2 * n);
          } else {
            put(s2);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) s2[j] = 0;
            mark -= kRunPixels;
          }
        }
      }
#pragma unroll 1
      for (; left > 0; --left, at += step) {
        Raw<DT, VEC> r;
        r.load(at);
        if (left == pixels) start(r);
        add(r);
      }
      if (pixels >= kRunPixels) add_own(s2);
      // Now the mean, and the squares about it: less those of what its rounding
      // left, the squared deviations.
      if (pixels > 1) {
        const float n = static_cast<float>(pixels);
        center(n);
        const float i = -rcp_approx(n);
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
          s2[j] = f2_fma(f2_mul(s1[j], f2_pack(i, i)), s1[j], s2[j]);
      }
    }
    // The threads of a column join: first the means, relative to the first
    // thread's, then the squared deviations about the mean of all.
    if (active) put(x0);
    __syncthreads();
    const float inv = 1.f / static_cast<float>(rows > 0 ? rows : 1);
#pragma unroll 1
    for (int i = threadIdx.x; i < wide; i += kThreads) {
      const float ref = cell[i];
      float all = 0.f, head = 0.f;
#pragma unroll 4
      for (int q = 0; q < k.lanes; ++q) {
        const float d = cell[q * wide + i] - ref;
        all += d;
        if (q < more) head += d;
      }
      const float sum = fmaf(static_cast<float>(each), all, head);
      ch.m[c0 + i] = fmaf(sum, inv, ref);
    }
    __syncthreads();
    if (pixels > 0) {
      const float n = static_cast<float>(pixels);
      float mean[2 * kPairs] = {};
      if constexpr (VEC == 1)
        mean[0] = ch.m[c0 + k.col];
      else
        get_vec<VEC>(ch.m + c0 + k.col * VEC, mean);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const uint64_t d = f2_add(x0[j], f2_pack(-mean[2 * j], -mean[2 * j + 1]));
        s2[j] = f2_fma(f2_mul(d, f2_pack(n, n)), d, s2[j]);
      }
    }
    if (active) put(s2);
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < wide; i += kThreads) {
      const int c = c0 + i;
      float sq = 0.f;
#pragma unroll 4
      for (int q = 0; q < k.lanes; ++q) sq += cell[q * wide + i];
      if (sq < 0.f) sq = 0.f;   // a rounding's; NaN stays NaN
      if constexpr (SCALED) {
        ch.w[c] = sq;
      } else {
        const float s = c == static_cast<int>(threadIdx.x) ? mine.scale : Params(a, c).scale;
        ch.m[c] *= s;
        ch.w[c] = sq * s * s;
      }
    }
    __syncthreads();
  }
}

// The same of every group, into part[].
template <int DT, int VEC, bool SCALED>
__device__ __forceinline__ void span_stats(const NormArgs &a, const typename Elem<DT>::type *x,
                                           int rows, uint8_t *area, float *cell,
                                           const Channels &ch, const Params &mine, float2 *part) {
  span_sums<DT, VEC, SCALED>(a, x, rows, area, cell, ch, mine);
  // Channels of a group all hold `rows` values: the mean of means (relative to
  // the first, so that a large mean costs no bits), and the squares plus `rows`
  // times the means' squared deviations.  2 to 32 lanes share a group.
  const int lane = threadIdx.x & 31;
  int share = 2;
  while (share < 32 && share < a.per_group) share *= 2;
  const int sub = lane & (share - 1);
  const float inv = 1.f / static_cast<float>(a.per_group);
  const float n = static_cast<float>(rows);
#pragma unroll 1
  for (int g0 = 0; g0 < a.groups; g0 += kThreads / share) {
    const int g = g0 + static_cast<int>(threadIdx.x) / share;
    const int first = (g < a.groups ? g : 0) * a.per_group;
    const float ref = ch.m[first];
    float mean = 0.f, sq = 0.f;
#pragma unroll 1
    for (int c = sub; c < a.per_group; c += share) mean += ch.m[first + c] - ref;
#pragma unroll 1
    for (int d = share >> 1; d > 0; d >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, d);
    mean = fmaf(mean, inv, ref);
#pragma unroll 1
    for (int c = sub; c < a.per_group; c += share) {
      const float d = ch.m[first + c] - mean;
      sq += fmaf(d * n, d, ch.w[first + c]);
    }
#pragma unroll 1
    for (int d = share >> 1; d > 0; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
    if (sub == 0 && g < a.groups) part[g] = make_float2(mean, sq);
  }
}

// The channels' constants of y = act((x - m) * w + b) from the image's
// statistics stat[g] = (mean, 1 / deviation).
__device__ __forceinline__ void channel_constants(const NormArgs &a, const float2 *stat,
                                                  const Channels &ch, const Params &mine) {
#pragma unroll 1
  for (int c = threadIdx.x; c < a.channels; c += kThreads) {
    const Params p = c == static_cast<int>(threadIdx.x) ? mine : Params(a, c);
    const float2 t = stat[c / a.per_group];
    const float w = t.y * p.gamma;
    const float m = p.scale == 1.f ? t.x : t.x / p.scale;
    if (!(fabsf(m) <= 1e37f)) {
      // A channel that is worth next to nothing beside the group's mean, or
      // nothing: the mean goes into the offset.
      ch.m[c] = 0.f;
      ch.w[c] = w * p.scale;
      ch.b[c] = fmaf(-t.x, w, p.beta);
    } else {
      ch.m[c] = m;
      ch.w[c] = w * p.scale;
      ch.b[c] = p.beta;
    }
  }
  __syncthreads();
}

// Pixels [0, rows) of x through the norm into y.
template <int DT, int OUT, int VEC, int ACT>
__device__ __forceinline__ void apply_span(const NormArgs &a, const typename Elem<DT>::type *x,
                                           typename Elem<OUT>::type *y, int rows,
                                           const uint8_t *area, const Channels &ch) {
  using T = typename Elem<DT>::type;
  using O = typename Elem<OUT>::type;
  constexpr int kBatch = batch<DT, VEC>();
  const int cols = a.channels / VEC;
  const uint4 *slot = reinterpret_cast<const uint4 *>(area);
  int kept = a.keep;
  for (int col0 = 0; col0 < cols; col0 += kThreads) {
    const Columns k(cols, col0);
    if (k.part >= k.lanes) continue;
    const int c0 = (col0 + k.col) * VEC;
    float m[VEC], w[VEC], b[VEC];
    get_vec<VEC>(ch.m + c0, m);
    get_vec<VEC>(ch.w + c0, w);
    get_vec<VEC>(ch.b + c0, b);
    const T *at = x + k.part * a.ldx + c0;
    O *to = y + k.part * a.ldy + c0;
    const int64_t step = k.lanes * a.ldx, to_step = k.lanes * a.ldy;
    int left = k.part < rows ? (rows - k.part - 1) / k.lanes + 1 : 0;
    auto finish = [&](const Raw<DT, VEC> &r) {
      float f[VEC];
      if constexpr (VEC == 1) {
        f[0] = activate<ACT, OUT == INT8CONV_FP32>(fmaf(r.get(0) - m[0], w[0], b[0]));
        if constexpr (OUT == INT8CONV_INT8) f[0] *= a.inv_out_scale;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          const uint64_t d = f2_add(r.pair(j), f2_pack(-m[j], -m[j + 1]));
          f2_unpack(f2_fma(d, f2_pack(w[j], w[j + 1]), f2_pack(b[j], b[j + 1])), f[j], f[j + 1]);
          activate2<ACT, OUT == INT8CONV_FP32>(f[j], f[j + 1]);
          if constexpr (OUT == INT8CONV_INT8)
            f2_unpack(f2_mul(f2_pack(f[j], f[j + 1]), f2_pack(a.inv_out_scale, a.inv_out_scale)),
                      f[j], f[j + 1]);
        }
      }
      store_vec<OUT, VEC>(to, f);
      to += to_step;
    };
    // A batch is read before its first pixel is written: y may be x, so the
    // compiler may not move a load above a store itself.
#pragma unroll 1
    for (; left >= kBatch; left -= kBatch) {
      Raw<DT, VEC> r[kBatch];
      bool here = false;
      if constexpr (VEC > 1) {
        here = kept > 0;
        if (here) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u, slot += Raw<DT, VEC>::kWords * kThreads) r[u].kept(slot);
          kept -= kBatch;
          at += kBatch * step;
        }
      }
      if (!here) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u, at += step) r[u].load(at);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) finish(r[u]);
    }
#pragma unroll 1
    for (; left > 0; --left, at += step) {
      Raw<DT, VEC> r;
      r.load(at);
      finish(r);
    }
  }
}

template <int DT, int OUT, int VEC>
__device__ __forceinline__ void apply_span_act(const NormArgs &a, const typename Elem<DT>::type *x,
                                               typename Elem<OUT>::type *y, int rows,
                                               const uint8_t *area, const Channels &ch) {
  switch (a.activation) {
    case INT8CONV_ACT_RELU:
      apply_span<DT, OUT, VEC, INT8CONV_ACT_RELU>(a, x, y, rows, area, ch);
      break;
    case INT8CONV_ACT_GELU:
      apply_span<DT, OUT, VEC, INT8CONV_ACT_GELU>(a, x, y, rows, area, ch);
      break;
    case INT8CONV_ACT_GELU_TANH:
      apply_span<DT, OUT, VEC, INT8CONV_ACT_GELU_TANH>(a, x, y, rows, area, ch);
      break;
    case INT8CONV_ACT_SILU:
      apply_span<DT, OUT, VEC, INT8CONV_ACT_SILU>(a, x, y, rows, area, ch);
      break;
    default:
      apply_span<DT, OUT, VEC, INT8CONV_ACT_NONE>(a, x, y, rows, area, ch);
  }
}

__device__ __forceinline__ float2 finish_stat(const NormArgs &a, float mean, float sq) {
  const float n = static_cast<float>(a.pixels) * static_cast<float>(a.per_group);
  return make_float2(mean, rsqrtf(sq / n + a.eps));
}

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(addr)
               : "memory");
  return v;
}

constexpr int kMaxCluster = 8;

// One kernel: the CTAs of a cluster share an image.
template <int DT, int OUT, int VEC, bool SCALED>
__global__ void __launch_bounds__(kThreads, 2) norm_cluster_kernel(const NormArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  using T = typename Elem<DT>::type;
  using O = typename Elem<OUT>::type;
  const NormSmem plan = norm_smem(VEC, sizeof(T), a.channels, a.groups, a.keep);
  const Channels ch(smem, plan, a.channels);
  float2 *part = reinterpret_cast<float2 *>(smem + plan.part_off);
  float2 *stat = reinterpret_cast<float2 *>(smem + plan.stat_off);
  griddep_wait();
  griddep_launch_dependents();
  const Params mine(a, threadIdx.x);
  const int64_t image = blockIdx.x / a.spans;
  const int span = static_cast<int>(blockIdx.x) % a.spans;   // rank in the cluster
  const int rows = rows_of(a, span);
  const int64_t first = image * a.pixels + static_cast<int64_t>(span) * a.span_pixels;
  const T *x = static_cast<const T *>(a.x) + first * a.ldx;
  span_stats<DT, VEC, SCALED>(a, x, rows, smem, reinterpret_cast<float *>(smem + plan.cell_off), ch,
                              mine, part);
  cluster_sync_all();
  // 8 lanes share a group, one for each CTA of the cluster.
  const int k = threadIdx.x & (kMaxCluster - 1);
  const float n = k < a.spans ? static_cast<float>(rows_of(a, k)) : 0.f;
  const float share = n / static_cast<float>(a.pixels);
#pragma unroll 1
  for (int g0 = 0; g0 < a.groups; g0 += kThreads / kMaxCluster) {
    const int g = g0 + static_cast<int>(threadIdx.x) / kMaxCluster;
    float2 e = make_float2(0.f, 0.f);
    if (n > 0.f && g < a.groups) e = ld_cluster_f2(mapa_shared(smem_u32(part + g), k));
    const float ref = __shfl_sync(0xffffffffu, e.x, 0, kMaxCluster);   // span 0 is never empty
    float mean = n > 0.f ? share * (e.x - ref) : 0.f;
#pragma unroll
    for (int d = kMaxCluster / 2; d > 0; d >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, d);
    mean += ref;
    const float dev = e.x - mean;
    float sq = n > 0.f ? fmaf(dev * n * static_cast<float>(a.per_group), dev, e.y) : 0.f;
#pragma unroll
    for (int d = kMaxCluster / 2; d > 0; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
    if (k == 0 && g < a.groups) stat[g] = finish_stat(a, mean, sq);
  }
  // No CTA leaves while another may still read its part; and stat[] is complete.
  cluster_sync_all();
  channel_constants(a, stat, ch, mine);
  O *y = static_cast<O *>(a.y) + first * a.ldy;
  apply_span_act<DT, OUT, VEC>(a, x, y, rows, smem, ch);
}

// Two kernels, the first: statistics of one chunk of pixels.
template <int DT, int VEC, bool SCALED>
__global__ void __launch_bounds__(kThreads, 2) norm_stats_kernel(const NormArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  using T = typename Elem<DT>::type;
  const NormSmem plan = norm_smem(VEC, sizeof(T), a.channels, a.groups, 0);
  const Channels ch(smem, plan, a.channels);
  float2 *part = reinterpret_cast<float2 *>(smem + plan.part_off);
  griddep_wait();
  griddep_launch_dependents();
  const Params mine(a, threadIdx.x);
  const int64_t image = blockIdx.x / a.spans;
  const int span = static_cast<int>(blockIdx.x) % a.spans;
  const int64_t first = image * a.pixels + static_cast<int64_t>(span) * a.span_pixels;
  span_stats<DT, VEC, SCALED>(a, static_cast<const T *>(a.x) + first * a.ldx, rows_of(a, span),
                              smem, reinterpret_cast<float *>(smem + plan.cell_off), ch, mine,
                              part);
  __syncthreads();
  for (int g = threadIdx.x; g < a.groups; g += kThreads)
    a.partial[(image * a.groups + g) * a.spans + span] = part[g];
}

// The second: a warp joins the chunks of a group, then the chunk is normalised.
template <int DT, int OUT, int VEC>
__global__ void __launch_bounds__(kThreads, 2) norm_apply_kernel(const NormArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  using T = typename Elem<DT>::type;
  using O = typename Elem<OUT>::type;
  const NormSmem plan = norm_smem(VEC, sizeof(T), a.channels, a.groups, 0);
  const Channels ch(smem, plan, a.channels);
  float2 *stat = reinterpret_cast<float2 *>(smem + plan.stat_off);
  griddep_wait();
  griddep_launch_dependents();
  const Params mine(a, threadIdx.x);
  const int64_t image = blockIdx.x / a.spans;
  const int span = static_cast<int>(blockIdx.x) % a.spans;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float inv = 1.f / static_cast<float>(a.pixels);
  for (int g = warp; g < a.groups; g += kWarps) {
    const float2 *e = a.partial + (image * a.groups + g) * a.spans;
    const float ref = e[0].x;
    float mean = 0.f, sq = 0.f;
    for (int k = lane; k < a.spans; k += 32)
      mean = fmaf(static_cast<float>(rows_of(a, k)) * inv, e[k].x - ref, mean);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, d);
    mean += ref;
    for (int k = lane; k < a.spans; k += 32) {
      const float n = static_cast<float>(rows_of(a, k)) * static_cast<float>(a.per_group);
      const float d = e[k].x - mean;
      sq += fmaf(d * n, d, e[k].y);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
    if (lane == 0) stat[g] = finish_stat(a, mean, sq);
  }
  __syncthreads();
  channel_constants(a, stat, ch, mine);
  const int64_t first = image * a.pixels + static_cast<int64_t>(span) * a.span_pixels;
  apply_span_act<DT, OUT, VEC>(a, static_cast<const T *>(a.x) + first * a.ldx,
                               static_cast<O *>(a.y) + first * a.ldy, rows_of(a, span), smem, ch);
}

struct NormKernels {
  const void *cluster, *stats, *apply;
};

template <int DT, int OUT, int VEC, bool SCALED>
NormKernels kernels_of() {
  return NormKernels{reinterpret_cast<const void *>(&norm_cluster_kernel<DT, OUT, VEC, SCALED>),
                     reinterpret_cast<const void *>(&norm_stats_kernel<DT, VEC, SCALED>),
                     reinterpret_cast<const void *>(&norm_apply_kernel<DT, OUT, VEC>)};
}

template <int DT, int VEC, bool SCALED>
NormKernels kernels_for_out(int out) {
  switch (out) {
    case INT8CONV_BF16:
      return kernels_of<DT, INT8CONV_BF16, VEC, SCALED>();
    case INT8CONV_FP16:
      return kernels_of<DT, INT8CONV_FP16, VEC, SCALED>();
    case INT8CONV_FP32:
      return kernels_of<DT, INT8CONV_FP32, VEC, SCALED>();
    default:
      return kernels_of<DT, INT8CONV_INT8, VEC, SCALED>();
  }
}

template <int DT>
NormKernels kernels_for(bool vec, bool scaled, int out) {
  if constexpr (DT != INT8CONV_INT32) {   // int32 takes its scale after the sums
    if (scaled) return vec ? kernels_for_out<DT, 8, true>(out) : kernels_for_out<DT, 1, true>(out);
  }
  return vec ? kernels_for_out<DT, 8, false>(out) : kernels_for_out<DT, 1, false>(out);
}

// How a call runs: spans of an image, and whether they are one cluster.
struct NormShape {
  bool cluster;
  int spans;
  int64_t span_pixels;
};

NormShape norm_shape(const int8conv_group_norm &d) {
  const int64_t bytes = d.pixels * d.channels * dtype_bytes(d.x_dtype);   // of one image
  // Clusters that fill the GPU: 128 CTAs, or, with 16 MB and more to read, two
  // for each SM (measured, us: 32 images of 196 x 512 bf16 in clusters of 1 / 4 /
  // 8: 15.6 / 9.6 / 11.1; 64 of 3136 x 256 int32: 191 / 86 / 90).  16 CTAs never
  // pay: at most 7 such clusters find room on the GPU at one time.
  const int64_t total = d.n * bytes;
  const int64_t want = total < (16 << 20) ? 128 : 256;
  int spans = 1;
  while (spans < kMaxCluster && d.n * spans < want && bytes > spans * int64_t(8 * 1024)) spans *= 2;
  if (spans > d.pixels) spans = 1;
  NormShape s{true, spans, (d.pixels + spans - 1) / spans};
  // Few images with much for each CTA of such a cluster: two kernels over chunks
  // of all images (8 images of 4096 x 320 bf16: 19.2 us, in clusters of 8 28.4; 1
  // image 9.9 and 24.6; 16 of 8192 x 256 50 and 91; but 10 of 1400 x 112 10.4 and
  // 8.4, 32 of 4096 x 512 100 and 83).  One, two or four chunks for each of the 148
  // SMs, by what there is to read (bf16 with silu, 148 / 296 / 592 chunks, us: 10 MB
  // 13.7 / 14.6 / 24.2; 14 MB 19.3 / 22.8 / 25.0; 20 MB 24.4 / 18.9 / 26.9; 40 MB
  // 42.0 / 29.0 / 36.5; 56 MB 56.8 / 49.7 / 52.0; 147 MB 133 / 126 / 112; one image
  // of 98 MB 78 / 67 / 79).
  const int64_t each = bytes / spans;
  if ((d.n * spans < 96 && each > 64 * 1024) || (d.n * spans <= 148 && each > 256 * 1024)) {
    const int64_t all = total > (64 << 20) ? 592 : total > (19 << 20) ? 296 : 148;
    int64_t chunks = (all + d.n - 1) / d.n;
    if (chunks > d.pixels) chunks = d.pixels;
    s.cluster = false;
    s.span_pixels = (d.pixels + chunks - 1) / chunks;
    s.spans = static_cast<int>((d.pixels + s.span_pixels - 1) / s.span_pixels);
  }
  return s;
}

}  // namespace

int64_t group_norm_blocks(const int8conv_group_norm &d) {
  if (d.n == 0 || d.pixels == 0) return 0;
  return d.n * norm_shape(d).spans;
}

size_t group_norm_workspace(const int8conv_group_norm &d) {
  if (d.n == 0 || d.pixels == 0) return 0;
  const NormShape s = norm_shape(d);
  return s.cluster ? 0 : static_cast<size_t>(d.n) * s.spans * d.groups * sizeof(float2);
}

int8conv_status launch_group_norm_impl(const int8conv_group_norm &d, const void *x, void *y,
                                       void *workspace, cudaStream_t stream) {
  const NormShape shape = norm_shape(d);
  NormArgs a{};
  a.x = x;
  a.y = y;
  a.scale = d.scale;
  a.gamma = d.gamma;
  a.beta = d.beta;
  a.partial = static_cast<float2 *>(workspace);
  a.ldx = d.ldx;
  a.ldy = d.ldy;
  a.pixels = static_cast<int32_t>(d.pixels);
  a.channels = d.channels;
  a.groups = d.groups;
  a.per_group = d.channels / d.groups;
  a.spans = shape.spans;
  a.span_pixels = static_cast<int32_t>(shape.span_pixels);
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
  const bool scaled = d.scale != nullptr;
  const NormKernels kernels =
      d.x_dtype == INT8CONV_BF16   ? kernels_for<INT8CONV_BF16>(vec, scaled, d.y_dtype)
      : d.x_dtype == INT8CONV_FP16 ? kernels_for<INT8CONV_FP16>(vec, scaled, d.y_dtype)
      : d.x_dtype == INT8CONV_FP32 ? kernels_for<INT8CONV_FP32>(vec, scaled, d.y_dtype)
                                   : kernels_for<INT8CONV_INT32>(vec, scaled, d.y_dtype);
  const int width = vec ? 8 : 1;
  LaunchPlan plan;
  plan.block = dim3(kThreads);
  plan.grid = dim3(static_cast<unsigned>(d.n * shape.spans));
  if (shape.cluster) {
    // Each thread's share of the span, as far as shared memory reaches.
    const int cols = d.channels / width;
    int64_t need = 0;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
      const int w = cols - col0 < kThreads ? cols - col0 : kThreads;
      const int lanes = kThreads / w;
      need += (shape.span_pixels + lanes - 1) / lanes;
    }
    const uint32_t base = norm_smem(width, xs, d.channels, d.groups, 0).total;
    // Clusters that all find room with one CTA for each SM take more than half
    // an SM's shared memory, so that no two CTAs land on the same one.
    const int32_t clusters[9] = I8C_B200_CLUSTERS;
    const bool alone = d.n <= clusters[shape.spans];
    const uint32_t limit = alone ? kMaxSmem : kHalfSmem;
    const int64_t room =
        base < limit ? (limit - base) / static_cast<uint32_t>(kThreads * width * xs) : 0;
    // Whole batches, of the wide vectors only.
    const int64_t batch = xs == 2 ? 4 : 2;
    a.keep = vec ? static_cast<int32_t>((need < room ? need : room) / batch * batch) : 0;
    plan.func = kernels.cluster;
    plan.smem = norm_smem(width, xs, d.channels, d.groups, a.keep).total;
    if (alone && plan.smem <= kHalfSmem) plan.smem = kHalfSmem + 1024;
    plan.cluster = static_cast<uint32_t>(shape.spans);
    if (!ensure_smem_attr(plan.func, static_cast<int>(plan.smem))) return INT8CONV_CUDA_ERROR;
    plan_args(plan, a);
    return launch_plan(plan, stream);
  }
  plan.func = kernels.stats;
  plan.smem = norm_smem(width, xs, d.channels, d.groups, 0).total;
  if (!ensure_smem_attr(plan.func, static_cast<int>(plan.smem))) return INT8CONV_CUDA_ERROR;
  plan_args(plan, a);
  const int8conv_status st = launch_plan(plan, stream);
  if (st != INT8CONV_OK) return st;
  plan.func = kernels.apply;
  plan.smem = norm_smem(width, xs, d.channels, d.groups, 0).total;
  if (!ensure_smem_attr(plan.func, static_cast<int>(plan.smem))) return INT8CONV_CUDA_ERROR;
  return launch_plan(plan, stream);
}

}  // namespace i8c
