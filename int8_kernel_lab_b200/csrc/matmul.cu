// matmul.cu - int8 matrix products with a floating-point epilogue, plain and
// grouped by expert:
//   y[i,j] = act(acc * row_scale[i] * col_scale[j] + bias[j]) + residual[i,j],
//   acc[i,j] = sum_k a[i,k] * b[j,k]   (int32, exact: k <= 131071)
//
// One persistent kernel, 10 warps, one CTA per SM or CTA pairs
// (tcgen05 cta_group::2, 256-row tiles):
//   warp 0     TMA producer: A and B tiles of 256 bytes of k (two boxes of 128
//              bytes, 128-byte swizzle) into an mbarrier ring.  Rows and columns
//              past the matrices and bytes past k arrive as zeros, so no size
//              has to divide a tile.
//   warp 1     MMA issuer: tcgen05.mma kind::i8, int32 accumulators in TMEM,
//              two buffers, so the epilogue of a tile runs under the next one.
//   Both run as whole warps with one elected lane issuing, so that addresses
//   and descriptors are uniform values, and with 8 MMAs between barriers: with
//   one thread and 4 MMAs the issuer needed 490 cycles for each 128 bytes of k
//   (a commit alone over 200), whatever the tile, against the 512 that the
//   largest tile computes.
//   warps 2-9  epilogue, two warps for each TMEM lane quarter, each taking
//              every other 32 columns: one row per thread, the column scales
//              and biases of the tile in shared memory, the residual read a
//              block ahead, one rounding to the output type, then blocks of 32
//              rows x 64 bytes staged in swizzled shared memory and each
//              written by one TMA store (or, where the pitch or a ragged
//              group's end does not allow one, by row segments of 16 bytes or
//              elements).
// A rows are loaded in boxes of 8 to 128 rows (smaller for few tokens, and for
// experts with few rows): the tile rows that no box covers keep whatever the
// ring held.  They are integers, so they can only reach their own accumulator
// rows, which nothing stores.
//
// Grouped: A rows are sorted by expert and B is [groups][n][k].  Every CTA
// scans the device-side offsets into a table of row tiles in shared memory, and
// its roles walk the same list of (expert, column tile, row tile) units.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <math.h>

#include <mutex>

#include "conv_common.h"
#include "epilogue.cuh"
#include "int8conv_rules.h"
#include "launch.h"
#include "sm100.cuh"

namespace i8c {

namespace {

constexpr int kBlockK = 128;                  // bytes of k of one swizzled box
constexpr int kSub = 2;                       // boxes of each operand in a stage
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kTableBytes = 1024;             // 128 columns x (scale, bias) per warp
constexpr int kMaxStages = 14;

// Forms of the kernel.
constexpr int kPlain = 0;
constexpr int kGrouped = 1;     // rows grouped by expert
constexpr int kResidentB = 2;   // a CTA's column tile of B stays in shared memory

struct MatmulGeom {
  int32_t M, N;
  int32_t kblocks;     // boxes of 128 bytes of k
  int32_t bn;          // tile width (multiple of 32)
  int32_t a_rows;      // rows of A that a stage has room for (8..128)
  int32_t box_rows;    // rows of one A box: a tile loads as many as its rows need
  int32_t n_tiles, m_tiles;
  int32_t band;        // row tiles of one band of the tile order
  int32_t stages;
  int32_t tmem_cols;
  int32_t tma_store;   // 1: whole blocks leave as TMA stores
  int32_t vec_store;   // 1: rows of y are 16-byte aligned
  int32_t vec_res;     // 1: rows of the residual are 16-byte aligned
  int32_t activation;
  int32_t groups;      // 0: plain product
  int32_t splits;      // CTAs that share a tile's k (split kernel)
  float inv_out_scale;
  int64_t ldy, ldr;    // elements
  const float *row_scale, *col_scale, *bias;
  const void *residual;
  void *y;
  const int32_t *offsets;
};

template <int OUT>
__host__ __device__ constexpr int out_bytes() {
  return OUT == INT8CONV_FP32 ? 4 : OUT == INT8CONV_INT8 ? 1 : 2;
}

// Epilogue staging of one warp: a block of 32 rows x 64 bytes (32 bytes for
// int8), which is 32 columns, or 16 of fp32.
constexpr int kStageBytes = 2048;
__host__ __device__ constexpr int block_cols(int out_size) { return out_size == 4 ? 16 : 32; }

// Shared-memory plan, identical on host and device.  A boxes take the rows that
// are loaded; an MMA reads 128 rows from a box's start, the surplus being bytes
// of other boxes (the rings and the staging that follow the last box are longer
// than 16 KB).
struct MatmulSmem {
  uint32_t a_box, b_box;       // bytes of one box, this CTA's share
  uint32_t b_off, staging_off, table_off, bar_off, group_off, total;
};

// `resident`: boxes of B that stay in shared memory for the whole launch, instead
// of B's share of the ring.
__host__ __device__ inline MatmulSmem matmul_smem(int a_rows, int b_rows, int stages, int groups,
                                                  int resident) {
  MatmulSmem p;
  p.a_box = a_rows * kBlockK;
  p.b_box = b_rows * kBlockK;
  p.b_off = stages * kSub * p.a_box;
  // Boxes are multiples of 1024 bytes.
  p.staging_off = p.b_off + (resident > 0 ? resident : stages * kSub) * p.b_box;
  p.table_off = p.staging_off + kEpiWarps * kStageBytes;
  p.bar_off = p.table_off + kEpiWarps * kTableBytes;
  // full/empty[stages], tfull[2], tempty[2], drain, resident B, TMEM slot
  p.group_off = p.bar_off + (2 * stages + 6) * 8 + 8;
  p.total = 1024 + p.group_off + (groups > 0 ? (2 * groups + 2) * 4 : 0);
  return p;
}

struct Tile {
  int m0;      // first row
  int m_end;   // rows at and past this one are not this tile's to store
  int n0;      // first column
  int group;
};

// Work units of a launch.  Plain: bands of `band` row tiles, and inside a band
// column by column, so that the CTAs running at one time share few rows of A
// and of B.  Grouped: expert by expert, column by column.
template <int MODE>
__device__ __forceinline__ Tile tile_at(const MatmulGeom &g, int tile_rows, const int32_t *row_start,
                                        const int32_t *tile_start, int u) {
  Tile t;
  if constexpr (MODE == kResidentB) {
    t.group = 0;
    t.m0 = u / g.n_tiles * tile_rows;
    t.m_end = g.M;
    t.n0 = u % g.n_tiles * g.bn;
  } else if constexpr (MODE == kGrouped) {
    int lo = 0, hi = g.groups;   // tile_start[lo] * n_tiles <= u < tile_start[hi] * n_tiles
    const int at = u / g.n_tiles;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tile_start[mid] <= at) lo = mid;
      else hi = mid;
    }
    const int first = tile_start[lo];
    const int count = tile_start[lo + 1] - first;
    const int local = u - first * g.n_tiles;
    const int n = local / count;
    t.group = lo;
    t.m0 = row_start[lo] + (local - n * count) * tile_rows;
    t.m_end = row_start[lo + 1];
    t.n0 = n * g.bn;
  } else {
    const int per_band = g.band * g.n_tiles;
    const int b = u / per_band;
    const int local = u - b * per_band;
    const int left = g.m_tiles - b * g.band;
    const int height = left < g.band ? left : g.band;
    const int n = local / height;
    t.group = 0;
    t.m0 = (b * g.band + local - n * height) * tile_rows;
    t.m_end = g.M;
    t.n0 = n * g.bn;
  }
  return t;
}

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A wait of the whole warp; the vote makes the outcome uniform.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, const WaitCtx &ctx,
                                          uint32_t bit) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx, bit));
}

template <bool PAIR>
__device__ __forceinline__ void commit_mma(uint64_t *bar) {
  if constexpr (PAIR)
    umma_commit_pair(bar, 0x3);
  else
    umma_commit(bar);
}

// scale, bias and activation of one 32-column block of a thread's row;
// `table`: the block's columns in pairs, (scale, scale, bias, bias).
template <int ACT, int OUT>
__device__ __forceinline__ void finish_block(uint32_t (&v)[32], float rs, const float4 *table) {
  const uint64_t row = f2_pack(rs, rs);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float4 t = table[j];
    const uint64_t x = f2_pack(static_cast<float>(static_cast<int32_t>(v[2 * j])),
                               static_cast<float>(static_cast<int32_t>(v[2 * j + 1])));
    float a, b;
    f2_unpack(f2_fma(f2_mul(x, f2_pack(t.x, t.y)), row, f2_pack(t.z, t.w)), a, b);
    activate2<ACT, OUT == INT8CONV_FP32>(a, b);
    v[2 * j] = __float_as_uint(a);
    v[2 * j + 1] = __float_as_uint(b);
  }
}

// 16-byte chunk `j` of row `row` in a staged block, under the TMA swizzle whose
// span is the block's row (64 or 32 bytes).
template <int OUT>
__device__ __forceinline__ int chunk_at(int row, int j) {
  if constexpr (OUT == INT8CONV_INT8) return row * 2 + (j ^ ((row >> 2) & 1));
  return row * 4 + (j ^ ((row >> 1) & 3));
}

// The residual's 32 columns of one row: loaded a block ahead of their use, since
// a read from memory takes longer than a block's arithmetic (2900 against 800
// cycles, loaded where they were added).
template <int OUT>
struct ResidualBlock {
  using T = typename Elem<OUT>::type;
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  uint4 w[32 / kPer];

  __device__ __forceinline__ void load(const T *r) {
#pragma unroll
    for (int j = 0; j < 32 / kPer; ++j) w[j] = reinterpret_cast<const uint4 *>(r)[j];
  }
  __device__ __forceinline__ void add_to(uint32_t (&v)[32]) const {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      v[j] = __float_as_uint(__uint_as_float(v[j]) +
                             Elem<OUT>::load(reinterpret_cast<const T *>(w)[j]));
  }
};

// Element by element: `cols` of the 32 columns at r.
template <int OUT>
__device__ __forceinline__ void add_residual(uint32_t (&v)[32],
                                             const typename Elem<OUT>::type *r, int cols) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j < cols) v[j] = __float_as_uint(__uint_as_float(v[j]) + Elem<OUT>::load(r[j]));
}

// One block's columns of a thread's 32 values, from column FROM on, rounded,
// into its row of the staged block.
template <int OUT, int FROM>
__device__ __forceinline__ void stage_row(const uint32_t (&v)[32], uint4 *stg, int row,
                                          float inv_out_scale) {
  auto f = [&](int i) { return __uint_as_float(v[i]); };
  if constexpr (OUT == INT8CONV_FP32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = FROM + 4 * j;
      stg[chunk_at<OUT>(row, j)] = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
  } else if constexpr (OUT == INT8CONV_INT8) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = 16 * j + 4 * t;
        w[t] = pack_int8(f(i) * inv_out_scale, f(i + 1) * inv_out_scale, f(i + 2) * inv_out_scale,
                         f(i + 3) * inv_out_scale);
      }
      stg[chunk_at<OUT>(row, j)] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = 8 * j + 2 * t;
        w[t] = OUT == INT8CONV_BF16 ? pack_bf16(f(i), f(i + 1)) : pack_fp16(f(i), f(i + 1));
      }
      stg[chunk_at<OUT>(row, j)] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// The staged block to global memory without TMA: rows [0, rows), columns
// [0, cols) at `y` (the block's first element).
template <int OUT>
__device__ __forceinline__ void copy_out(const uint4 *stg, typename Elem<OUT>::type *y, int64_t ldy,
                                         int rows, int cols, bool vec, int lane) {
  using T = typename Elem<OUT>::type;
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  constexpr int kChunks = block_cols(sizeof(T)) / kPer;   // 16-byte chunks per row
  constexpr int kRows = 32 / kChunks;          // rows per pass of the warp
  if (vec) {
    const int j = lane % kChunks;
    for (int r = lane / kChunks; r < rows; r += kRows) {
      const uint4 raw = stg[chunk_at<OUT>(r, j)];
      T *dst = y + r * ldy + j * kPer;
      if ((j + 1) * kPer <= cols) {
        *reinterpret_cast<uint4 *>(dst) = raw;
      } else {
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int t = 0; t < kPer; ++t)
          if (j * kPer + t < cols) dst[t] = e[t];
      }
    }
  } else if (lane < cols) {
    // Element by element, a row segment per instruction; eight rows are read
    // before the first is written.
    const T *e = reinterpret_cast<const T *>(stg);
    T *dst = y + lane;
    for (int r0 = 0; r0 < rows; r0 += 8) {
      T t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        t[u] = e[chunk_at<OUT>(r0 + u, lane / kPer) * kPer + lane % kPer];
#pragma unroll
      for (int u = 0; u < 8; ++u, dst += ldy)
        if (r0 + u < rows) *dst = t[u];
    }
  }
}

template <bool PAIR, int MODE, int OUT>
__global__ void __launch_bounds__(kThreads, 1)
    matmul_kernel(const __grid_constant__ CUtensorMap tmap_a,
                  const __grid_constant__ CUtensorMap tmap_b,
                  const __grid_constant__ CUtensorMap tmap_y, const MatmulGeom g,
                  const RunCtl ctl) {
  extern __shared__ uint8_t smem_raw[];
  // 1024-byte alignment for the 128-byte swizzle; the same offset in both CTAs
  // of a pair.
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr bool GROUPED = MODE == kGrouped, RESIDENT = MODE == kResidentB;
  static_assert(!(PAIR && RESIDENT), "resident B runs single CTAs");
  constexpr int kTileRows = PAIR ? 2 * kBlockM : kBlockM;
  const MatmulSmem plan = matmul_smem(g.a_rows, PAIR ? g.bn / 2 : g.bn, g.stages,
                                      GROUPED ? g.groups : 0, RESIDENT ? g.kblocks : 0);
  uint8_t *a_ring = smem;
  uint8_t *b_ring = smem + plan.b_off;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + plan.bar_off);
  uint64_t *empty = full + g.stages;
  uint64_t *tfull = empty + g.stages;
  uint64_t *tempty = tfull + 2;
  uint64_t *drain = tempty + 2;
  uint64_t *b_here = drain + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(b_here + 1);
  int32_t *row_start = reinterpret_cast<int32_t *>(smem + plan.group_off);
  int32_t *tile_start = row_start + g.groups + 1;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0);   // uniform
  const int lane = threadIdx.x & 31;
  const WaitCtx wctx{ctl.wait_ns, ctl.status};
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int first = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int step = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

  if (warp == 0) {
    for (int i = lane; i < 2 * g.stages + 6; i += 32) {
      // tempty: one arrival per epilogue warp (of both CTAs for a pair).
      const bool te = i >= 2 * g.stages + 2 && i < 2 * g.stages + 4;
      mbar_init(&full[i], te ? (PAIR ? 2 : 1) * kEpiWarps : 1);
    }
    fence_mbar_init();
    if (lane == 0) {
      tma_prefetch_desc(&tmap_a);
      tma_prefetch_desc(&tmap_b);
    }
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, g.tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, g.tmem_cols);
      tmem_relinquish();
    }
  }
  int num_tiles = g.m_tiles * g.n_tiles;
  if constexpr (GROUPED) {
    // Nothing is read before the previous kernel in the stream is complete.
    griddep_wait();
    for (int i = threadIdx.x; i <= g.groups; i += kThreads) {
      const int32_t o = __ldg(g.offsets + i);
      row_start[i] = o < 0 ? 0 : (o > g.M ? g.M : o);
    }
    __syncthreads();
    if (warp == 0) {
      // Running maximum of the offsets, then running count of row tiles.
      int32_t top = 0, tiles = 0;
      if (lane == 0) tile_start[0] = 0;
      for (int base = 0; base <= g.groups; base += 32) {
        const int i = base + lane;
        int32_t end = i <= g.groups ? row_start[i] : 0;
        end = end > top ? end : top;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int32_t o = __shfl_up_sync(0xffffffffu, end, d);
          if (lane >= d && o > end) end = o;
        }
        int32_t begin = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) begin = base == 0 ? end : top;   // entry 0 opens no group
        int32_t count = i <= g.groups ? (end - begin + kTileRows - 1) / kTileRows : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int32_t o = __shfl_up_sync(0xffffffffu, count, d);
          if (lane >= d) count += o;
        }
        if (i <= g.groups) {
          row_start[i] = end;
          tile_start[i] = tiles + count;
        }
        top = __shfl_sync(0xffffffffu, end, 31);
        tiles += __shfl_sync(0xffffffffu, count, 31);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();   // both CTAs' barriers are set up
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if constexpr (GROUPED) num_tiles = tile_start[g.groups] * g.n_tiles;
  // Nothing touches global memory, and no wait's limit starts to count, before
  // the previous kernel in the stream is complete.
  if constexpr (!GROUPED) griddep_wait();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    int stage = 0;
    uint32_t phase = 0;
    int armed = 0;
    const uint32_t box_bytes = static_cast<uint32_t>(g.box_rows * kBlockK);
    if constexpr (RESIDENT) {
      if (!ctl.starve) {
        const int n0 = first % g.n_tiles * g.bn;
        if (elect_one()) {
          mbar_arrive_expect_tx(b_here, g.kblocks * plan.b_box);
          for (int kb = 0; kb < g.kblocks; ++kb)
            tma_load_3d(b_ring + kb * plan.b_box, &tmap_b, b_here, kb * kBlockK, n0, 0);
        }
        __syncwarp();
      }
    }
    bool ok = true;
    for (int u = first; u < num_tiles && ok; u += step) {
      const Tile t = tile_at<MODE>(g, kTileRows, row_start, tile_start, u);
      const int m0 = t.m0 + static_cast<int>(rank) * kBlockM;
      const int n0 = t.n0 + static_cast<int>(rank) * (PAIR ? g.bn / 2 : 0);
      // A plain product's boxes cover the tile; a group's as many as its rows need.
      int parts = 1;
      if (GROUPED && !PAIR && g.box_rows < g.a_rows) {
        const int rows = t.m_end - m0 < g.a_rows ? t.m_end - m0 : g.a_rows;
        parts = __shfl_sync(0xffffffffu, (rows + g.box_rows - 1) / g.box_rows, 0);
      }
      // Bytes of 128 bytes of k.
      const uint32_t tx = (PAIR ? 2u : 1u) * (parts * box_bytes + (RESIDENT ? 0 : plan.b_box));
      for (int kb = 0; kb < g.kblocks; kb += kSub) {
        if (!warp_wait(&empty[stage], phase ^ 1u, wctx, kStatusTimeoutEmpty)) {
          ok = false;
          break;
        }
        if (!ctl.starve) {
          const int boxes = g.kblocks - kb < kSub ? g.kblocks - kb : kSub;
          if (elect_one()) {
            // A pair credits both CTAs' bytes to the leader's barrier.
            if (leader) mbar_arrive_expect_tx(&full[stage], boxes * tx);
            uint8_t *adst = a_ring + stage * (kSub * plan.a_box);
            uint8_t *bdst = b_ring + stage * (kSub * plan.b_box);
#pragma unroll
            for (int i = 0; i < kSub; ++i) {
              if (i < boxes) {
                if constexpr (PAIR) {
                  const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
                  tma_load_3d_pair(adst + i * plan.a_box, &tmap_a, bar, (kb + i) * kBlockK, m0, 0);
                  tma_load_3d_pair(bdst + i * plan.b_box, &tmap_b, bar, (kb + i) * kBlockK, n0,
                                   t.group);
                } else {
                  for (int j = 0; j < parts; ++j)
                    tma_load_3d(adst + i * plan.a_box + j * box_bytes, &tmap_a, &full[stage],
                                (kb + i) * kBlockK, m0 + j * g.box_rows, 0);
                  if constexpr (!RESIDENT)
                    tma_load_3d(bdst + i * plan.b_box, &tmap_b, &full[stage], (kb + i) * kBlockK,
                                n0, t.group);
                }
              }
            }
          }
          __syncwarp();
          if (leader && armed < g.stages) ++armed;
        }
        if (++stage == g.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // Copies still in flight land before the CTA exits: wait for the fills
    // armed last (the leader's barriers count both CTAs' copies).
    for (int i = 0; i < armed; ++i) {
      if (--stage < 0) {
        stage = g.stages - 1;
        phase ^= 1u;
      }
      warp_wait(&full[stage], phase, wctx, kStatusTimeoutTeardown);
    }
    if (RESIDENT && !ctl.starve) warp_wait(b_here, 0, wctx, kStatusTimeoutTeardown);
  } else if (warp == 1) {
    if (leader) {
      // ---------------- MMA issuer (the leader of a pair) ----------------
      const uint32_t idesc = idesc_s8(kTileRows, g.bn);
      const uint64_t a_desc0 = smem_desc(smem_u32(a_ring), 16, 8 * kBlockK, Layout::kSw128);
      const uint64_t b_desc0 = smem_desc(smem_u32(b_ring), 16, 8 * kBlockK, Layout::kSw128);
      const uint32_t a_step = plan.a_box >> 4;   // descriptor units, one box on
      const uint32_t b_step = plan.b_box >> 4;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      if constexpr (RESIDENT) ok = warp_wait(b_here, 0, wctx, kStatusTimeoutFull);
      for (int u = first; u < num_tiles && ok; u += step) {
        if (!warp_wait(&tempty[acc], acc_phase ^ 1u, wctx, kStatusTimeoutDrain)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * g.bn);
        for (int kb = 0; kb < g.kblocks; kb += kSub) {
          if (!warp_wait(&full[stage], phase, wctx, kStatusTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int boxes = g.kblocks - kb < kSub ? g.kblocks - kb : kSub;
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kSub; ++i) {
              if (i < boxes) {
                const uint64_t ad = a_desc0 + (stage * kSub + i) * a_step;
                const uint64_t bd = b_desc0 + (RESIDENT ? kb + i : stage * kSub + i) * b_step;
#pragma unroll
                for (int k = 0; k < kBlockK / 32; ++k) {
                  const uint32_t accumulate = kb + i + k > 0 ? 1u : 0u;
                  if constexpr (PAIR)
                    umma_i8_pair(d_tmem, ad + 2 * k, bd + 2 * k, idesc, accumulate);
                  else
                    umma_i8(d_tmem, ad + 2 * k, bd + 2 * k, idesc, accumulate);
                }
              }
            }
            commit_mma<PAIR>(&empty[stage]);
            if (kb + kSub >= g.kblocks) commit_mma<PAIR>(&tfull[acc]);
          }
          __syncwarp();
          if (++stage == g.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      // Every MMA issued must finish before TMEM is released (in both CTAs).
      // A commit covers the MMAs of the thread that issues it: the lane elected
      // from the whole warp is always the same one.
      if (elect_one()) commit_mma<PAIR>(drain);
      __syncwarp();
      warp_wait(drain, 0, wctx, kStatusTimeoutTeardown);
    } else if constexpr (PAIR) {
      warp_wait(drain, 0, wctx, kStatusTimeoutTeardown);
    }
  } else {
    // ---------------- epilogue (warps 2..9) ----------------
    using T = typename Elem<OUT>::type;
    if (warp == 2) griddep_launch_dependents();
    const int quarter = warp & 3;           // TMEM lane quarter this warp may access
    const int half = (warp - 2) >> 2;       // 32-column blocks half, half + 2, ...
    constexpr int kCols = block_cols(out_bytes<OUT>());
    uint8_t *staging = smem + plan.staging_off + (warp - 2) * kStageBytes;
    float *table = reinterpret_cast<float *>(smem + plan.table_off + (warp - 2) * kTableBytes);
    // The leader's tempty barriers, 8 bytes apart (a pair signals them remotely).
    const uint32_t tempty_at = PAIR ? mapa_shared(smem_u32(tempty), 0) : smem_u32(tempty);
    T *y = static_cast<T *>(g.y);
    const T *residual = static_cast<const T *>(g.residual);
    int acc = 0;
    uint32_t acc_phase = 0;
    int table_n0 = -1, table_group = -1;
    for (int u = first; u < num_tiles; u += step) {
      const Tile t = tile_at<MODE>(g, kTileRows, row_start, tile_start, u);
      const int row0 = t.m0 + static_cast<int>(rank) * kBlockM + quarter * 32;
      const int rows = t.m_end - row0;        // rows of this warp's 32 that count (may be <= 0)
      const bool mine = lane < rows;
      if (t.n0 != table_n0 || t.group != table_group) {
        __syncwarp();
        const int64_t at = static_cast<int64_t>(t.group) * g.N;
        for (int b = 0, c0 = 32 * half; c0 < g.bn; ++b, c0 += 64) {
          const int c = t.n0 + c0 + lane;
          float scale = 0.f, bias = 0.f;
          if (c < g.N) {
            scale = g.col_scale != nullptr ? __ldg(g.col_scale + at + c) : 1.f;
            bias = g.bias != nullptr ? __ldg(g.bias + at + c) : 0.f;
          }
          float *pair = table + (b * 16 + (lane >> 1)) * 4 + (lane & 1);
          pair[0] = scale;
          pair[2] = bias;
        }
        __syncwarp();
        table_n0 = t.n0;
        table_group = t.group;
      }
      float rs = 1.f;
      if (g.row_scale != nullptr) rs = mine ? __ldg(g.row_scale + row0 + lane) : 0.f;
      // This row of the residual, and its block that the loop adds next.
      constexpr bool kResidual = !GROUPED && OUT != INT8CONV_INT8;
      using Block = ResidualBlock<kResidual ? OUT : INT8CONV_BF16>;
      Block ahead;
      const T *res = nullptr;
      if constexpr (kResidual) {
        if (residual != nullptr && mine) {
          res = residual + static_cast<int64_t>(row0 + lane) * g.ldr + t.n0;
          if (g.vec_res && 32 * half < g.bn && t.n0 + 32 * half + 32 <= g.N)
            ahead.load(res + 32 * half);
        }
      }
      // All lanes wait; the vote keeps the warp converged for tcgen05.ld even
      // if the wait runs out on some lanes only.
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, wctx, kStatusTimeoutAccum)))
        break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(acc * g.bn);
      bool released = false;
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR)
            mbar_arrive_cluster(tempty_at + 8u * static_cast<uint32_t>(acc));
          else
            mbar_arrive(&tempty[acc]);
        }
        released = true;
      };
      if (rows > 0) {
        for (int i = 0, c0 = 32 * half; c0 < g.bn; ++i, c0 += 64) {
          const int col0 = t.n0 + c0;
          const int cols = g.N - col0;
          if (cols <= 0) break;
          Block now;
          if constexpr (kResidual) {
            now = ahead;
            if (res != nullptr && g.vec_res && c0 + 64 < g.bn && cols >= 96) ahead.load(res + c0 + 64);
          }
          uint32_t v[32];
          tmem_ld_32x32b_x32(taddr + c0, v);
          tmem_ld_wait();
          if (c0 + 64 >= g.bn || cols <= 64) release();   // this warp's last read of the tile
          const float4 *tb = reinterpret_cast<const float4 *>(table) + i * 16;
          switch (g.activation) {
            case INT8CONV_ACT_RELU:
              finish_block<INT8CONV_ACT_RELU, OUT>(v, rs, tb);
              break;
            case INT8CONV_ACT_GELU:
              finish_block<INT8CONV_ACT_GELU, OUT>(v, rs, tb);
              break;
            case INT8CONV_ACT_GELU_TANH:
              finish_block<INT8CONV_ACT_GELU_TANH, OUT>(v, rs, tb);
              break;
            case INT8CONV_ACT_SILU:
              finish_block<INT8CONV_ACT_SILU, OUT>(v, rs, tb);
              break;
            default:
              finish_block<INT8CONV_ACT_NONE, OUT>(v, rs, tb);
          }
          if constexpr (kResidual) {
            if (res != nullptr) {
              if (g.vec_res && cols >= 32)
                now.add_to(v);
              else
                add_residual<OUT>(v, res + c0, cols);
            }
          }
          uint4 *stg = reinterpret_cast<uint4 *>(staging);
          const bool tma = g.tma_store != 0 && (!GROUPED || rows >= 32);
          auto put = [&](auto from) {
            constexpr int kFrom = decltype(from)::value;
            if (kFrom >= cols) return;
            // The store that last read the buffer has finished reading it.
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
            stage_row<OUT, kFrom>(v, stg, lane, g.inv_out_scale);
            if (tma) fence_proxy_async_smem();
            __syncwarp();
            if (tma) {
              if (lane == 0) {
                tma_store_2d(&tmap_y, stg, col0 + kFrom, row0);
                bulk_commit_group();
              }
            } else {
              const int wide = cols - kFrom < kCols ? cols - kFrom : kCols;
              copy_out<OUT>(stg, y + static_cast<int64_t>(row0) * g.ldy + col0 + kFrom, g.ldy,
                            rows < 32 ? rows : 32, wide, g.vec_store != 0, lane);
            }
            __syncwarp();
          };
          put(std::integral_constant<int, 0>());
          if constexpr (kCols == 16) put(std::integral_constant<int, 16>());
        }
      }
      if (!released) release();   // no row or column of this tile for this warp
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    // Stores still reading shared memory finish before the CTA exits.
    if (lane == 0) bulk_wait_group_read_all();
  }

  tc_fence_before();
  __syncthreads();
  // Neither CTA of a pair leaves while the other may still touch its shared
  // memory (remote barrier arrivals, MMA operand reads).
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, g.tmem_cols);
    else
      tmem_dealloc(tmem_base, g.tmem_cols);
  }
}

__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}

template <int OUT>
__device__ __forceinline__ float activate_any(float v, int activation) {
  switch (activation) {
    case INT8CONV_ACT_RELU:
      return activate<INT8CONV_ACT_RELU, OUT == INT8CONV_FP32>(v);
    case INT8CONV_ACT_GELU:
      return activate<INT8CONV_ACT_GELU, OUT == INT8CONV_FP32>(v);
    case INT8CONV_ACT_GELU_TANH:
      return activate<INT8CONV_ACT_GELU_TANH, OUT == INT8CONV_FP32>(v);
    case INT8CONV_ACT_SILU:
      return activate<INT8CONV_ACT_SILU, OUT == INT8CONV_FP32>(v);
    default:
      return v;
  }
}

// Few rows: one tile per cluster of g.splits CTAs, each taking a share of k.
//
// With few tiles a narrow one on every SM was bound by the tensor core, which
// reads 128 rows of A for each instruction however few columns it multiplies
// (16 x 4096 x 4096 in 128 tiles of 32 columns: 128 instructions of 60 cycles a
// CTA).  Shares of k keep the tiles wide: the same bytes of B for each SM, a
// quarter of the instructions.  The int32 partial sums of the tile's rows meet
// in distributed shared memory (the operand ring's, which is free by then); CTA
// r adds, finishes and stores the r-th share of the columns, four columns a thread.
// Integer sums are exact, so the split changes no result.
template <int OUT>
__global__ void __launch_bounds__(kThreads, 1)
    matmul_split_kernel(const __grid_constant__ CUtensorMap tmap_a,
                        const __grid_constant__ CUtensorMap tmap_b, const MatmulGeom g,
                        const RunCtl ctl) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const MatmulSmem plan = matmul_smem(g.a_rows, g.bn, g.stages, 0, 0);
  uint8_t *a_ring = smem;
  uint8_t *b_ring = smem + plan.b_off;
  int32_t *partial = reinterpret_cast<int32_t *>(smem);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + plan.bar_off);
  uint64_t *empty = full + g.stages;
  uint64_t *tfull = empty + g.stages;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tfull + 6);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0);   // uniform
  const int lane = threadIdx.x & 31;
  const WaitCtx wctx{ctl.wait_ns, ctl.status};
  const int rank = static_cast<int>(blockIdx.x) % g.splits;
  const int tile = static_cast<int>(blockIdx.x) / g.splits;
  const int n0 = tile % g.n_tiles * g.bn;
  const int m0 = tile / g.n_tiles * kBlockM;
  const int rows = g.M - m0 < kBlockM ? g.M - m0 : kBlockM;
  // Shares of k in whole stages; the last ones may be shorter, or empty.
  const int share = (g.kblocks + g.splits * kSub - 1) / (g.splits * kSub) * kSub;
  const int kb_begin = rank * share < g.kblocks ? rank * share : g.kblocks;
  const int kb_end = kb_begin + share < g.kblocks ? kb_begin + share : g.kblocks;
  const int pitch = g.bn + 4;   // words; 16-byte stores of neighbouring rows meet no bank twice

  if (warp == 0) {
    for (int i = lane; i < 2 * g.stages + 1; i += 32) mbar_init(&full[i], 1);
    fence_mbar_init();
    if (lane == 0) {
      tma_prefetch_desc(&tmap_a);
      tma_prefetch_desc(&tmap_b);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, g.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  // Nothing touches global memory, and no wait's limit starts to count, before
  // the previous kernel in the stream is complete.
  griddep_wait();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    int stage = 0, armed = 0;
    uint32_t phase = 0;
    for (int kb = kb_begin; kb < kb_end; kb += kSub) {
      if (!warp_wait(&empty[stage], phase ^ 1u, wctx, kStatusTimeoutEmpty)) break;
      if (!ctl.starve) {
        const int boxes = kb_end - kb < kSub ? kb_end - kb : kSub;
        if (elect_one()) {
          mbar_arrive_expect_tx(&full[stage], boxes * (plan.a_box + plan.b_box));
          uint8_t *adst = a_ring + stage * (kSub * plan.a_box);
          uint8_t *bdst = b_ring + stage * (kSub * plan.b_box);
#pragma unroll
          for (int i = 0; i < kSub; ++i) {
            if (i < boxes) {
              tma_load_3d(bdst + i * plan.b_box, &tmap_b, &full[stage], (kb + i) * kBlockK, n0, 0);
              tma_load_3d(adst + i * plan.a_box, &tmap_a, &full[stage], (kb + i) * kBlockK, m0, 0);
            }
          }
        }
        __syncwarp();
        if (armed < g.stages) ++armed;
      }
      if (++stage == g.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Copies still in flight land before the ring is reused.
    for (int i = 0; i < armed; ++i) {
      if (--stage < 0) {
        stage = g.stages - 1;
        phase ^= 1u;
      }
      warp_wait(&full[stage], phase, wctx, kStatusTimeoutTeardown);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const uint32_t idesc = idesc_s8(kBlockM, g.bn);
    const uint64_t a_desc0 = smem_desc(smem_u32(a_ring), 16, 8 * kBlockK, Layout::kSw128);
    const uint64_t b_desc0 = smem_desc(smem_u32(b_ring), 16, 8 * kBlockK, Layout::kSw128);
    const uint32_t a_step = plan.a_box >> 4;
    const uint32_t b_step = plan.b_box >> 4;
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb_begin; kb < kb_end; kb += kSub) {
      if (!warp_wait(&full[stage], phase, wctx, kStatusTimeoutFull)) break;
      tc_fence_after();
      const int boxes = kb_end - kb < kSub ? kb_end - kb : kSub;
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
          if (i < boxes) {
            const uint64_t ad = a_desc0 + (stage * kSub + i) * a_step;
            const uint64_t bd = b_desc0 + (stage * kSub + i) * b_step;
#pragma unroll
            for (int k = 0; k < kBlockK / 32; ++k)
              umma_i8(tmem_base, ad + 2 * k, bd + 2 * k, idesc, kb - kb_begin + i + k > 0 ? 1u : 0u);
          }
        }
        umma_commit(&empty[stage]);
      }
      __syncwarp();
      if (++stage == g.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Also after a wait that ran out: every MMA issued finishes before the ring
    // is reused and TMEM is released.
    if (elect_one()) umma_commit(tfull);
    __syncwarp();
    warp_wait(tfull, 0, wctx, kStatusTimeoutTeardown);
  } else {
    // ---------------- partial sums to shared memory (warps 2..9) ----------------
    if (warp == 2) griddep_launch_dependents();
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    if (warp_wait(tfull, 0, wctx, kStatusTimeoutAccum) && quarter * 32 < rows && kb_begin < kb_end) {
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      for (int c0 = 32 * half; c0 < g.bn; c0 += 64) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(taddr + c0, v);
        tmem_ld_wait();
        if (quarter * 32 + lane < rows) {
          int4 *dst = reinterpret_cast<int4 *>(partial + (quarter * 32 + lane) * pitch + c0);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            dst[j] = make_int4(static_cast<int32_t>(v[4 * j]), static_cast<int32_t>(v[4 * j + 1]),
                               static_cast<int32_t>(v[4 * j + 2]), static_cast<int32_t>(v[4 * j + 3]));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp >= 2) {
    using T = typename Elem<OUT>::type;
    const int wide = g.bn / g.splits / 4;                   // this CTA's columns, in fours
    const int parts = (g.kblocks + share - 1) / share;      // CTAs that hold a partial sum
    const uint32_t here = smem_u32(partial);
    for (int i = static_cast<int>(threadIdx.x) - 64; i < rows * wide; i += kThreads - 64) {
      const int r = i / wide, c = (rank * wide + i - r * wide) * 4;
      const int row = m0 + r, col = n0 + c;
      if (col >= g.N) continue;
      const uint32_t at = here + (r * pitch + c) * 4;
      int4 part[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        part[k] = k < parts ? ld_cluster_v4(mapa_shared(at, k)) : make_int4(0, 0, 0, 0);
      float cs[4], b[4], res[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = col + j < g.N;
        cs[j] = in && g.col_scale != nullptr ? __ldg(g.col_scale + col + j) : 1.f;
        b[j] = in && g.bias != nullptr ? __ldg(g.bias + col + j) : 0.f;
        res[j] = 0.f;
        if constexpr (OUT != INT8CONV_INT8) {
          if (in && g.residual != nullptr)
            res[j] = Elem<OUT>::load(static_cast<const T *>(g.residual)[row * g.ldr + col + j]);
        }
      }
      const float rs = g.row_scale != nullptr ? __ldg(g.row_scale + row) : 1.f;
      int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sum.x += part[k].x;
        sum.y += part[k].y;
        sum.z += part[k].z;
        sum.w += part[k].w;
      }
      const int32_t acc[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v = activate_any<OUT>(fmaf(static_cast<float>(acc[j]) * cs[j], rs, b[j]), g.activation);
        v = OUT == INT8CONV_INT8 ? v * g.inv_out_scale : v + res[j];
        if (col + j < g.N) static_cast<T *>(g.y)[row * g.ldy + col + j] = Elem<OUT>::store(v);
      }
    }
  }
  // No CTA leaves while another may still read its partial sums.
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, g.tmem_cols);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// Tile choice of one launch.
struct TileChoice {
  bool pair;
  int bn;
  int splits;
  bool resident;
};

// The candidate with the least estimated time, in cycles.  For each 128 bytes
// of k a CTA's tensor core needs 2 * bn (128 x bn x 32 bytes in bn / 2; a pair
// 256 x bn in the same), its loads (a_rows rows of A and its share of B, 128
// bytes each) come at about 72 bytes a cycle, and the issuer needs 285; the
// slowest counts.  The epilogue of the tile before runs meanwhile, 5 cycles a
// column and 400 for its latencies (those of a plain epilogue: gelu_tanh to int8
// takes some 8000 for 256 columns, so with a costly activation and k of 2048 and
// less it is the epilogue that counts, which this does not see).  A pair loses
// about 2500 cycles between two tiles and 3000 at the start.  The rates were
// fitted to plain and grouped shapes timed at every width, single, in pairs and
// with resident B, 25 without an activation, two with gelu and one with gelu_tanh:
// the choice is within 5 % of the fastest on each, within 1 % on most (2048 x 4096
// x 4096: pairs of 256 columns 27.7 us, best of 15 27.7, worst 69; 32768 x 320 x
// 320: resident, 160 columns, 11.0 us, not resident 11.9, worst 21.6).  Few tiles may
// also share k (the split kernel): 1 x 4096 x 4096 in 4 shares of 128 columns
// 5.9 us, unsplit 7.0; 8 x 4096 x 16384 10.3 and 20.5; 128 x 4096 x 4096 9.4 and
// 7.4 (unsplit taken).
TileChoice choose_tile(double row_tiles128, double row_tiles256, int64_t n, int kblocks, int a_rows,
                       int sms, int rows, bool grouped) {
  TileChoice best{false, 128, 1, false};
  double best_cost = 1e300;
  auto consider = [&](bool pair, int bn) {
    const double tiles = (pair ? row_tiles256 : row_tiles128) * static_cast<double>((n + bn - 1) / bn);
    const double waves = ceil(tiles / (pair ? sms / 2 : sms) - 1e-9);
    const double mma = 2.0 * bn;
    const double load = (a_rows + (pair ? bn / 2 : bn)) * (kBlockK / 72.0);
    const double box = fmax(fmax(mma, load), 285.0);
    const double finish = 400.0 + 5.0 * bn;
    const double cost = waves * (fmax(kblocks * box, finish) + (pair ? 2500.0 : 100.0)) + finish +
                        (pair ? 3000.0 : 0.0);
    if (cost < best_cost) {
      best_cost = cost;
      best = TileChoice{pair, bn, 1, false};
    }
  };
  if (a_rows == kBlockM && pairing_mode() != 1) {
    for (int bn = 256; bn >= 64; bn -= 32) consider(true, bn);
    if (pairing_mode() == 2) return best;
  }
  for (int bn = 256; bn >= 32; bn -= 32) consider(false, bn);
  if (!grouped && pairing_mode() == 0 && a_rows == kBlockM) {
    // A column tile of B that stays: only A is loaded for each row tile.
    for (int bn = 256; bn >= 32; bn -= 32) {
      const int64_t n_tiles = (n + bn - 1) / bn;
      if (n_tiles > sms ||
          matmul_smem(kBlockM, bn, 3, 0, kblocks).total > static_cast<uint32_t>(kMaxSmem))
        continue;
      const double waves = ceil(row_tiles128 / static_cast<double>(sms / n_tiles) - 1e-9);
      const double box = fmax(fmax(2.0 * bn, kBlockM * (kBlockK / 72.0)), 285.0);
      const double finish = 400.0 + 5.0 * bn;
      const double cost = waves * (fmax(kblocks * box, finish) + 100.0) + finish +
                          kblocks * bn * (kBlockK / 72.0);
      if (waves > 1.0 && cost < best_cost) {
        best_cost = cost;
        best = TileChoice{false, bn, 1, true};
      }
    }
  }
  if (!grouped && pairing_mode() == 0) {
    // Shares of k, where all clusters run at one time.
    const int32_t clusters[9] = I8C_B200_CLUSTERS;
    for (int splits = 2; splits <= 8; splits *= 2) {
      for (int bn = 256; bn >= 64; bn -= 64) {
        if (row_tiles128 * static_cast<double>((n + bn - 1) / bn) > clusters[splits]) continue;
        const int share = (kblocks + 2 * splits - 1) / (2 * splits) * 2;
        const double box = fmax(fmax(2.0 * bn, (a_rows + bn) * (kBlockK / 72.0)), 285.0);
        // Cluster launch and barriers, more of them for 8 CTAs, and the sums:
        // 16 bytes from each of the CTAs for 1024 values at a time.
        const double cost = share * box + (splits == 8 ? 4500.0 : 2500.0) +
                            1200.0 * ceil(rows * bn / (1024.0 * splits));
        if (cost < best_cost) {
          best_cost = cost;
          best = TileChoice{false, bn, splits, false};
        }
      }
    }
  }
  return best;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void *p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// int8 operand [outer][rows][k]: boxes of 128 bytes of k x `box_rows` rows.
bool operand_map(CUtensorMap *map, const int8_t *p, int64_t k, int64_t rows, int64_t ld,
                 int64_t outer, int64_t outer_stride, int box_rows) {
  const auto encode = encode_tiled();
  if (encode == nullptr) return false;
  cuuint64_t dims[3] = {(cuuint64_t)k, (cuuint64_t)rows, (cuuint64_t)outer};
  cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)outer_stride};
  cuuint32_t box[3] = {kBlockK, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t *>(p), dims, strides, box,
                estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Output [M][N], boxes of one staged block, swizzled over the box's row.
bool result_map(CUtensorMap *map, void *y, int dtype, int64_t m, int64_t n, int64_t ldy) {
  const auto encode = encode_tiled();
  if (encode == nullptr) return false;
  const int size = dtype_bytes(dtype);
  cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)m};
  cuuint64_t strides[1] = {(cuuint64_t)ldy * size};
  cuuint32_t box[2] = {(cuuint32_t)block_cols(size), 32};
  cuuint32_t estr[2] = {1, 1};
  // Elements are moved, not computed with: unsigned types of the same size.
  const CUtensorMapDataType type = size == 4   ? CU_TENSOR_MAP_DATA_TYPE_UINT32
                                   : size == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                               : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUtensorMapSwizzle swizzle =
      size == 1 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_64B;
  return encode(map, type, 2, y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_NONE,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool PAIR, int MODE>
const void *kernel_for(int dtype) {
  switch (dtype) {
    case INT8CONV_BF16:
      return reinterpret_cast<const void *>(&matmul_kernel<PAIR, MODE, INT8CONV_BF16>);
    case INT8CONV_FP16:
      return reinterpret_cast<const void *>(&matmul_kernel<PAIR, MODE, INT8CONV_FP16>);
    case INT8CONV_FP32:
      return reinterpret_cast<const void *>(&matmul_kernel<PAIR, MODE, INT8CONV_FP32>);
    default:
      return reinterpret_cast<const void *>(&matmul_kernel<PAIR, MODE, INT8CONV_INT8>);
  }
}

const void *split_kernel_for(int dtype) {
  switch (dtype) {
    case INT8CONV_BF16:
      return reinterpret_cast<const void *>(&matmul_split_kernel<INT8CONV_BF16>);
    case INT8CONV_FP16:
      return reinterpret_cast<const void *>(&matmul_split_kernel<INT8CONV_FP16>);
    case INT8CONV_FP32:
      return reinterpret_cast<const void *>(&matmul_split_kernel<INT8CONV_FP32>);
    default:
      return reinterpret_cast<const void *>(&matmul_split_kernel<INT8CONV_INT8>);
  }
}

bool aligned(const void *p, int64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes)) == 0;
}

// The tiles of one launch on a device of `sms` SMs.
struct MatmulTiles {
  int a_rows, box_rows;
  TileChoice choice;
};

MatmulTiles choose_tiles(int64_t m, int64_t n, int64_t k, int32_t groups, int sms) {
  const bool grouped = groups > 0;
  MatmulTiles t;
  t.a_rows = 8;
  while (t.a_rows < kBlockM && t.a_rows < m) t.a_rows *= 2;
  // Row tiles: exact for a plain product; grouped, those of experts that share
  // the rows about evenly (the host does not know the offsets): half a tile of
  // each is empty.
  const auto row_tiles = [&](int64_t rows) -> double {
    if (!grouped) return static_cast<double>((m + rows - 1) / rows);
    const int64_t active = groups < m ? groups : m;
    const double each = static_cast<double>(m) / active;
    return active * fmax(1.0, each / rows + 0.5);
  };
  // Experts with few rows each: boxes of about that many rows.
  t.box_rows = t.a_rows;
  if (grouped) {
    const int64_t each = (m + groups - 1) / groups;
    while (t.box_rows > 8 && t.box_rows > each) t.box_rows /= 2;
  }
  t.choice = choose_tile(row_tiles(kBlockM), row_tiles(2 * kBlockM), n,
                         static_cast<int>((k + kBlockK - 1) / kBlockK), t.box_rows, sms,
                         static_cast<int>(m < kBlockM ? m : kBlockM), grouped);
  return t;
}

}  // namespace

int32_t matmul_form(int64_t m, int64_t n, int64_t k, int32_t groups, int sms) {
  const TileChoice c = choose_tiles(m, n, k, groups, sms).choice;
  return c.bn | (c.pair ? 1 << 16 : 0) | (c.resident ? 1 << 17 : 0) | c.splits << 20;
}

int8conv_status launch_matmul_impl(const int8conv_matmul &d, const int8_t *a, const int8_t *b,
                                   int64_t group_stride, const int32_t *offsets, int32_t groups,
                                   void *y, cudaStream_t stream) {
  const bool grouped = groups > 0;
  const int sms = device_info().sm_count;
  const int size = dtype_bytes(d.y_dtype);
  MatmulGeom g{};
  g.M = static_cast<int32_t>(d.m);
  g.N = static_cast<int32_t>(d.n);
  g.kblocks = static_cast<int32_t>((d.k + kBlockK - 1) / kBlockK);
  const MatmulTiles tiles_of = choose_tiles(d.m, d.n, d.k, groups, sms);
  g.a_rows = tiles_of.a_rows;
  g.box_rows = tiles_of.box_rows;
  const TileChoice c = tiles_of.choice;
  g.bn = c.bn;
  const int tile_rows = c.pair ? 2 * kBlockM : kBlockM;
  g.n_tiles = static_cast<int32_t>((d.n + g.bn - 1) / g.bn);
  // At most this many row tiles: a group adds at most one partly filled tile.
  const int64_t m_tiles =
      grouped ? d.m / tile_rows + (groups < d.m ? groups : d.m) : (d.m + tile_rows - 1) / tile_rows;
  if (m_tiles * g.n_tiles >= (int64_t(1) << 30)) return INT8CONV_BAD_ARGUMENT;
  g.m_tiles = static_cast<int32_t>(m_tiles);
  g.band = 8;
  g.tmem_cols = 32;
  while (g.tmem_cols < 2 * g.bn) g.tmem_cols *= 2;
  const int b_rows = c.pair ? g.bn / 2 : g.bn;
  const auto smem_of = [&](int stages) {
    return matmul_smem(g.a_rows, b_rows, stages, groups, c.resident ? g.kblocks : 0).total;
  };
  g.stages = kMaxStages;
  while (g.stages > 2 && smem_of(g.stages) > static_cast<uint32_t>(kMaxSmem)) --g.stages;
  g.vec_store = (d.ldy * size) % 16 == 0 && aligned(y, 16);
  // A TMA store clips the last column in units of 16 bytes, so a row that ends
  // inside one (in a wider pitch) is stored without it.
  g.tma_store = g.vec_store && (d.n * size) % 16 == 0;
  g.vec_res = d.residual != nullptr && (d.ldr * size) % 16 == 0 && aligned(d.residual, 16);
  g.activation = d.activation;
  g.groups = groups;
  g.inv_out_scale = d.y_dtype == INT8CONV_INT8 ? 1.0f / d.out_scale : 1.0f;
  g.ldy = d.ldy;
  g.ldr = d.ldr;
  g.row_scale = d.row_scale;
  g.col_scale = d.col_scale;
  g.bias = d.bias;
  g.residual = d.residual;
  g.y = y;
  g.offsets = offsets;

  CUtensorMap tmap_a, tmap_b, tmap_y{};
  if (!operand_map(&tmap_a, a, d.k, d.m, d.lda, 1, d.lda, g.box_rows) ||
      !operand_map(&tmap_b, b, d.k, d.n, d.ldb, grouped ? groups : 1,
                   groups > 1 ? group_stride : d.ldb, b_rows))
    return INT8CONV_CUDA_ERROR;
  if (g.tma_store && !result_map(&tmap_y, y, d.y_dtype, d.m, d.n, d.ldy)) return INT8CONV_CUDA_ERROR;

  LaunchPlan plan;
  if (c.splits > 1) {
    g.splits = c.splits;
    g.tmem_cols = 32;
    while (g.tmem_cols < g.bn) g.tmem_cols *= 2;
    plan.func = split_kernel_for(d.y_dtype);
    // The partial sums take the place of the ring, with which the largest tile
    // of them (128 rows x 256 columns, 130 KB) always fits.
    const MatmulSmem layout = matmul_smem(g.a_rows, g.bn, g.stages, 0, 0);
    const uint32_t sums = static_cast<uint32_t>(g.M < kBlockM ? g.M : kBlockM) * (g.bn + 4) * 4;
    if (sums > layout.bar_off) return INT8CONV_CUDA_ERROR;
    plan.smem = layout.total;
    if (plan.smem < kMaxSmem / 2 + 1024) plan.smem = kMaxSmem / 2 + 1024;
    if (!ensure_smem_attr(plan.func, static_cast<int>(plan.smem))) return INT8CONV_CUDA_ERROR;
    plan.cluster = static_cast<uint32_t>(c.splits);
    plan.grid = dim3(static_cast<unsigned>(g.m_tiles * g.n_tiles * c.splits));
    plan.block = dim3(kThreads);
    plan_args(plan, tmap_a, tmap_b, g, run_ctl());
    return launch_plan(plan, stream);
  }
  plan.func = c.pair      ? (grouped ? kernel_for<true, kGrouped>(d.y_dtype)
                                     : kernel_for<true, kPlain>(d.y_dtype))
              : grouped    ? kernel_for<false, kGrouped>(d.y_dtype)
              : c.resident ? kernel_for<false, kResidentB>(d.y_dtype)
                           : kernel_for<false, kPlain>(d.y_dtype);
  plan.smem = smem_of(g.stages);
  // At least half an SM's shared memory: one CTA per SM, so that none waits
  // for another's TMEM columns.
  const uint32_t floor_bytes = kMaxSmem / 2 + 1024;
  if (plan.smem < floor_bytes) plan.smem = floor_bytes;
  if (!ensure_smem_attr(plan.func, static_cast<int>(plan.smem))) return INT8CONV_CUDA_ERROR;
  plan.cluster = c.pair ? 2 : 1;
  const int64_t tiles = m_tiles * g.n_tiles;
  const int64_t slots = c.pair ? sms / 2 : c.resident ? sms / g.n_tiles * g.n_tiles : sms;
  plan.grid = dim3(static_cast<unsigned>((tiles < slots ? tiles : slots) * plan.cluster));
  plan.block = dim3(kThreads);
  plan_args(plan, tmap_a, tmap_b, tmap_y, g, run_ctl());
  return launch_plan(plan, stream);
}

}  // namespace i8c
