// Products of e4m3 operands with an fp32 scale per group of 128 along the summed dimension, and the kernels that bring operands into that format.
//
//   fp8_rows      x [T, K] -> e4m3 [T, K], scales [ceil(K / 128), T]
//   fp8_both      the same, and the transpose e4m3 [K, T] in groups of 128 rows of x, scales [ceil(T / 128), K], from one read of x
//   fp8_squares   w [N, K] -> e4m3 [N, K] and its transpose [K, N], one scale per 128 x 128 block
//   fp8_matmul    C[m, n] = sum_g sa[m, g] sb[n, g] sum_{k in g} a[m, k] b[n, k]
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <torch/extension.h>

#include "fp8_format.cuh"
#include "once.h"
#include "ptx.cuh"
#include "tensor_map.h"

namespace cg = cooperative_groups;

namespace ob200 {
namespace {

using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------------------
// Into the format.  Bound by HBM: one read of x, one byte written per value and operand.  bf16, 16384 x 8192: rows 72 us (5.6 TB/s), both
// layouts 96 us (5.6 TB/s); fp32 8192 x 2048 into squares and their transpose 23 us (4.5 TB/s).
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, magnitude_bits(v[k]));
  return top;
}

// Largest of each of kCount values over sixteen lanes, a value per lane at the end: lane l holds that of number l * kCount / 16.  One division
// per lane then serves all groups.
template <int kCount>
__device__ __forceinline__ uint32_t spread_max(uint32_t (&v)[kCount], int lane) {
  int o = 8;
#pragma unroll
  for (int n = kCount; n > 1; n >>= 1, o >>= 1) {
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const bool high = lane & o;
      const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? v[i] : v[i + n / 2], o);
      v[i] = max(high ? v[i + n / 2] : v[i], got);
    }
  }
#pragma unroll
  for (; o > 0; o >>= 1) v[0] = max(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
  return v[0];
}

// Eight rows of eight neighbouring values as a thread of the tile kernel holds them.  bf16 stays packed: half the registers, and
// magnitudes are compared two at a time as 16-bit integers.
template <typename T>
struct Patch {
  float v[8][8];
  template <bool kVec>
  __device__ __forceinline__ void load(int r, const float* row, int col, int cols) { load8<kVec>(row, col, cols, v[r]); }
  __device__ __forceinline__ void clear(int r) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[r][k] = 0.f;
  }
  __device__ __forceinline__ float at(int r, int k) const { return v[r][k]; }
  __device__ __forceinline__ uint32_t row_top(int r) const { return top_of(v[r]); }
  __device__ __forceinline__ void column_tops(uint32_t (&down)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t t = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) t = max(t, magnitude_bits(v[r][k]));
      down[k] = max(t, __shfl_xor_sync(0xffffffffu, t, 16));
    }
  }
};

template <>
struct Patch<bf16> {
  uint32_t w[8][4];
  template <bool kVec>
  __device__ __forceinline__ void load(int r, const bf16* row, int col, int cols) {
    if constexpr (kVec) {
      const uint4 u = col < cols ? *reinterpret_cast<const uint4*>(row + col) : make_uint4(0u, 0u, 0u, 0u);
      w[r][0] = u.x; w[r][1] = u.y; w[r][2] = u.z; w[r][3] = u.w;
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = col + 2 * k < cols ? h[col + 2 * k] : 0u, hi = col + 2 * k + 1 < cols ? h[col + 2 * k + 1] : 0u;
        w[r][k] = lo | (hi << 16);
      }
    }
  }
  __device__ __forceinline__ void clear(int r) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[r][k] = 0;
  }
  __device__ __forceinline__ float at(int r, int k) const { return __uint_as_float((k & 1) ? w[r][k >> 1] & 0xffff0000u : w[r][k >> 1] << 16); }
  __device__ __forceinline__ uint32_t magnitudes(int r, int k) const { return w[r][k] & 0x7fff7fffu; }
  __device__ __forceinline__ uint32_t row_top(int r) const {
    const uint32_t t = __vimax3_u16x2(__vimax3_u16x2(magnitudes(r, 0), magnitudes(r, 1), magnitudes(r, 2)), magnitudes(r, 3), 0u);
    return max(t << 16, t & 0xffff0000u);
  }
  __device__ __forceinline__ void column_tops(uint32_t (&down)[8]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t t = magnitudes(0, k);
#pragma unroll
      for (int r = 1; r < 7; r += 2) t = __vimax3_u16x2(t, magnitudes(r, k), magnitudes(r + 1, k));
      t = __vimax3_u16x2(t, magnitudes(7, k), 0u);
      t = __vimax3_u16x2(t, __shfl_xor_sync(0xffffffffu, t, 16), 0u);
      down[2 * k] = t << 16;
      down[2 * k + 1] = t & 0xffff0000u;
    }
  }
};

template <typename T>
__device__ __forceinline__ uint2 row_bytes(const Patch<T>& x, int r, float f) {
  const float v[8] = {x.at(r, 0), x.at(r, 1), x.at(r, 2), x.at(r, 3), x.at(r, 4), x.at(r, 5), x.at(r, 6), x.at(r, 7)};
  return e4m3x8(v, f);
}

enum TileFormat { kRowGroups, kBothGroups, kSquareGroups };

// A CTA takes a 128 x 128 tile: thread (ty, tx) holds rows 8 ty .. 8 ty + 7 and columns 8 tx .. 8 tx + 7.  The transpose goes through
// shared memory, where a thread has eight neighbouring bytes of each of its columns; piece p of row c lies at p ^ (c / 8), so that the
// threads of a row of tiles write to different banks.
constexpr int kTileThreads = 256;

template <typename T, bool kVec, TileFormat kFormat>
__global__ void __launch_bounds__(kTileThreads, sizeof(T) == 2 ? 3 : 2)
fp8_tile_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, float* __restrict__ scale, uint8_t* __restrict__ qt,
                long long ldt, float* __restrict__ scale_t, long long rows, int K) {
  __shared__ __align__(16) uint32_t col_top[kTileThreads / 32][kFp8Group];
  __shared__ __align__(16) float col_factor[kFp8Group];
  __shared__ __align__(16) uint8_t flipped[kFp8Group * kFp8Group];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, warp = threadIdx.x >> 5;
  const int kb = blockIdx.x;
  const long long tb = blockIdx.y;
  const int col = kb * kFp8Group + tx * 8;
  const long long row0 = tb * kFp8Group + ty * 8;
  Patch<T> v;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if (row0 + r < rows) v.template load<kVec>(r, x + (row0 + r) * ldx, col, K);
    else v.clear(r);
  }
  uint32_t tops[8];  // of a thread's rows
#pragma unroll
  for (int r = 0; r < 8; ++r) tops[r] = v.row_top(r);
  float factor_t[8];
  if constexpr (kFormat == kSquareGroups) {
    uint32_t t = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) t = max(t, tops[r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
    if ((threadIdx.x & 31) == 0) col_top[0][warp] = t;
    __syncthreads();
    t = 0;
#pragma unroll
    for (int w = 0; w < kTileThreads / 32; ++w) t = max(t, col_top[0][w]);
    const GroupScale s = group_scale(t);
#pragma unroll
    for (int k = 0; k < 8; ++k) factor_t[k] = s.factor;
    if (threadIdx.x == 0) scale[tb * gridDim.x + kb] = s.scale;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (row0 + r < rows && col < K) *reinterpret_cast<uint2*>(q + (row0 + r) * ldq + col) = row_bytes(v, r, s.factor);
    if (qt == nullptr) return;
  } else {
    if constexpr (kFormat == kBothGroups) {
      uint32_t down[8];  // of a thread's columns, with the other eight rows of the warp
      v.column_tops(down);
      if ((threadIdx.x & 16) == 0) {
        *reinterpret_cast<uint4*>(&col_top[warp][tx * 8]) = make_uint4(down[0], down[1], down[2], down[3]);
        *reinterpret_cast<uint4*>(&col_top[warp][tx * 8 + 4]) = make_uint4(down[4], down[5], down[6], down[7]);
      }
    }
    const GroupScale mine = group_scale(spread_max(tops, tx));  // of row tx / 2
    if ((tx & 1) == 0 && row0 + tx / 2 < rows) scale[static_cast<long long>(kb) * rows + row0 + tx / 2] = mine.scale;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float factor = __shfl_sync(0xffffffffu, mine.factor, (threadIdx.x & 16) + 2 * r);
      if (row0 + r < rows && col < K) *reinterpret_cast<uint2*>(q + (row0 + r) * ldq + col) = row_bytes(v, r, factor);
    }
    if constexpr (kFormat == kRowGroups) return;
    __syncthreads();
    if (threadIdx.x < kFp8Group) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < kTileThreads / 32; ++w) t = max(t, col_top[w][threadIdx.x]);
      const GroupScale s = group_scale(t);
      col_factor[threadIdx.x] = s.factor;
      if (kb * kFp8Group + threadIdx.x < K) scale_t[tb * K + kb * kFp8Group + threadIdx.x] = s.scale;
    }
    __syncthreads();
    const float4 f0 = *reinterpret_cast<const float4*>(&col_factor[tx * 8]), f1 = *reinterpret_cast<const float4*>(&col_factor[tx * 8 + 4]);
    factor_t[0] = f0.x; factor_t[1] = f0.y; factor_t[2] = f0.z; factor_t[3] = f0.w;
    factor_t[4] = f1.x; factor_t[5] = f1.y; factor_t[6] = f1.z; factor_t[7] = f1.w;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float c[8] = {v.at(0, k), v.at(1, k), v.at(2, k), v.at(3, k), v.at(4, k), v.at(5, k), v.at(6, k), v.at(7, k)};
    *reinterpret_cast<uint2*>(flipped + (tx * 8 + k) * kFp8Group + (ty ^ tx) * 8) = e4m3x8(c, factor_t[k]);
  }
  __syncthreads();
  // Row c of the transpose: 128 bytes, of which those beyond the pitch do not exist (the pitch is a multiple of 16).
  for (int i = threadIdx.x; i < kFp8Group * 8; i += kTileThreads) {
    const int c = i >> 3, part = i & 7, turn = c >> 3;
    if (kb * kFp8Group + c < K && tb * kFp8Group + part * 16 < ldt) {
      const uint4 u = *reinterpret_cast<const uint4*>(flipped + c * kFp8Group + ((2 * part ^ turn) & ~1) * 8);
      *reinterpret_cast<uint4*>(qt + static_cast<long long>(kb * kFp8Group + c) * ldt + tb * kFp8Group + part * 16) =
          (turn & 1) ? make_uint4(u.z, u.w, u.x, u.y) : u;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// The product.  A tile of 128 x kN results goes over K in steps of one group of 128: TMA brings 128 x 128 bytes of A and kN x 128 of B,
// four tcgen05.mma sum the group into a TMEM buffer of its own, and eight epilogue warps read the buffer, apply the two scales
// of the group and add it to sums that stay in fp32 registers, while the MMAs of the next groups fill the other buffers.
//
// A thread of an epilogue warp holds one row where B has a scale per 128 rows: one multiply-add per value with the product of both
// scales.  With a scale per row of B (a column of the tile) it holds every fourth column of four rows: two operations per value, but a
// quarter of the scales to fetch from shared memory.  TMEM gives whole rows at 244 bytes per clock and 32 lanes, the latter
// arrangement at 124 (column pairs of eight rows would come at 64); the fp32 units take one operation per clock.  So the epilogue needs about
// 256 or 512 clocks per group of a 128 x 256 tile, next to 512 of the MMAs.  The next piece of a buffer is on its way while one is added.
//
// Large products are computed by pairs of CTAs, 256 x 256 results each.  With 128 x 256 per CTA a group moves 48 KB into shared memory and
// 48 KB from there to the tensor cores, 768 clocks of 128 bytes for 512 of MMAs; a pair moves 32 and 32 KB per SM.
//
// What bounds it: the epilogue, about 950 clocks per group, of which 256 are multiply-adds (two warps per scheduler that run in step) and the
// rest TMEM loads, barriers and their latencies; with a scale per row of B about 1550.  16384 x 2048 x 8192 by pairs: 160 us without
// an epilogue, 184 without the multiply-adds, 238 as it is (2.31 PFLOP/s; 1.62 for the bf16 library product); 8192 x 16384 x 2048 with a
// scale per row of B 389 us (1.41 PFLOP/s), 242 without the multiply-adds.  Sixteen epilogue warps with half the columns each spill
// (429 us); reading TMEM as column pairs of eight rows took 305 us, single CTAs of 128 x 256 265 us.
//
// Products with few tiles are cut along K among the CTAs of a cluster, whose partial sums meet in distributed shared memory: each CTA adds
// the sums of all ranks, in rank order, for its share of the tile.
// ------------------------------------------------------------------------------------------------
constexpr int kTileM = 128;
constexpr int kEpilogueWarps = 8;
constexpr int kFirstEpilogueWarp = 4;
constexpr int kProductThreads = 384;  // warps 0 TMA, 1 and 2 MMA, one idle; 4 .. 11 epilogue
constexpr int kMaxSplits = 8;

template <int kN, bool kPair, bool kColumnScale, typename Out>
struct ProductCfg {
  static constexpr int kRowsB = kPair ? kN / 2 : kN;  // that this CTA loads
  static constexpr int kStageBytes = (kTileM + kRowsB) * kFp8Group;
  static constexpr int kBuffers = kN == 256 ? 2 : 4;  // TMEM buffers of kN columns
  static constexpr int kOwn = kN / 2;                 // columns of one epilogue warp: two warps share a 32-row stripe
  // Whole rows in bf16 leave through shared memory and TMA, 64 columns at a time.
  static constexpr bool kStaged = sizeof(Out) == 2 && !kColumnScale && kN >= 128;
  static constexpr int kStagingBytes = kStaged ? kEpilogueWarps * 32 * kOwn * 2 : 0;
  static constexpr int kStages = kN == 64 ? 8 : kStaged ? 4 : 6;
  static constexpr int kScaleSlots = 4;  // groups whose scales are on their way
  static constexpr int kScaleFloats = kTileM + (kColumnScale ? kN : 32);             // of one group: rows of A, columns or blocks of B
  static constexpr int kBarrierBytes = 320;
  // 1 KB to align the stages
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kStagingBytes + kScaleSlots * kScaleFloats * 4 + kBarrierBytes;
  // Registers: 128 sums per epilogue thread do not fit into an even split of 168, so the first warpgroup gives up some of its own.
  static constexpr bool kUneven = kN == 256;
  static constexpr int kLaunchRegs = 168, kEpilogueRegs = 232, kOtherRegs = 40;
  static_assert(256 * kEpilogueRegs + 128 * kOtherRegs <= kProductThreads * kLaunchRegs, "the shares must fit into the registers at launch");
  static_assert(kN == 256 || kTileM * kN * 4 <= kStages * kStageBytes, "partial sums take the place of the stages");
  static_assert(kSmemBytes <= 227 * 1024, "shared memory of a CTA");
};

struct ProductArgs {
  const float *sa, *sb;
  long long sa_row, sa_group, sb_row, sb_group;  // strides of the scales; kColumnScale false: sb_row counts blocks of 128 rows of B
  void* c;
  const float* addend;  // fp32, C's layout, or null
  long long ldc;
  int M, N, groups, tiles_m, tiles, splits;
  bool staged;  // results leave by TMA
  int* status;
};

// Four neighbouring results of one row, from a column that is a multiple of four.
template <typename Out>
__device__ __forceinline__ void store_quad(const ProductArgs& p, int row, int col, float4 v) {
  if (row >= p.M || col >= p.N) return;
  const long long at = row * p.ldc + col;
  float x[4] = {v.x, v.y, v.z, v.w};
  if (p.addend != nullptr) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < p.N) x[k] += p.addend[at + k];
  }
  Out* dst = static_cast<Out*>(p.c) + at;
  if ((p.ldc & 3) == 0) {  // whole quads, 16 or 8 bytes apart
    if constexpr (sizeof(Out) == 4) {
      *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      uint2 u;
      *reinterpret_cast<__nv_bfloat162*>(&u.x) = __floats2bfloat162_rn(x[0], x[1]);
      *reinterpret_cast<__nv_bfloat162*>(&u.y) = __floats2bfloat162_rn(x[2], x[3]);
      *reinterpret_cast<uint2*>(dst) = u;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (col + k >= p.N) continue;
    if constexpr (sizeof(Out) == 4) dst[k] = x[k];
    else dst[k] = __float2bfloat16_rn(x[k]);
  }
}

template <int kN, bool kPair, bool kColumnScale, typename Out>
__global__ void __launch_bounds__(kProductThreads, 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c,
                  const __grid_constant__ ProductArgs p) {
  using C = ProductCfg<kN, kPair, kColumnScale, Out>;
  constexpr int kStages = C::kStages, kBuffers = C::kBuffers, kOwn = C::kOwn;
  constexpr uint32_t kIdesc = make_idesc(/*e4m3*/ 0, kPair ? 2 * kTileM : kTileM, kN);
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + kStages * C::kStageBytes;
  float* scales = reinterpret_cast<float*>(staging + C::kStagingBytes);  // [slot][kScaleFloats]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + C::kScaleSlots * C::kScaleFloats);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + kBuffers;
  uint64_t* scale_full = acc_empty + kBuffers;
  uint64_t* scale_empty = scale_full + C::kScaleSlots;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(scale_empty + C::kScaleSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert(2 * (kStages + kBuffers + C::kScaleSlots) * 8 + 8 <= C::kBarrierBytes, "barrier region");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBuffers; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kPair ? 2 * kEpilogueWarps : kEpilogueWarps);
    }
    for (int i = 0; i < C::kScaleSlots; ++i) {
      mbar_init(&scale_full[i], 32);
      mbar_init(&scale_empty[i], kEpilogueWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(tmem_holder, kN * kBuffers);
    } else {
      tmem_alloc(tmem_holder, kN * kBuffers);
      tmem_relinquish();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) cg::this_cluster().sync();  // the other CTA's barriers exist
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  const int member = kPair ? static_cast<int>(blockIdx.x) & 1 : 0;  // of the pair

  const int rank = kPair || p.splits == 1 ? 0 : static_cast<int>(blockIdx.x) % p.splits;
  const int per_tile = kPair ? 2 : p.splits;  // CTAs
  const int first_tile = static_cast<int>(blockIdx.x) / per_tile, tile_step = static_cast<int>(gridDim.x) / per_tile;
  const int g0 = static_cast<int>(static_cast<long long>(p.groups) * rank / p.splits);
  const int g1 = static_cast<int>(static_cast<long long>(p.groups) * (rank + 1) / p.splits);
  // Neighbouring tiles share operands: eight rows of tiles at a time, down the rows first.
  const int tiles_n = p.tiles / p.tiles_m;
  auto place = [&](int t, int& m0, int& n0) {
    const int band = t / (8 * tiles_n), in = t - band * 8 * tiles_n;
    const int high = min(8, p.tiles_m - band * 8);
    m0 = (band * 8 + in % high) * (kPair ? 2 * kTileM : kTileM) + member * kTileM;
    n0 = in / high * kN;
  };

  if (warp < kFirstEpilogueWarp) {
    if constexpr (C::kUneven) setmaxnreg_dec<C::kOtherRegs>();
    // The whole warp walks the loops and one lane gives the commands: values that all lanes share stay in uniform registers, where
    // the commands need them.  (With the loops inside one lane's branch the MMAs of a group took 660 clocks to issue, more than to run.)
    if (warp == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first_tile; t < p.tiles && ok; t += tile_step) {
        int m0, n0;
        place(t, m0, n0);
        for (int g = g0; g < g1; ++g) {
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, abort_flag));
          if (!ok) break;
          if (elect_one()) {
            uint8_t* s = smem + stage * C::kStageBytes;
            if constexpr (kPair) {  // both CTAs' loads are counted by the barrier of the first
              if (member == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::kStageBytes);
              const uint32_t bar = cluster_addr(&full[stage], 0);
              tma_load_2d_pair(s, &map_a, bar, g * kFp8Group, m0);
              tma_load_2d_pair(s + kTileM * kFp8Group, &map_b, bar, g * kFp8Group, n0 + member * C::kRowsB);
            } else {
              mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
              tma_load_2d(s, &map_a, &full[stage], g * kFp8Group, m0);
              tma_load_2d(s + kTileM * kFp8Group, &map_b, &full[stage], g * kFp8Group, n0);
            }
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    } else if (warp <= 2 && member == 0) {
      // Two warps take the groups in turn: one waits for its operands and its buffer while the MMAs of the other run.  (A warp that has
      // given commands is held until they start, so that with one warp its waits for the next group, some 300 clocks, lay between
      // the MMAs: the products of 16384 x 2048 x 8192 took 3 us longer.)
      static_assert(kStages % 2 == 0 && kBuffers % 2 == 0, "each warp has its own stages and buffers");
      const long long mine = first_tile < p.tiles ? static_cast<long long>((p.tiles - 1 - first_tile) / tile_step + 1) * (g1 - g0) : 0;
      int stage = warp - 1, buf = warp - 1;
      uint32_t phase = 0, round = 0;
      const uint64_t first_a = make_kmajor_sw128_desc(smem_u32(smem)), first_b = make_kmajor_sw128_desc(smem_u32(smem) + kTileM * kFp8Group);
      for (long long i = warp - 1; i < mine; i += 2) {
        const bool ok = mbar_wait(&full[stage], phase, abort_flag) && mbar_wait(&acc_empty[buf], round ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t a = first_a + stage * (C::kStageBytes >> 4), b = first_b + stage * (C::kStageBytes >> 4);
#pragma unroll
          for (int k = 0; k < kFp8Group / 32; ++k) {
            if constexpr (kPair) umma_f8_pair(tmem + buf * kN, a + 2 * k, b + 2 * k, kIdesc, k != 0);
            else umma_f8(tmem + buf * kN, a + 2 * k, b + 2 * k, kIdesc, k != 0);
          }
          if constexpr (kPair) {
            umma_commit_pair(&empty[stage]);
            umma_commit_pair(&acc_full[buf]);
          } else {
            umma_commit(&empty[stage]);
            umma_commit(&acc_full[buf]);
          }
        }
        __syncwarp();
        if ((stage += 2) >= kStages) {
          stage -= kStages;
          phase ^= 1;
        }
        if ((buf += 2) >= kBuffers) {
          buf -= kBuffers;
          round ^= 1;
        }
      }
    } else if (warp == 3) {
      // Scales: the epilogue would wait for the latency of their loads, some 800 clocks, once per group.
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first_tile; t < p.tiles && ok; t += tile_step) {
        int m0, n0;
        place(t, m0, n0);
        for (int g = g0; g < g1; ++g) {
          ok = __all_sync(0xffffffffu, mbar_wait(&scale_empty[slot], phase ^ 1, abort_flag));
          if (!ok) break;
          float* s = scales + slot * C::kScaleFloats;
#pragma unroll
          for (int i = lane; i < kTileM; i += 32) cp_async4(s + i, p.sa + min(m0 + i, p.M - 1) * p.sa_row + g * p.sa_group);
          if constexpr (kColumnScale) {
#pragma unroll
            for (int i = lane; i < kN; i += 32) cp_async4(s + kTileM + i, p.sb + min(n0 + i, p.N - 1) * p.sb_row + g * p.sb_group);
          } else if (lane < 2) {  // of the two halves of the tile's columns
            cp_async4(s + kTileM + lane, p.sb + min(n0 + lane * kOwn, p.N - 1) / kFp8Group * p.sb_row + g * p.sb_group);
          }
          cp_async_arrive(&scale_full[slot]);
          if (++slot == C::kScaleSlots) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
    }
    if (warp == 0 && *abort_flag) {  // a pipeline that gave up leaves with no load of its own still on its way
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
    __syncwarp();
    if (!kPair && p.splits > 1) {
      cg::this_cluster().sync();
      cg::this_cluster().sync();
    }
  } else {
    if constexpr (C::kUneven) setmaxnreg_inc<C::kEpilogueRegs>();
    constexpr int kRowsOwn = kColumnScale ? 4 : 1;  // rows of a thread
    const int stripe = warp & 3, half = (warp - kFirstEpilogueWarp) >> 2;
    const int q = lane & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(stripe * 32) << 16) + half * kOwn;
    uint8_t* my_staging = staging + (warp - kFirstEpilogueWarp) * 32 * kOwn * 2;
    const uint32_t own_rank = kPair ? member : rank;  // in the cluster
    const uint32_t back_to_mma = cluster_addr(acc_empty, kPair ? 0 : own_rank), back_to_loads = cluster_addr(scale_empty, own_rank);
    int buf = 0, slot = 0;
    uint32_t round = 0, turn = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles; t += tile_step) {
      int row0, col0;
      place(t, row0, col0);
      const int row_in = stripe * 32 + (kColumnScale ? lane >> 2 : lane);  // of the tile: rows row_in + 8 i
      row0 += row_in;
      col0 += half * kOwn;
      // Sums, in pairs.  Whole rows: two neighbouring columns.  Else sums[h * kOwn / 4 + i] for the rows row0 + 16 h and row0 + 16 h + 8 and the
      // column 4 i + q.
      uint64_t sums[kOwn / 2];
#pragma unroll
      for (int i = 0; i < kOwn / 2; ++i) sums[i] = 0;
      // Of the group that is being added: its scales and, in v, pieces of its sums.  The first piece of the next group is already on its way
      // when the last one of this group is added.  (A wait that gave up lets everything run through; the flag is looked at below.)
      constexpr int kPiece = kColumnScale || kN == 256 ? 32 : 16;                // columns
      constexpr int kPieces = kColumnScale ? 2 * kOwn / kPiece : kOwn / kPiece;  // upper and lower 16 rows apart where B has a scale per row
      constexpr int kQuarter = kPiece / 4;
      static_assert(kPieces % 2 == 0, "the first piece of a group goes where the last one is not");
      uint32_t v[2][kColumnScale ? kPiece / 2 : kPiece];
      float scale[kRowsOwn], s[kColumnScale ? kQuarter : 1];
      const float* of_columns = nullptr;
      auto issue = [&](int c) {
        const uint32_t from = lanes + buf * kN;
        if constexpr (kColumnScale) tmem_ld_16_issue(from + (static_cast<uint32_t>((c & 1) * 16) << 16) + (c >> 1) * kPiece, v[c & 1]);
        else tmem_ld_32_issue(from + c * kPiece, v[c & 1]);
      };
      float next[kRowsOwn];
      bool scales_there = false, sums_there = false;  // of the next group, as seen while this one is added
      auto begin = [&]() {                            // of a group
        if (!scales_there) mbar_wait(&scale_full[slot], turn, abort_flag);
        const float* of_rows = scales + slot * C::kScaleFloats;
#pragma unroll
        for (int i = 0; i < kRowsOwn; ++i) next[i] = of_rows[row_in + 8 * i];
        if constexpr (!kColumnScale) next[0] *= of_rows[kTileM + half];
        of_columns = of_rows + kTileM + half * kOwn;
        if (!sums_there) mbar_wait(&acc_full[buf], round, abort_flag);
        tc_fence_after_sync();
        issue(0);
      };
      auto look = [&](bool at_sums) {
        const bool last_buf = buf + 1 == kBuffers, last_slot = slot + 1 == C::kScaleSlots;
        if (at_sums) sums_there = mbar_test(&acc_full[last_buf ? 0 : buf + 1], last_buf ? round ^ 1 : round);
        else scales_there = mbar_test(&scale_full[last_slot ? 0 : slot + 1], last_slot ? turn ^ 1 : turn);
      };
      auto finish = [&]() {  // the buffer goes back to the MMAs, the scales' slot to their loads
        tc_fence_before_sync();
        mbar_arrive_at(back_to_mma + buf * 8, lane == 0);
        mbar_arrive_at(back_to_loads + slot * 8, lane == 0);
        if (++buf == kBuffers) {
          buf = 0;
          round ^= 1;
        }
        if (++slot == C::kScaleSlots) {
          slot = 0;
          turn ^= 1;
        }
      };
      if (g0 < g1) begin();
      for (int g = g0; g < g1; ++g) {
#pragma unroll
        for (int i = 0; i < kRowsOwn; ++i) scale[i] = next[i];
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          if constexpr (kColumnScale) {
            if ((c & 1) == 0) {
#pragma unroll
              for (int i = 0; i < kQuarter; ++i) s[i] = of_columns[(c >> 1) * kPiece + 4 * i + q];
            }
          }
          uint64_t by = kColumnScale ? pack2(scale[kColumnScale ? 2 * (c & 1) : 0], scale[kColumnScale ? 2 * (c & 1) + 1 : 0]) : pack2(scale[0], scale[0]);
          tmem_ld_wait(by);
          if (c + 1 < kPieces) {
            issue(c + 1);
            if (c == 0) look(false);
            if (c + 2 == kPieces) look(true);
          } else {
            finish();
            if (g + 1 < g1) begin();
          }
          if constexpr (!kColumnScale) {
#pragma unroll
            for (int j = 0; j < kPiece / 2; ++j) {
              uint64_t& sum = sums[c * kPiece / 2 + j];
              sum = fma2_loaded(v[c & 1][2 * j], v[c & 1][2 * j + 1], by, sum);
            }
          } else {
#pragma unroll
            for (int i = 0; i < kQuarter; ++i) {
              uint64_t& sum = sums[(c & 1) * (kOwn / 4) + (c >> 1) * kQuarter + i];
              sum = fma2(mul2_loaded(v[c & 1][2 * i], v[c & 1][2 * i + 1], by), pack2(s[i], s[i]), sum);
            }
          }
        }
      }
      ok = *abort_flag == 0;
      float acc[kOwn];  // the same, row by row: [column] or [row0 + 8 i][column of this lane]
#pragma unroll
      for (int j = 0; j < kOwn / 2; ++j) {
        float2 x = unpack2(sums[j]);
        if (!ok) x = make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));  // a pipeline that gave up leaves no plausible numbers
        const int at = kColumnScale ? j / (kOwn / 4) * (kOwn / 2) + j % (kOwn / 4) : 2 * j;
        acc[at] = x.x;
        acc[at + (kColumnScale ? kOwn / 4 : 1)] = x.y;
      }
      if constexpr (kColumnScale) {
        // Four lanes have every fourth column of a row: each takes four neighbours of sixteen.
#pragma unroll
        for (int i = 0; i < kOwn; i += 4) {
          float* w = acc + i;
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, (q & 1) ? w[k] : w[k + 1], 1);
            if (q & 1) w[k] = got;
            else w[k + 1] = got;
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float got = __shfl_xor_sync(0xffffffffu, (q & 2) ? w[k] : w[k + 2], 2);
            if (q & 2) w[k] = got;
            else w[k + 2] = got;
          }
        }
      }
      // Quad j: four neighbouring columns of a row.
      auto place_quad = [&](int j, int& row, int& col) {
        row = kColumnScale ? row0 + 8 * (j / (kOwn / 16)) : row0;
        col = kColumnScale ? col0 + 16 * (j % (kOwn / 16)) + 4 * q : col0 + 4 * j;
      };
      if (!kPair && p.splits > 1) {
        // The stages are idle, every load has arrived and every MMA is done, unless this CTA gave up a wait: then a load that is still on its way may
        // write over these sums, and the flag says so in their place.  [quad][thread]
        float4* mine = reinterpret_cast<float4*>(smem);
        const int thread = threadIdx.x - 32 * kFirstEpilogueWarp;
#pragma unroll
        for (int j = 0; j < kOwn / 4; ++j) mine[j * 32 * kEpilogueWarps + thread] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();  // behind the last wait of every warp
        ok = __all_sync(0xffffffffu, *cluster.map_shared_rank(const_cast<int*>(abort_flag), min(lane, p.splits - 1)) == 0);
        for (int j = kOwn / 4 * rank / p.splits; j < kOwn / 4 * (rank + 1) / p.splits; ++j) {
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int r = 0; r < p.splits; ++r) {
            const float4 u = cluster.map_shared_rank(mine, r)[j * 32 * kEpilogueWarps + thread];
            sum.x += u.x; sum.y += u.y; sum.z += u.z; sum.w += u.w;
          }
          if (!ok) sum.x = sum.y = sum.z = sum.w = __int_as_float(0x7fffffff);
          int row, col;
          place_quad(j, row, col);
          store_quad<Out>(p, row, col, sum);
        }
        __syncwarp();
        cluster.sync();  // nobody leaves while its sums are read
        continue;
      }
      if (C::kStaged && p.addend == nullptr) {
        // 32 rows x 64 columns are 128 bytes a row, swizzled as TMA reads them: conflict-free, and the store itself runs beside the next tile.
        if (lane == 0) bulk_wait_read();  // of the tile before
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kOwn / 64; ++c) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __nv_bfloat162 v = __floats2bfloat162_rn(acc[c * 64 + j * 8 + 2 * k], acc[c * 64 + j * 8 + 2 * k + 1]);
              u[k] = *reinterpret_cast<const uint32_t*>(&v);
            }
            *reinterpret_cast<uint4*>(my_staging + c * 4096 + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
        if (!p.staged) {  // rows that TMA cannot write (their pitch is no multiple of 16 bytes): neighbouring lanes store neighbours
          __syncwarp();
          const int from = row0 - lane;
          for (int r = 0; r < 32 && from + r < p.M; ++r) {
            bf16* dst = static_cast<bf16*>(p.c) + (from + r) * p.ldc;
#pragma unroll
            for (int c = lane; c < kOwn; c += 32) {
              const uint8_t* at = my_staging + (c / 64) * 4096 + r * 128 + ((((c % 64) / 8) ^ (r & 7)) << 4) + (c % 8) * 2;
              if (col0 + c < p.N) dst[col0 + c] = *reinterpret_cast<const bf16*>(at);
            }
          }
          __syncwarp();
          continue;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          for (int c = 0; c < kOwn / 64; ++c)
            if (row0 < p.M && col0 + c * 64 < p.N) tma_store_2d(&map_c, my_staging + c * 4096, col0 + c * 64, row0);
          bulk_commit();
        }
        continue;
      }
#pragma unroll
      for (int j = 0; j < kOwn / 4; ++j) {
        int row, col;
        place_quad(j, row, col);
        store_quad<Out>(p, row, col, make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]));
      }
    }
    if (C::kStaged && lane == 0) bulk_wait_read();
    if (!ok && lane == 0) *p.status = 1;
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) cg::this_cluster().sync();  // nothing of this CTA is read or signalled any more
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (kPair) tmem_dealloc_pair(tmem, kN * kBuffers);
    else tmem_dealloc(tmem, kN * kBuffers);
  }
  if constexpr (kPair) cg::this_cluster().sync();
}

// Once per kernel and device: room in shared memory, and that a kernel which moves registers between its warpgroups
// has the registers at launch that it was written for (an increase beyond them would wait forever).
void prepare_product(const void* kernel, int smem, int launch_regs) {
  static Once<std::pair<const void*, int>> once;
  int device = 0;
  C10_CUDA_CHECK(cudaGetDevice(&device));
  once({kernel, device}, [&] {
    if (launch_regs > 0) {
      cudaFuncAttributes attr;
      C10_CUDA_CHECK(cudaFuncGetAttributes(&attr, kernel));
      TORCH_CHECK(attr.numRegs >= launch_regs, "fp8: the product was built with ", attr.numRegs, " registers per thread; it needs ", launch_regs);
    }
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  });
}

// Results [M, N] in bf16, in boxes of 32 rows and 64 columns.
CUtensorMap result_map(const torch::Tensor& out, int64_t M, int64_t N) {
  CUtensorMap map;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(N) * 2};
  const cuuint32_t box[2] = {64, 32}, elem_strides[2] = {1, 1};
  const CUresult res = get_encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out.data_ptr(), dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(res == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", static_cast<int>(res));
  return map;
}

CUtensorMap operand_map(const torch::Tensor& t, int box_rows) {
  CUtensorMap map;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(t.size(1)), static_cast<cuuint64_t>(t.size(0))};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(t.stride(0))};
  const cuuint32_t box[2] = {kFp8Group, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem_strides[2] = {1, 1};
  const CUresult res = get_encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, t.data_ptr(), dims, strides, box, elem_strides,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(res == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", static_cast<int>(res));
  return map;
}

bool fp32_or_bf16(const torch::Tensor& t) { return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16; }

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t groups_of(int64_t n) { return (n + kFp8Group - 1) / kFp8Group; }

void check_source(const torch::Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && fp32_or_bf16(x), "fp8: the source is an fp32 or bf16 CUDA matrix");
  TORCH_CHECK(x.size(1) <= 1 || x.stride(1) == 1, "fp8: the source's rows are contiguous");
  TORCH_CHECK(x.size(1) < (1LL << 30), "fp8: the source is too wide");
}

bool vec_rows(const torch::Tensor& x) {
  return x.size(1) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && (x.stride(0) * x.element_size()) % 16 == 0;
}

template <typename F>
void with_source(const torch::Tensor& x, F&& f) {
  auto go = [&](auto* p) {
    if (vec_rows(x)) f(p, std::true_type{});
    else f(p, std::false_type{});
  };
  if (x.scalar_type() == torch::kFloat32) go(static_cast<const float*>(x.data_ptr()));
  else go(static_cast<const bf16*>(x.data_ptr()));
}

torch::Tensor bytes_of(const torch::Tensor& like, int64_t rows, int64_t cols) {
  return torch::empty({rows, up16(cols)}, like.options().dtype(torch::kUInt8));
}

struct ProductPlan {
  int n;  // columns of a tile; 256, and uncut 128 with a scale per row of B, by pairs of CTAs
  int splits;
};

// The shape of a tile by what the product would take with it: waves of tiles times the time of one group step of a tile, in units of a step of 128 x 128
// (measured on 16384 x 8192 x 2048: 269 us with pairs, 326 with 128 x 128, 644 with 128 x 64; a scale per row of B: 482, 499 as pairs of 256 x 128,
// 695).  Tiles of single CTAs are cut along K among up to eight while SMs are idle; joining two or
// four takes about two steps, eight (which have to start on one GPC) about twelve.
ProductPlan plan_product(int64_t M, int64_t N, int64_t K, bool column, int sms) {
  auto up = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
  const int64_t groups = groups_of(K);
  const double wide_step = column ? 1.93 : 1.63, narrow_step = column ? 0.7 : 1.0;
  const double wide = up(up(M, 256) * up(N, 256), sms / 2) * wide_step * groups;
  const double middle = (column ? up(up(M, 256) * up(N, 128), sms / 2) : up(up(M, 128) * up(N, 128), sms)) * static_cast<double>(groups);
  double best = std::min(wide, middle);
  ProductPlan plan{wide <= middle ? 256 : 128, 1};
  for (int n : {64, 128}) {
    const int64_t tiles = up(M, 128) * up(N, n);
    for (int s = n == 64 ? 1 : 2; s <= kMaxSplits && (s == 1 || (tiles * s <= sms && groups >= 2 * s)); s *= 2) {
      const double t = up(tiles * s, sms) * (n == 64 ? narrow_step : 1.) * up(groups, s) + (s == 8 ? 12. : s > 1 ? 2. : 0.);
      if (t < best) {
        best = t;
        plan = {n, s};
      }
    }
  }
  return plan;
}

void check_operand(const torch::Tensor& a, const torch::Tensor& s, const char* what) {
  TORCH_CHECK(a.is_cuda() && a.dim() == 2 && a.scalar_type() == torch::kUInt8, "fp8: operand ", what, " is a CUDA matrix of e4m3 bytes");
  TORCH_CHECK(a.stride(1) == 1 && a.stride(0) % 16 == 0 && a.stride(0) >= a.size(1) && reinterpret_cast<uintptr_t>(a.data_ptr()) % 16 == 0,
              "fp8: rows of operand ", what, " are contiguous and start at multiples of 16 bytes");
  TORCH_CHECK(s.device() == a.device() && s.dim() == 2 && s.scalar_type() == torch::kFloat32, "fp8: scales of operand ", what, " are an fp32 matrix on its device");
  TORCH_CHECK(s.size(1) == groups_of(a.size(1)), "fp8: operand ", what, " has ", groups_of(a.size(1)), " groups per row, its scales ", s.size(1));
  TORCH_CHECK(a.size(0) < (1LL << 30) && a.size(1) < (1LL << 30), "fp8: operand ", what, " is too large");
}

}  // namespace

// x [T, K] -> (e4m3 bytes [T, up16(K)], scales [groups, T])
std::tuple<torch::Tensor, torch::Tensor> fp8_rows(const torch::Tensor& x) {
  check_source(x);
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), K = x.size(1), G = groups_of(K);
  auto q = bytes_of(x, T, K);
  auto scale = torch::empty({G, T}, x.options().dtype(torch::kFloat32));
  if (T == 0 || K == 0) return {q, scale};
  TORCH_CHECK(groups_of(T) <= 65535, "fp8: the source has too many rows");
  auto st = at::cuda::getCurrentCUDAStream();
  with_source(x, [&](auto* p, auto vec) {
    using T_ = std::remove_cv_t<std::remove_pointer_t<decltype(p)>>;
    fp8_tile_kernel<T_, decltype(vec)::value, kRowGroups><<<dim3(static_cast<unsigned>(G), static_cast<unsigned>(groups_of(T))), kTileThreads, 0, st>>>(
        p, x.stride(0), q.data_ptr<uint8_t>(), q.stride(0), scale.data_ptr<float>(), nullptr, 0, nullptr, T, static_cast<int>(K));
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, scale};
}

// x [T, K] -> (bytes [T, up16(K)], scales [groups of K, T], bytes of the transpose [K, up16(T)], its scales [groups of T, K])
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> fp8_both(const torch::Tensor& x) {
  check_source(x);
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), K = x.size(1), G = groups_of(K), H = groups_of(T);
  auto f32 = x.options().dtype(torch::kFloat32);
  auto q = bytes_of(x, T, K), qt = bytes_of(x, K, T);
  auto scale = torch::empty({G, T}, f32), scale_t = torch::empty({H, K}, f32);
  if (T == 0 || K == 0) return {q, scale, qt, scale_t};
  TORCH_CHECK(H <= 65535, "fp8: the source has too many rows");
  auto st = at::cuda::getCurrentCUDAStream();
  with_source(x, [&](auto* p, auto vec) {
    using T_ = std::remove_cv_t<std::remove_pointer_t<decltype(p)>>;
    fp8_tile_kernel<T_, decltype(vec)::value, kBothGroups><<<dim3(static_cast<unsigned>(G), static_cast<unsigned>(H)), kTileThreads, 0, st>>>(
        p, x.stride(0), q.data_ptr<uint8_t>(), q.stride(0), scale.data_ptr<float>(), qt.data_ptr<uint8_t>(), qt.stride(0), scale_t.data_ptr<float>(), T,
        static_cast<int>(K));
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, scale, qt, scale_t};
}

// w [N, K] -> (bytes [N, up16(K)], bytes of the transpose [K, up16(N)] or empty, scales [groups of N, groups of K])
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> fp8_squares(const torch::Tensor& w, bool transpose) {
  check_source(w);
  c10::cuda::CUDAGuard guard(w.device());
  const int64_t N = w.size(0), K = w.size(1), G = groups_of(K), H = groups_of(N);
  auto q = bytes_of(w, N, K), qt = bytes_of(w, transpose ? K : 0, N);
  auto scale = torch::empty({H, G}, w.options().dtype(torch::kFloat32));
  if (N == 0 || K == 0) return {q, qt, scale};
  TORCH_CHECK(H <= 65535, "fp8: the source has too many rows");
  auto st = at::cuda::getCurrentCUDAStream();
  with_source(w, [&](auto* p, auto vec) {
    using T_ = std::remove_cv_t<std::remove_pointer_t<decltype(p)>>;
    fp8_tile_kernel<T_, decltype(vec)::value, kSquareGroups><<<dim3(static_cast<unsigned>(G), static_cast<unsigned>(H)), kTileThreads, 0, st>>>(
        p, w.stride(0), q.data_ptr<uint8_t>(), q.stride(0), scale.data_ptr<float>(), transpose ? qt.data_ptr<uint8_t>() : nullptr, qt.stride(0), nullptr, N,
        static_cast<int>(K));
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, qt, scale};
}

// a [M, K], b [N, K] e4m3 bytes; sa [M, groups]; sb [N, groups] or, per block of 128 rows of b, [ceil(N / 128), groups]; any strides.
// -> a b' [M, N] in fp32 or bf16, plus `addend` (fp32 [M, N]); as a tensor of `shape` where that is given.
torch::Tensor fp8_matmul(const torch::Tensor& a, const torch::Tensor& sa, const torch::Tensor& b, const torch::Tensor& sb, bool column_scales, bool out_bf16,
                         const std::optional<torch::Tensor>& addend, torch::Tensor status, std::optional<std::vector<int64_t>> shape) {
  check_operand(a, sa, "a");
  check_operand(b, sb, "b");
  const int64_t M = a.size(0), N = b.size(0), K = a.size(1);
  TORCH_CHECK(a.device() == b.device() && b.size(1) == K, "fp8: the operands have one inner size and one device");
  TORCH_CHECK(sa.size(0) == M && sb.size(0) == (column_scales ? N : groups_of(N)), "fp8: rows of the scales");
  TORCH_CHECK(status.device() == a.device() && status.scalar_type() == torch::kInt32 && status.numel() == 1, "fp8: status is one int32");
  c10::cuda::CUDAGuard guard(a.device());
  auto out = torch::empty(shape.has_value() ? *shape : std::vector<int64_t>{M, N}, sa.options().dtype(out_bf16 ? torch::kBFloat16 : torch::kFloat32));
  TORCH_CHECK(out.numel() == M * N, "fp8: shape of the result");
  if (addend.has_value())
    TORCH_CHECK(addend->device() == a.device() && addend->scalar_type() == torch::kFloat32 && addend->is_contiguous() && addend->sizes() == out.sizes(), "fp8: the addend is fp32 [M, N]");
  if (out.numel() == 0) return out;
  if (K == 0) return addend.has_value() ? out.copy_(*addend) : out.zero_();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  auto st = at::cuda::getCurrentCUDAStream();
  ProductArgs p{sa.data_ptr<float>(), sb.data_ptr<float>(), sa.stride(0), sa.stride(1), sb.stride(0), sb.stride(1), out.data_ptr(),
                addend.has_value() ? addend->data_ptr<float>() : nullptr, N, static_cast<int>(M), static_cast<int>(N), static_cast<int>(groups_of(K)),
                static_cast<int>((M + kTileM - 1) / kTileM), 0, 1, out_bf16 && !addend.has_value() && N % 8 == 0, status.data_ptr<int>()};
  auto go = [&](auto n, auto pair, auto column, auto out_tag, int splits) {
    constexpr int kN = decltype(n)::value;
    constexpr bool kPair = decltype(pair)::value;
    using Out = decltype(out_tag);
    using Cfg = ProductCfg<kN, kPair, decltype(column)::value, Out>;
    constexpr int kRows = kPair ? 2 * kTileM : kTileM;
    p.tiles_m = static_cast<int>((M + kRows - 1) / kRows);
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * ((N + kN - 1) / kN);
    TORCH_CHECK(tiles < (1LL << 31), "fp8: the product is too large");
    p.tiles = static_cast<int>(tiles);
    p.splits = splits;
    const CUtensorMap map_a = operand_map(a, kTileM), map_b = operand_map(b, Cfg::kRowsB);
    const CUtensorMap map_c = Cfg::kStaged && p.staged ? result_map(out, M, N) : map_a;
    auto* kernel = fp8_matmul_kernel<kN, kPair, decltype(column)::value, Out>;
    prepare_product(reinterpret_cast<const void*>(kernel), Cfg::kSmemBytes, Cfg::kUneven ? Cfg::kLaunchRegs : 0);
    cudaLaunchConfig_t cfg{};
    const int per_tile = kPair ? 2 : p.splits;  // CTAs, one cluster
    cfg.gridDim = dim3(p.splits > 1 ? p.tiles * p.splits : static_cast<unsigned>(std::min<int64_t>(tiles, sms / per_tile)) * per_tile);
    cfg.blockDim = dim3(kProductThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(per_tile), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = per_tile > 1 ? 1 : 0;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, map_c, p));
  };
  auto with_n = [&](auto column, auto out_tag) {
    constexpr bool kColumn = decltype(column)::value;
    const ProductPlan plan = plan_product(M, N, K, kColumn, sms);
    if (plan.n == 64) go(std::integral_constant<int, 64>{}, std::false_type{}, column, out_tag, plan.splits);
    else if (plan.n == 256) go(std::integral_constant<int, 256>{}, std::true_type{}, column, out_tag, 1);
    else if (plan.splits > 1) go(std::integral_constant<int, 128>{}, std::false_type{}, column, out_tag, plan.splits);
    else go(std::integral_constant<int, 128>{}, std::integral_constant<bool, kColumn>{}, column, out_tag, 1);
  };
  auto with_out = [&](auto column) {
    if (out_bf16) with_n(column, bf16{});
    else with_n(column, float{});
  };
  if (column_scales) with_out(std::true_type{});
  else with_out(std::false_type{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

void register_fp8_ops(pybind11::module_& m) {
  m.def("fp8_rows", &fp8_rows);
  m.def("fp8_both", &fp8_both);
  m.def("fp8_squares", &fp8_squares);
  m.def("fp8_plan", [](int64_t M, int64_t N, int64_t K, bool column_scales, int sms) {
    const ProductPlan plan = plan_product(M, N, K, column_scales, sms);
    return std::make_tuple(plan.n, plan.splits);
  });
  namespace py = pybind11;
  m.def("fp8_matmul", &fp8_matmul, py::arg("a"), py::arg("sa"), py::arg("b"), py::arg("sb"), py::arg("column_scales"), py::arg("out_bf16"), py::arg("addend"),
        py::arg("status"), py::arg("shape") = py::none());
}

}  // namespace ob200
