// Products of e4m3 operands with an fp32 scale per group of 128 along the summed dimension, and the kernels that bring operands into that format.
//
//   fp8_rows      x [T, K] -> e4m3 [T, K], scales [ceil(K / 128), T]
//   fp8_both      the same, and the transpose e4m3 [K, T] in groups of 128 rows of x, scales [ceil(T / 128), K], from one read of x
//   fp8_squares   w [N, K] -> e4m3 [N, K] and its transpose [K, N], one scale per 128 x 128 block
//   fp8_matmul    C[m, n] = sum_g sa[m, g] sb[n, g] sum_{k in g} a[m, k] b[n, k]
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "fp8_format.cuh"
#include "ptx.cuh"
#include "tensor_map.h"

namespace ob200 {
namespace {

using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------------------
// Into the format.  Bound by HBM: one read of x, one byte written per value and operand.
// ------------------------------------------------------------------------------------------------
constexpr int kRowsThreads = 256;

// Sixteen lanes take one group, eight values each.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowsThreads)
fp8_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, float* __restrict__ scale, long long rows, int K) {
  const int groups = (K + kFp8Group - 1) / kFp8Group, lane = threadIdx.x & 15;
  const long long total = rows * groups;
  const long long g = (static_cast<long long>(blockIdx.x) * kRowsThreads + threadIdx.x) >> 4;
  const long long row = g < total ? g / groups : 0;
  const int kb = g < total ? static_cast<int>(g % groups) : 0;
  const int col = kb * kFp8Group + lane * 8;
  float v[8];
  load8<kVec>(x + row * ldx, col, K, v);
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, magnitude_bits(v[k]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (g >= total) return;
  const GroupScale s = group_scale(top);
  if (col < K) *reinterpret_cast<uint2*>(q + row * ldq + col) = e4m3x8(v, s.factor);  // the pitch is a multiple of 16
  if (lane == 0) scale[static_cast<long long>(kb) * rows + row] = s.scale;
}

// A CTA takes a 128 x 128 tile: thread (ty, tx) holds rows 8 ty .. 8 ty + 7 and columns 8 tx .. 8 tx + 7.  The transpose goes through
// shared memory, where a thread has eight neighbouring bytes of each of its columns.
constexpr int kTileThreads = 256;
constexpr int kTilePitch = 128 + 16;  // bytes

template <typename T, bool kVec, bool kSquares>
__global__ void __launch_bounds__(kTileThreads)
fp8_tile_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, float* __restrict__ scale, uint8_t* __restrict__ qt,
                long long ldt, float* __restrict__ scale_t, long long rows, int K) {
  __shared__ uint32_t col_top[kFp8Group];
  __shared__ __align__(16) uint8_t flipped[kFp8Group * kTilePitch];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int kb = blockIdx.x;
  const long long tb = blockIdx.y;
  const int col = kb * kFp8Group + tx * 8;
  const long long row0 = tb * kFp8Group + ty * 8;
  if (threadIdx.x < kFp8Group) col_top[threadIdx.x] = 0;
  float v[8][8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if (row0 + r < rows) {
      load8<kVec>(x + (row0 + r) * ldx, col, K, v[r]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[r][k] = 0.f;
    }
  }
  __syncthreads();
  uint32_t tops[8];  // of a thread's columns
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t t = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) t = max(t, magnitude_bits(v[r][k]));
    tops[k] = t;
  }
  float factor_t[8];
  if constexpr (kSquares) {
    uint32_t t = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) t = max(t, tops[k]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
    if ((threadIdx.x & 31) == 0) atomicMax(&col_top[0], t);
    __syncthreads();
    const GroupScale s = group_scale(col_top[0]);
#pragma unroll
    for (int k = 0; k < 8; ++k) factor_t[k] = s.factor;
    if (threadIdx.x == 0) scale[tb * gridDim.x + kb] = s.scale;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (row0 + r < rows && col < K) *reinterpret_cast<uint2*>(q + (row0 + r) * ldq + col) = e4m3x8(v[r], s.factor);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) atomicMax(&col_top[tx * 8 + k], tops[k]);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      uint32_t t = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) t = max(t, magnitude_bits(v[r][k]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
      const GroupScale s = group_scale(t);
      if (row0 + r < rows) {
        if (col < K) *reinterpret_cast<uint2*>(q + (row0 + r) * ldq + col) = e4m3x8(v[r], s.factor);
        if (tx == 0) scale[static_cast<long long>(kb) * rows + row0 + r] = s.scale;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const GroupScale s = group_scale(col_top[tx * 8 + k]);
      factor_t[k] = s.factor;
      if (ty == 0 && col + k < K) scale_t[tb * K + col + k] = s.scale;
    }
  }
  if (kSquares && qt == nullptr) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float c[8] = {v[0][k], v[1][k], v[2][k], v[3][k], v[4][k], v[5][k], v[6][k], v[7][k]};
    *reinterpret_cast<uint2*>(flipped + (tx * 8 + k) * kTilePitch + ty * 8) = e4m3x8(c, factor_t[k]);
  }
  __syncthreads();
  // Row c of the transpose: 128 bytes, of which those beyond the pitch do not exist (the pitch is a multiple of 16).
  for (int i = threadIdx.x; i < kFp8Group * 8; i += kTileThreads) {
    const int c = i >> 3, part = (i & 7) * 16;
    if (kb * kFp8Group + c < K && tb * kFp8Group + part < ldt)
      *reinterpret_cast<uint4*>(qt + static_cast<long long>(kb * kFp8Group + c) * ldt + tb * kFp8Group + part) =
          *reinterpret_cast<const uint4*>(flipped + c * kTilePitch + part);
  }
}

// ------------------------------------------------------------------------------------------------
// The product.  A tile of 128 x kN results goes over K in steps of one group of 128: TMA brings 128 x 128 bytes of A and kN x 128 of B,
// four tcgen05.mma sum the group into a TMEM buffer of its own, and eight epilogue warps read the buffer, apply the two scales
// of the group and add it to sums that stay in fp32 registers, while the MMAs of the next groups fill the other buffers.
// ------------------------------------------------------------------------------------------------
constexpr int kTileM = 128;
constexpr int kEpilogueWarps = 8;
constexpr int kProductThreads = 32 * (kEpilogueWarps + 2);

template <int kN>
struct ProductCfg {
  static constexpr int kStageBytes = (kTileM + kN) * kFp8Group;
  static constexpr int kStages = kN == 256 ? 4 : kN == 128 ? 6 : 8;
  static constexpr int kBuffers = kN == 256 ? 2 : 4;  // TMEM buffers of kN columns
  static constexpr int kOwn = kN / 2;                 // columns of one epilogue warp: two warps share a 32-row stripe
  static constexpr int kScaleFloats = kEpilogueWarps * kOwn;
  static constexpr int kBarrierBytes = 256;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kScaleFloats * 4 + kBarrierBytes;  // 1 KB to align the stages
};

struct ProductArgs {
  const float *sa, *sb;
  long long sa_row, sa_group, sb_row, sb_group;  // strides of the scales; kColumnScale false: sb_row counts blocks of 128 rows of B
  void* c;
  const float* addend;  // fp32, C's layout, or null
  long long ldc;
  int M, N, groups, tiles_m, tiles;
  int* status;
};

template <int kN, bool kColumnScale, typename Out>
__global__ void __launch_bounds__(kProductThreads, 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const ProductArgs p) {
  using C = ProductCfg<kN>;
  constexpr int kStages = C::kStages, kBuffers = C::kBuffers, kOwn = C::kOwn;
  constexpr uint32_t kIdesc = make_idesc(/*e4m3*/ 0, kTileM, kN);
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  float* col_scales = reinterpret_cast<float*>(smem + kStages * C::kStageBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(col_scales + C::kScaleFloats);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + kBuffers;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + kBuffers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert(2 * (kStages + kBuffers) * 8 + 8 <= C::kBarrierBytes, "barrier region");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBuffers; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpilogueWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == kEpilogueWarps + 1) {
    tmem_alloc(tmem_holder, kN * kBuffers);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_holder;

  // Neighbouring tiles share operands: eight rows of tiles at a time, down the rows first.
  const int tiles_n = p.tiles / p.tiles_m;
  auto place = [&](int t, int& m0, int& n0) {
    const int band = t / (8 * tiles_n), in = t - band * 8 * tiles_n;
    const int high = min(8, p.tiles_m - band * 8);
    m0 = (band * 8 + in % high) * kTileM;
    n0 = in / high * kN;
  };

  if (warp == kEpilogueWarps) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
        int m0, n0;
        place(t, m0, n0);
        for (int g = 0; g < p.groups; ++g) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* s = smem + stage * C::kStageBytes;
          mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
          tma_load_2d(s, &map_a, &full[stage], g * kFp8Group, m0);
          tma_load_2d(s + kTileM * kFp8Group, &map_b, &full[stage], g * kFp8Group, n0);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == kEpilogueWarps + 1) {
    if (lane == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, round = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
        for (int g = 0; g < p.groups; ++g) {
          if (!mbar_wait(&acc_empty[buf], round ^ 1, abort_flag) || !mbar_wait(&full[stage], phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t s = smem_u32(smem + stage * C::kStageBytes);
          const uint64_t a = make_kmajor_sw128_desc(s), b = make_kmajor_sw128_desc(s + kTileM * kFp8Group);
#pragma unroll
          for (int k = 0; k < kFp8Group / 32; ++k) umma_f8(tmem + buf * kN, a + 2 * k, b + 2 * k, kIdesc, k != 0);
          umma_commit(&empty[stage]);
          umma_commit(&acc_full[buf]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
          if (++buf == kBuffers) {
            buf = 0;
            round ^= 1;
          }
        }
      }
    }
  } else {
    const int stripe = warp & 3, half = warp >> 2;
    float* my_scales = col_scales + warp * kOwn;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(stripe * 32) << 16) + half * kOwn;
    int buf = 0;
    uint32_t round = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x) {
      int m0, n0;
      place(t, m0, n0);
      const int row = m0 + stripe * 32 + lane, col0 = n0 + half * kOwn;
      const float* sa = p.sa + min(row, p.M - 1) * p.sa_row;
      float acc[kOwn];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) acc[j] = 0.f;
      for (int g = 0; g < p.groups && ok; ++g) {
        float scale = sa[g * p.sa_group];
        if constexpr (kColumnScale) {
          __syncwarp();
#pragma unroll
          for (int j = lane; j < kOwn; j += 32) my_scales[j] = p.sb[min(col0 + j, p.N - 1) * p.sb_row + g * p.sb_group];
          __syncwarp();
        } else {
          scale *= p.sb[min(col0, p.N - 1) / kFp8Group * p.sb_row + g * p.sb_group];
        }
        ok = mbar_wait(&acc_full[buf], round, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < kOwn / 32; ++c) {
          float v[32];
          tmem_ld_32x32(lanes + buf * kN + c * 32, v);
          if (c == kOwn / 32 - 1) {  // the buffer goes back to the MMAs
            tc_fence_before_sync();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c * 32 + j] = fmaf(kColumnScale ? v[j] * my_scales[c * 32 + j] : v[j], scale, acc[c * 32 + j]);
        }
        if (++buf == kBuffers) {
          buf = 0;
          round ^= 1;
        }
      }
      if (row >= p.M) continue;
      Out* dst = static_cast<Out*>(p.c) + row * p.ldc;
      const float* add = p.addend == nullptr ? nullptr : p.addend + row * p.ldc;
      const bool vec = (p.ldc & 7) == 0;
#pragma unroll
      for (int j = 0; j < kOwn; j += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = ok ? acc[j + k] : __int_as_float(0x7fffffff);  // a pipeline that gave up leaves no plausible numbers
          if (add != nullptr && col0 + j + k < p.N) v[k] += add[col0 + j + k];
        }
        if (vec && col0 + j + 8 <= p.N) store8<true>(dst, col0 + j, p.N, v);
        else store8<false>(dst, col0 + j, p.N, v);
      }
    }
    if (!ok && lane == 0) *p.status = 1;
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kEpilogueWarps + 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kN * kBuffers);
  }
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
  const int64_t grid = (T * G * 16 + kRowsThreads - 1) / kRowsThreads;
  TORCH_CHECK(grid < (1LL << 31), "fp8: the source is too large");
  auto st = at::cuda::getCurrentCUDAStream();
  with_source(x, [&](auto* p, auto vec) {
    using T_ = std::remove_cv_t<std::remove_pointer_t<decltype(p)>>;
    fp8_rows_kernel<T_, decltype(vec)::value><<<static_cast<unsigned>(grid), kRowsThreads, 0, st>>>(
        p, x.stride(0), q.data_ptr<uint8_t>(), q.stride(0), scale.data_ptr<float>(), T, static_cast<int>(K));
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
    fp8_tile_kernel<T_, decltype(vec)::value, false><<<dim3(static_cast<unsigned>(G), static_cast<unsigned>(H)), kTileThreads, 0, st>>>(
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
    fp8_tile_kernel<T_, decltype(vec)::value, true><<<dim3(static_cast<unsigned>(G), static_cast<unsigned>(H)), kTileThreads, 0, st>>>(
        p, w.stride(0), q.data_ptr<uint8_t>(), q.stride(0), scale.data_ptr<float>(), transpose ? qt.data_ptr<uint8_t>() : nullptr, qt.stride(0), nullptr, N,
        static_cast<int>(K));
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, qt, scale};
}

// a [M, K], b [N, K] e4m3 bytes; sa [M, groups]; sb [N, groups] or, per block of 128 rows of b, [ceil(N / 128), groups]; any strides.
// -> a b' [M, N] in fp32 or bf16, plus `addend` (fp32 [M, N]).
torch::Tensor fp8_matmul(const torch::Tensor& a, const torch::Tensor& sa, const torch::Tensor& b, const torch::Tensor& sb, bool column_scales, bool out_bf16,
                         const std::optional<torch::Tensor>& addend, torch::Tensor status) {
  check_operand(a, sa, "a");
  check_operand(b, sb, "b");
  const int64_t M = a.size(0), N = b.size(0), K = a.size(1);
  TORCH_CHECK(a.device() == b.device() && b.size(1) == K, "fp8: the operands have one inner size and one device");
  TORCH_CHECK(sa.size(0) == M && sb.size(0) == (column_scales ? N : groups_of(N)), "fp8: rows of the scales");
  TORCH_CHECK(status.device() == a.device() && status.scalar_type() == torch::kInt32 && status.numel() == 1, "fp8: status is one int32");
  c10::cuda::CUDAGuard guard(a.device());
  auto out = torch::empty({M, N}, sa.options().dtype(out_bf16 ? torch::kBFloat16 : torch::kFloat32));
  if (addend.has_value())
    TORCH_CHECK(addend->device() == a.device() && addend->scalar_type() == torch::kFloat32 && addend->is_contiguous() && addend->sizes() == out.sizes(), "fp8: the addend is fp32 [M, N]");
  if (out.numel() == 0) return out;
  if (K == 0) return addend.has_value() ? out.copy_(*addend) : out.zero_();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  auto st = at::cuda::getCurrentCUDAStream();
  ProductArgs p{sa.data_ptr<float>(), sb.data_ptr<float>(), sa.stride(0), sa.stride(1), sb.stride(0), sb.stride(1), out.data_ptr(),
                addend.has_value() ? addend->data_ptr<float>() : nullptr, N, static_cast<int>(M), static_cast<int>(N), static_cast<int>(groups_of(K)),
                static_cast<int>((M + kTileM - 1) / kTileM), 0, status.data_ptr<int>()};
  auto go = [&](auto n, auto column, auto out_tag) {
    constexpr int kN = decltype(n)::value;
    using Out = decltype(out_tag);
    using Cfg = ProductCfg<kN>;
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * ((N + kN - 1) / kN);
    TORCH_CHECK(tiles < (1LL << 31), "fp8: the product is too large");
    p.tiles = static_cast<int>(tiles);
    auto* kernel = fp8_matmul_kernel<kN, decltype(column)::value, Out>;
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes));
    kernel<<<static_cast<unsigned>(std::min<int64_t>(tiles, sms)), kProductThreads, Cfg::kSmemBytes, st>>>(operand_map(a, kTileM), operand_map(b, kN), p);
  };
  auto with_n = [&](auto column, auto out_tag) {
    if (p.tiles_m * ((N + 255) / 256) >= sms) go(std::integral_constant<int, 256>{}, column, out_tag);
    else if (p.tiles_m * ((N + 127) / 128) >= sms) go(std::integral_constant<int, 128>{}, column, out_tag);
    else go(std::integral_constant<int, 64>{}, column, out_tag);
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
  m.def("fp8_matmul", &fp8_matmul);
}

}  // namespace ob200
