// Token embedding with a scale, and the dense gradient of its table.
//
//   embed_fwd      y[t] = scale * table[id[t]]
//   embed_bwd      dtable[v] = scale * sum over t with id[t] == v of dy[t], added in a fixed order; rows of absent tokens are zero
//
// The gradient takes three launches:
//   1. sort    one cluster of eight CTAs sorts the (token, position) pairs in its shared memory, exchanging them over distributed
//              shared memory, while every other CTA writes the zeros of the table: the sort (tens of microseconds of latency, almost no bandwidth)
//              hides behind the write that the result needs anyway.
//   2. pieces  runs of kPiece sorted pairs, each summed by one CTA per column slice whatever tokens it holds, so that a token that fills half
//              of the batch costs no more than others.  A token whose pairs lie in one piece goes straight into the table; the
//              others leave a partial sum per piece.
//   3. joins   adds the partial sums of a token, every eighth piece in a chain of its own, then the eight chains.
// Up to 128 tokens take one launch instead.
// No floating-point atomics: the same inputs give the same bits.  16384 tokens over 50257 x 768 fp32: 27 + 14 + 11 us; the write of the table alone
// takes 24.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <torch/extension.h>

#include <map>
#include <mutex>

#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace ob200 {
namespace {

template <typename T>
__device__ __forceinline__ float as_float(T x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T as(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else return __float2bfloat16_rn(x);
}

// N consecutive values, as one or two 16-byte accesses where kVec (the address is then a multiple of that size).
template <int N, typename T>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T e[N];
};

template <typename Id>
__device__ __forceinline__ long long token_at(const Id* ids, long long i) {
  return static_cast<long long>(ids[i]);
}

// ------------------------------------------------------------------------------------------------
// Forward: bound by HBM and the L2 (rows of frequent tokens stay there).  A warp takes 128 packs of one row, four loads in
// flight per lane.  A token outside the table gives a row of NaN.  16384 x 768 fp32: 16 us (6.1 TB/s).
// ------------------------------------------------------------------------------------------------
template <int N, typename T, typename Out, typename Id>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(const Id* __restrict__ ids, const T* __restrict__ table, Out* __restrict__ out, long long n, long long V, int C, float scale) {
  const int packs = C / N, segs = (packs + 127) / 128;
  const int lane = threadIdx.x & 31;
  const long long warp = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const long long row = warp / segs;
  if (row >= n) return;
  const int first = static_cast<int>(warp % segs) * 128 + lane;
  const long long id = token_at(ids, row);
  const bool known = id >= 0 && id < V;
  const auto* src = reinterpret_cast<const Pack<N, T>*>(table + (known ? id : 0) * C);
  auto* dst = reinterpret_cast<Pack<N, Out>*>(out + row * C);
  Pack<N, T> u[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (first + 32 * q < packs) u[q] = src[first + 32 * q];
  const float s = known ? scale : __int_as_float(0x7fffffff);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (first + 32 * q >= packs) break;
    Pack<N, Out> o;
#pragma unroll
    for (int k = 0; k < N; ++k) o.e[k] = as<Out>(s * as_float(u[q].e[k]));
    dst[first + 32 * q] = o;
  }
}

// ------------------------------------------------------------------------------------------------
// 1. Stable radix sort of up to 65536 (token, position) pairs, eight bits a pass, in the shared memory of one cluster.
// ------------------------------------------------------------------------------------------------
constexpr int kSortCtas = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxPerThread = 8;
constexpr int kSortCapacity = kSortCtas * kSortThreads * kMaxPerThread;
constexpr int kDigits = 256;

struct SortShared {
  unsigned hist[kSortWarps][kDigits];  // pairs of a digit in a warp, then in the warps before it
  unsigned total[kDigits];             // pairs of a digit in this CTA: read by the whole cluster
  unsigned base[kDigits];              // place of this CTA's first pair of a digit
  unsigned scan[kDigits / 32];
};

constexpr int kZeroBytes = 32768;
static_assert(sizeof(SortShared) >= kZeroBytes, "the zeros fit into what the sort takes");

size_t sort_smem(int per_thread) { return sizeof(SortShared) + 2 * 8ull * kSortThreads * per_thread; }

template <int kPer, typename Id>
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
embed_sort_kernel(const Id* __restrict__ ids, int n, long long V, int bits, unsigned* __restrict__ keys_out, int* __restrict__ pos_out,
                  uint4* __restrict__ zero, long long zero_vecs, unsigned char* __restrict__ zero_tail, int tail_bytes) {
  extern __shared__ __align__(16) unsigned char raw[];
  if (blockIdx.x >= kSortCtas) {
    // The zeros of the table: copies of 32 KB of zeros by the copy engine, which one thread commands (plain stores of all threads reached 3.9
    // TB/s, 40 us for 50257 x 768).
    for (int i = threadIdx.x; i < kZeroBytes / 16; i += kSortThreads) reinterpret_cast<uint4*>(raw)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
    __syncthreads();
    const int own = blockIdx.x - kSortCtas, all = gridDim.x - kSortCtas;
    if (threadIdx.x == 0) {
      const long long bytes = zero_vecs * 16;
      for (long long at = static_cast<long long>(own) * kZeroBytes; at < bytes; at += static_cast<long long>(all) * kZeroBytes)
        bulk_store(reinterpret_cast<unsigned char*>(zero) + at, raw, static_cast<uint32_t>(bytes - at < kZeroBytes ? bytes - at : kZeroBytes));
      bulk_commit();
      bulk_wait();
    }
    if (own == 0 && threadIdx.x < tail_bytes) zero_tail[threadIdx.x] = 0;
    return;
  }
  SortShared& sh = *reinterpret_cast<SortShared*>(raw);
  constexpr int kOwn = kSortThreads * kPer;  // pairs of one CTA
  uint2* buf[2] = {reinterpret_cast<uint2*>(raw + sizeof(SortShared)), reinterpret_cast<uint2*>(raw + sizeof(SortShared)) + kOwn};
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = warp * 32 * kPer + lane;  // a warp owns 32 * kPer neighbours and visits them in order
  for (int q = 0; q < kPer; ++q) {
    const int i = cta * kOwn + first + 32 * q;
    unsigned key = 0xffffffffu;  // behind the last pair
    if (i < n) {
      const long long id = token_at(ids, i);
      key = id >= 0 && id < V ? static_cast<unsigned>(id) : static_cast<unsigned>(V);  // tokens outside the table come last
    }
    buf[0][first + 32 * q] = make_uint2(key, static_cast<unsigned>(i));
  }
  int cur = 0;
  for (int shift = 0; shift < bits; shift += 8, cur ^= 1) {
    for (int d = lane; d < kDigits; d += 32) sh.hist[warp][d] = 0;
    __syncwarp();
    uint2 pair[kPer];
    unsigned rank[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      pair[q] = buf[cur][first + 32 * q];
      const unsigned d = (pair[q].x >> shift) & (kDigits - 1);
      const unsigned peers = __match_any_sync(0xffffffffu, d);
      const unsigned before = sh.hist[warp][d];
      __syncwarp();
      rank[q] = before + __popc(peers & ((1u << lane) - 1));
      if (lane == 31 - __clz(peers)) sh.hist[warp][d] = before + __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      unsigned run = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = sh.hist[w][threadIdx.x];
        sh.hist[w][threadIdx.x] = run;
        run += c;
      }
      sh.total[threadIdx.x] = run;
    }
    cluster.sync();
    unsigned all = 0, below = 0, incl = 0;
    if (threadIdx.x < kDigits) {
      for (int c = 0; c < kSortCtas; ++c) {
        const unsigned t = cluster.map_shared_rank(sh.total, c)[threadIdx.x];
        all += t;
        below += c < cta ? t : 0;
      }
      incl = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (lane == 31) sh.scan[warp] = incl;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      unsigned lower = 0;
      for (int w = 0; w < warp; ++w) lower += sh.scan[w];
      sh.base[threadIdx.x] = lower + incl - all + below;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const unsigned d = (pair[q].x >> shift) & (kDigits - 1);
      const unsigned to = sh.base[d] + sh.hist[warp][d] + rank[q];
      cluster.map_shared_rank(buf[cur ^ 1], to / kOwn)[to % kOwn] = pair[q];
    }
    cluster.sync();
  }
  for (int q = 0; q < kPer; ++q) {
    const int i = cta * kOwn + threadIdx.x + kSortThreads * q;
    if (i < n) {
      const uint2 p = buf[cur][threadIdx.x + kSortThreads * q];
      keys_out[i] = p.x;
      pos_out[i] = static_cast<int>(p.y);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// 2. and 3. Sums.  The row of a token that lies in one piece is written (kAdd: added to) by that piece; a token that crosses
// a border leaves its sum in partial[piece][0] where it came from the piece before, in partial[piece][1] where it starts.
// ------------------------------------------------------------------------------------------------
constexpr int kPiece = 32;
constexpr int kPieceUnroll = 8;

template <int N, typename T, bool kAdd>
__device__ __forceinline__ void store_row(T* table, long long at, const float (&v)[N]) {
  auto* dst = reinterpret_cast<Pack<N, T>*>(table + at);
  Pack<N, T> o;
  if constexpr (kAdd) o = *dst;
#pragma unroll
  for (int k = 0; k < N; ++k) o.e[k] = as<T>(kAdd ? as_float(o.e[k]) + v[k] : v[k]);
  *dst = o;
}

template <int N, typename Grad, typename T, bool kAdd>
__global__ void __launch_bounds__(256)
embed_pieces_kernel(const unsigned* __restrict__ keys, const int* __restrict__ pos, const Grad* __restrict__ dy, T* __restrict__ table,
                    float* __restrict__ partial, int n, unsigned V, int C, float scale) {
  __shared__ unsigned key[kPiece + 2];  // with the neighbours before and behind
  __shared__ int at[kPiece];
  const int i0 = blockIdx.x * kPiece, count = min(kPiece, n - i0);
  for (int i = threadIdx.x; i < kPiece + 2; i += blockDim.x) {
    const int g = i0 + i - 1;
    key[i] = g >= 0 && g < n ? keys[g] : 0xffffffffu;
    if (i < count) at[i] = pos[i0 + i];
  }
  __syncthreads();
  const int pack = blockIdx.y * blockDim.x + threadIdx.x;
  if (pack * N >= C) return;
  const long long col = static_cast<long long>(pack) * N;
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  bool from_before = key[0] == key[1];
  auto flush = [&](unsigned token, bool goes_on) {
    if (token < V) {
      if (from_before || goes_on) {
        float* dst = partial + (static_cast<long long>(blockIdx.x) * 2 + (from_before ? 0 : 1)) * C + col;
#pragma unroll
        for (int k = 0; k < N; ++k) dst[k] = acc[k];
      } else {
        float v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = scale * acc[k];
        store_row<N, T, kAdd>(table, static_cast<long long>(token) * C + col, v);
      }
    }
    from_before = false;
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
  };
  for (int i = 0; i < count; i += kPieceUnroll) {
    Pack<N, Grad> u[kPieceUnroll];
#pragma unroll
    for (int q = 0; q < kPieceUnroll; ++q)
      if (i + q < count) u[q] = *reinterpret_cast<const Pack<N, Grad>*>(dy + static_cast<long long>(at[i + q]) * C + col);
#pragma unroll
    for (int q = 0; q < kPieceUnroll; ++q) {
      if (i + q >= count) break;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += as_float(u[q].e[k]);
      if (i + q + 1 == count || key[i + q + 2] != key[i + q + 1])
        flush(key[i + q + 1], i + q + 1 == count && key[i + q + 2] == key[i + q + 1]);
    }
  }
}

constexpr int kJoinRows = 8;

// One CTA per piece in which a token starts that goes on behind it (all others return at once): eight rows of threads add every
// eighth piece each, then the eight sums are added in order.
template <typename T, bool kAdd>
__global__ void __launch_bounds__(32 * kJoinRows)
embed_join_kernel(const unsigned* __restrict__ keys, const float* __restrict__ partial, T* __restrict__ table, int n, unsigned V, int C, float scale) {
  __shared__ float sums[kJoinRows][128];
  const int pieces = (n + kPiece - 1) / kPiece, j = blockIdx.x;
  if (j + 1 >= pieces) return;
  const unsigned token = keys[j * kPiece + kPiece - 1];
  if (token >= V || keys[(j + 1) * kPiece] != token) return;
  if (keys[j * kPiece] == token && j > 0 && keys[j * kPiece - 1] == token) return;  // it started earlier
  int lo = j + 1;  // the last piece that begins with the token, looked for among as many as there are threads at a time
  for (int more = 32 * kJoinRows; more == 32 * kJoinRows; lo += more) {
    const int p = lo + 1 + static_cast<int>(threadIdx.x);
    more = __syncthreads_count(p < pieces && keys[p * kPiece] == token);
  }
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  for (int c0 = blockIdx.y * 128; c0 < C; c0 += gridDim.y * 128) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p = j + row; p <= lo; p += kJoinRows) {
      const float* from = partial + (static_cast<long long>(p) * 2 + (p == j ? 1 : 0)) * C;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c0 + 32 * k + lane < C) s[k] += from[c0 + 32 * k + lane];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[row][32 * k + lane] = s[k];
    __syncthreads();
    const int c = c0 + threadIdx.x;
    if (threadIdx.x < 128 && c < C) {
      float t = 0.f;
#pragma unroll
      for (int r = 0; r < kJoinRows; ++r) t += sums[r][threadIdx.x];
      const float v[1] = {scale * t};
      store_row<1, T, kAdd>(table, static_cast<long long>(token) * C + c, v);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------
// Up to 128 tokens: one launch, a warp per row of the table and 128 packs of it, which looks the row's number up among the tokens.  The
// three launches of the sort would cost more than the sums; beyond this the longest sum (one token throughout) would.
// ------------------------------------------------------------------------------------------------
constexpr int kFewTokens = 128;

template <int N, typename Grad, typename T, typename Id>
__global__ void __launch_bounds__(256)
embed_few_kernel(const Id* __restrict__ ids, const Grad* __restrict__ dy, T* __restrict__ table, int n, long long V, int C, float scale) {
  const int packs = C / N, segs = (packs + 127) / 128, lane = threadIdx.x & 31;
  long long mine[kFewTokens / 32];
#pragma unroll
  for (int h = 0; h < kFewTokens / 32; ++h) mine[h] = h * 32 + lane < n ? token_at(ids, h * 32 + lane) : -1;
  const long long items = V * segs, step = static_cast<long long>(gridDim.x) * 8;
  for (long long w = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); w < items; w += step) {
    const long long v = w / segs;
    const int first = static_cast<int>(w - v * segs) * 128 + lane;
    float acc[4][N];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int k = 0; k < N; ++k) acc[q][k] = 0.f;
#pragma unroll
    for (int h = 0; h < kFewTokens / 32; ++h) {
      unsigned who = __ballot_sync(0xffffffffu, mine[h] == v);
      while (who != 0) {  // in ascending order, two rows on their way at a time
        int t[2];
        t[0] = h * 32 + __ffs(who) - 1;
        who &= who - 1;
        t[1] = who != 0 ? h * 32 + __ffs(who) - 1 : -1;
        who &= who - 1;
        Pack<N, Grad> u[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (t[r] >= 0 && first + 32 * q < packs) u[r][q] = reinterpret_cast<const Pack<N, Grad>*>(dy + static_cast<long long>(t[r]) * C)[first + 32 * q];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (t[r] >= 0 && first + 32 * q < packs) {
#pragma unroll
              for (int k = 0; k < N; ++k) acc[q][k] += as_float(u[r][q].e[k]);
            }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (first + 32 * q >= packs) break;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[q][k] *= scale;
      store_row<N, T, false>(table, v * C + static_cast<long long>(first + 32 * q) * N, acc[q]);
    }
  }
}

// Clusters of the sort kernel that the device holds at once: the zeros are shared out among those, since a cluster of a second wave would double
// their time (18 clusters of eight are one per SM of 148, but 16 fit into the GPCs: 41 us instead of 27 for 50257 x 768).
template <typename Kernel>
int clusters_at_once(Kernel* kernel, size_t smem) {
  static std::mutex mutex;
  static std::map<std::pair<const void*, int>, int> known;
  int device = 0;
  C10_CUDA_CHECK(cudaGetDevice(&device));
  std::lock_guard<std::mutex> lock(mutex);
  int& n = known[{reinterpret_cast<const void*>(kernel), device}];
  if (n == 0) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kSortCtas);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {kSortCtas, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    C10_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    n = std::max(n, 2);
  }
  return n;
}

bool fp32_or_bf16(const torch::Tensor& t) { return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16; }

bool packs_of(const torch::Tensor& t, int64_t C, int N) {
  const int64_t bytes = std::min<int64_t>(16, N * t.element_size());
  return C % N == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0;
}

template <typename F>
void with_type(const torch::Tensor& t, F&& f) {
  if (t.scalar_type() == torch::kFloat32) f(static_cast<float*>(t.data_ptr()));
  else f(static_cast<__nv_bfloat16*>(t.data_ptr()));
}
template <typename F>
void with_ids(const torch::Tensor& ids, F&& f) {
  if (ids.scalar_type() == torch::kInt64) f(reinterpret_cast<const long long*>(ids.data_ptr()));
  else f(reinterpret_cast<const int*>(ids.data_ptr()));
}

void check_ids(const torch::Tensor& ids, const torch::Tensor& other) {
  TORCH_CHECK(ids.is_cuda() && ids.device() == other.device() && ids.is_contiguous() &&
                  (ids.scalar_type() == torch::kInt64 || ids.scalar_type() == torch::kInt32), "embedding: ids are contiguous int64 or int32 on the table's device");
}

}  // namespace

// ids [...], table [V, C] -> [..., C]
torch::Tensor embed_fwd(const torch::Tensor& ids, const torch::Tensor& table, double scale, bool out_bf16) {
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.is_contiguous() && fp32_or_bf16(table), "embedding: the table is contiguous fp32 or bf16 [V, C]");
  check_ids(ids, table);
  const int64_t n = ids.numel(), V = table.size(0), C = table.size(1);
  TORCH_CHECK(V > 0 && V < (1LL << 31) && C < (1LL << 31), "embedding: table size");
  c10::cuda::CUDAGuard guard(table.device());
  auto sizes = ids.sizes().vec();
  sizes.push_back(C);
  auto out = torch::empty(sizes, table.options().dtype(out_bf16 ? torch::kBFloat16 : torch::kFloat32));
  if (out.numel() == 0) return out;
  auto st = at::cuda::getCurrentCUDAStream();
  const int N = table.scalar_type() == torch::kFloat32 && !out_bf16 ? 4 : 8;
  const bool vec = packs_of(table, C, N) && packs_of(out, C, N);
  const int64_t packs = vec ? C / N : C;
  const int64_t warps = n * ((packs + 127) / 128), grid = (warps + 7) / 8;
  TORCH_CHECK(grid < (1LL << 31), "embedding: too many rows");
  with_ids(ids, [&](auto* idp) {
    with_type(table, [&](auto* tp) {
      with_type(out, [&](auto* op) {
        using T = std::remove_pointer_t<decltype(tp)>;
        using Out = std::remove_pointer_t<decltype(op)>;
        using Id = std::remove_cv_t<std::remove_pointer_t<decltype(idp)>>;
        constexpr int kN = sizeof(T) == 4 && sizeof(Out) == 4 ? 4 : 8;
        const auto g = static_cast<unsigned>(grid);
        const float s = static_cast<float>(scale);
        if (vec) embed_fwd_kernel<kN, T, Out, Id><<<g, 256, 0, st>>>(idp, tp, op, n, V, static_cast<int>(C), s);
        else embed_fwd_kernel<1, T, Out, Id><<<g, 256, 0, st>>>(idp, tp, op, n, V, static_cast<int>(C), s);
      });
    });
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

// ids [...], dy [..., C] -> gradient of the table [V, C], fp32 or bf16
torch::Tensor embed_bwd(const torch::Tensor& ids, const torch::Tensor& dy, int64_t V, double scale, bool out_bf16) {
  TORCH_CHECK(dy.is_cuda() && dy.dim() == ids.dim() + 1 && dy.is_contiguous() && fp32_or_bf16(dy) && dy.numel() == ids.numel() * dy.size(-1),
              "embedding: dy is contiguous fp32 or bf16 [..., C]");
  check_ids(ids, dy);
  const int64_t n = ids.numel(), C = dy.size(-1);
  TORCH_CHECK(V > 0 && V < (1LL << 31) && C < (1LL << 31), "embedding: table size");
  c10::cuda::CUDAGuard guard(dy.device());
  // Batches beyond the sort's capacity are taken in slices that add to the table, in fp32 whatever the result's type.
  const bool sliced = n > kSortCapacity;
  auto f32 = dy.options().dtype(torch::kFloat32);
  auto out = torch::empty({V, C}, out_bf16 && !sliced ? dy.options().dtype(torch::kBFloat16) : f32);
  if (out.numel() == 0) return out_bf16 ? out.to(torch::kBFloat16) : out;
  if (n == 0) return out.zero_();
  auto st = at::cuda::getCurrentCUDAStream();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int N = dy.scalar_type() == torch::kFloat32 ? 4 : 8;
  const bool vec = packs_of(dy, C, N) && packs_of(out, C, N);
  if (n <= kFewTokens) {
    const int64_t items = V * (((vec ? C / N : C) + 127) / 128);
    const auto grid = static_cast<unsigned>(std::min<int64_t>((items + 7) / 8, 8 * sms));
    with_ids(ids, [&](auto* idp) {
      with_type(dy, [&](auto* gp) {
        with_type(out, [&](auto* tp) {
          using Id = std::remove_cv_t<std::remove_pointer_t<decltype(idp)>>;
          using Grad = std::remove_pointer_t<decltype(gp)>;
          using T = std::remove_pointer_t<decltype(tp)>;
          const float s = static_cast<float>(scale);
          if (vec) embed_few_kernel<sizeof(Grad) == 4 ? 4 : 8, Grad, T, Id><<<grid, 256, 0, st>>>(idp, gp, tp, static_cast<int>(n), V, static_cast<int>(C), s);
          else embed_few_kernel<1, Grad, T, Id><<<grid, 256, 0, st>>>(idp, gp, tp, static_cast<int>(n), V, static_cast<int>(C), s);
        });
      });
    });
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return out;
  }
  const int64_t most = std::min<int64_t>(n, kSortCapacity);
  const int64_t most_pieces = (most + kPiece - 1) / kPiece;
  auto work = torch::empty({most_pieces * 2 * C + 2 * most}, f32);  // partial sums, keys, positions
  float* partial = work.data_ptr<float>();
  unsigned* keys = reinterpret_cast<unsigned*>(partial + most_pieces * 2 * C);
  int* pos = reinterpret_cast<int*>(keys + most);
  int bits = 1;
  while (bits < 32 && (V >> bits) != 0) ++bits;  // the value V itself stands for tokens outside the table
  const int64_t packs = vec ? C / N : C;
  const int threads = static_cast<int>(std::min<int64_t>(256, (packs + 31) / 32 * 32));
  const int64_t slices = (packs + threads - 1) / threads;
  TORCH_CHECK(slices <= 65535, "embedding: rows too wide");
  for (int64_t i0 = 0; i0 < n; i0 += kSortCapacity) {
    const int count = static_cast<int>(std::min<int64_t>(kSortCapacity, n - i0));
    const int64_t bytes = i0 == 0 ? out.numel() * out.element_size() : 0, vecs = bytes / 16;
    const int per = count <= kSortCtas * kSortThreads ? 1 : count <= 2 * kSortCtas * kSortThreads ? 2 : count <= 4 * kSortCtas * kSortThreads ? 4 : 8;
    with_ids(ids, [&](auto* idp) {
      using Id = std::remove_cv_t<std::remove_pointer_t<decltype(idp)>>;
      auto sort = [&](auto kPer) {
        auto* kernel = embed_sort_kernel<decltype(kPer)::value, Id>;
        const size_t smem = sort_smem(decltype(kPer)::value);
        const int zero_ctas = static_cast<int>(std::min<int64_t>(clusters_at_once(kernel, smem) - 1, (bytes + 8 * kZeroBytes - 1) / (8 * kZeroBytes))) * kSortCtas;
        kernel<<<kSortCtas + zero_ctas, kSortThreads, smem, st>>>(
            idp + i0, count, V, bits, keys, pos,
            reinterpret_cast<uint4*>(out.data_ptr()), vecs, reinterpret_cast<unsigned char*>(out.data_ptr()) + vecs * 16, static_cast<int>(bytes - vecs * 16));
      };
      if (per == 1) sort(std::integral_constant<int, 1>{});
      else if (per == 2) sort(std::integral_constant<int, 2>{});
      else if (per == 4) sort(std::integral_constant<int, 4>{});
      else sort(std::integral_constant<int, 8>{});
    });
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    const int pieces = (count + kPiece - 1) / kPiece;
    with_type(dy, [&](auto* gp) {
      with_type(out, [&](auto* tp) {
        using Grad = std::remove_pointer_t<decltype(gp)>;
        using T = std::remove_pointer_t<decltype(tp)>;
        constexpr int kN = sizeof(Grad) == 4 ? 4 : 8;
        const dim3 grid(pieces, static_cast<unsigned>(slices));
        const dim3 join_grid(pieces, static_cast<unsigned>(std::min<int64_t>((C + 511) / 512, 64)));
        auto go = [&](auto add) {
          constexpr bool kAdd = decltype(add)::value;
          auto* g = gp + i0 * C;
          const int c = static_cast<int>(C);
          const auto v = static_cast<unsigned>(V);
          const float s = static_cast<float>(scale);
          if (vec) embed_pieces_kernel<kN, Grad, T, kAdd><<<grid, threads, 0, st>>>(keys, pos, g, tp, partial, count, v, c, s);
          else embed_pieces_kernel<1, Grad, T, kAdd><<<grid, threads, 0, st>>>(keys, pos, g, tp, partial, count, v, c, s);
          C10_CUDA_KERNEL_LAUNCH_CHECK();
          if (pieces > 1) embed_join_kernel<T, kAdd><<<join_grid, 32 * kJoinRows, 0, st>>>(keys, partial, tp, count, v, c, s);
          C10_CUDA_KERNEL_LAUNCH_CHECK();
        };
        if (i0 == 0) go(std::false_type{});
        else go(std::true_type{});
      });
    });
  }
  return out_bf16 && sliced ? out.to(torch::kBFloat16) : out;
}

// Kernels that embed_bwd launches for `tokens` tokens.
int64_t embed_bwd_launches(int64_t tokens) {
  if (tokens <= kFewTokens) return tokens > 0;
  int64_t n = 0;
  for (int64_t i0 = 0; i0 < tokens; i0 += kSortCapacity) n += tokens - i0 > kPiece ? 3 : 2;
  return n;
}

void register_embed_ops(pybind11::module_& m) {
  m.def("embed_fwd", &embed_fwd);
  m.def("embed_bwd", &embed_bwd);
}

}  // namespace ob200
