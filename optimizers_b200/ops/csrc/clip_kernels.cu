// Norm over many gradients and their scaling by one factor, in two launches and without a table upload.
//
//   grad_sumsq   per-CTA sums of squares over all gradients (fp32, bf16, fp16, any alignment)
//   clip_scale   norm = sqrt(sum of those), factor = min(1, max_norm / (norm + 1e-6)), g <- factor * g
//
// The table of gradients (pointer, length, first chunk) travels as a kernel parameter: gradients have new addresses after
// every `zero_grad(set_to_none=True)`, so a table in device memory would need a copy in front of each call.  A gradient is seen
// as 16-byte vectors counted from the aligned address at or below its start; only its first and last vector are taken apart.
//
// A CTA owns a fixed, contiguous range of chunks and adds in a fixed order, and every CTA of the second launch adds the partial
// sums in the same order, so the norm does not depend on scheduling.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <algorithm>
#include <unordered_set>

namespace ob200 {
namespace {

constexpr int kClipThreads = 512;
constexpr int kChunkBytes = 32768;  // of one gradient, per turn of a CTA
constexpr int kChunkVecs = kChunkBytes / 16;

// Up to kMax gradients; the largest table is just below the 32764 bytes that kernel parameters may take.
template <int kMax>
struct GradTable {
  uintptr_t ptr[kMax];
  long long numel[kMax];
  int first_chunk[kMax + 1];
  unsigned char kind[kMax];  // 0 fp32, 1 bf16, 2 fp16
  int count;
};

__device__ __forceinline__ float block_sum(float v) {
  __shared__ float parts[kClipThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = threadIdx.x < kClipThreads / 32 ? parts[threadIdx.x] : 0.f;
  if (threadIdx.x < 32) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (threadIdx.x == 0) parts[0] = t;
  }
  __syncthreads();
  return parts[0];
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(x);
  else return __half2float(x);
}
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(x);
  else return __float2half_rn(x);
}

template <typename T>
__device__ __forceinline__ float square_of(const uint4& u) {
  const T* e = reinterpret_cast<const T*>(&u);
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < static_cast<int>(16 / sizeof(T)); ++k) {
    const float x = to_float(e[k]);
    s = fmaf(x, x, s);
  }
  return s;
}

// Runs body(T{}, vec0, vec1, head, total, base) for the chunks of this CTA's range, forwards or backwards.  Vectors [vec0, vec1)
// of the gradient at `base` (16-byte aligned); elements [head, total) in units counted from `base` exist.
template <int kMax, bool kBackward, typename Body>
__device__ __forceinline__ void for_each_chunk(const GradTable<kMax>& t, Body&& body) {
  const int chunks = t.first_chunk[t.count];
  int c0 = static_cast<int>(static_cast<long long>(chunks) * blockIdx.x / gridDim.x);
  int c1 = static_cast<int>(static_cast<long long>(chunks) * (blockIdx.x + 1) / gridDim.x);
  if (c0 >= c1) return;
  int lo = 0, hi = t.count - 1;  // the gradient of the first chunk to visit
  const int first = kBackward ? c1 - 1 : c0;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first_chunk[mid] <= first) lo = mid;
    else hi = mid - 1;
  }
  int at = lo;
  for (int i = 0; i < c1 - c0; ++i) {
    const int c = kBackward ? c1 - 1 - i : c0 + i;
    if (kBackward) {
      while (t.first_chunk[at] > c) --at;
    } else {
      while (t.first_chunk[at + 1] <= c) ++at;
    }
    const uintptr_t ptr = t.ptr[at], base = ptr & ~uintptr_t(15);
    const int kind = t.kind[at];
    const int shift = kind == 0 ? 2 : 1;
    const long long head = static_cast<long long>(ptr - base) >> shift, total = head + t.numel[at];
    const long long vecs = (total + (16 >> shift) - 1) >> (4 - shift);
    const long long v0 = static_cast<long long>(c - t.first_chunk[at]) * kChunkVecs;
    const long long v1 = v0 + kChunkVecs < vecs ? v0 + kChunkVecs : vecs;
    if (kind == 0) body(float{}, base, v0, v1, head, total);
    else if (kind == 1) body(__nv_bfloat16{}, base, v0, v1, head, total);
    else body(__half{}, base, v0, v1, head, total);
  }
}

// Bound by HBM.  Four 16-byte loads in flight per thread: 4 CTAs of 512 threads keep 128 KB per SM under way.  333M fp32 values: 218 us, 6.1 TB/s.
template <int kMax>
__global__ void __launch_bounds__(kClipThreads)
grad_sumsq_kernel(const __grid_constant__ GradTable<kMax> table, float* __restrict__ partial) {
  float sum = 0.f;
  for_each_chunk<kMax, false>(table, [&](auto tag, uintptr_t base, long long v0, long long v1, long long head, long long total) {
    using T = decltype(tag);
    constexpr int kPer = 16 / sizeof(T);
    const uint4* src = reinterpret_cast<const uint4*>(base);
    const T* elems = reinterpret_cast<const T*>(base);
    auto one = [&](long long v) {
      if (v * kPer >= head && (v + 1) * kPer <= total) return square_of<T>(src[v]);
      float s = 0.f;
      for (int k = 0; k < kPer; ++k) {
        const long long e = v * kPer + k;
        if (e >= head && e < total) {
          const float x = to_float(elems[e]);
          s = fmaf(x, x, s);
        }
      }
      return s;
    };
    if (v1 - v0 == kChunkVecs && v0 * kPer >= head && v1 * kPer <= total) {
      static_assert(kChunkVecs == 4 * kClipThreads, "a whole chunk is four vectors per thread");
      const uint4* p = src + v0 + threadIdx.x;
      const uint4 a = p[0], b = p[kClipThreads], c = p[2 * kClipThreads], d = p[3 * kClipThreads];
      sum += (square_of<T>(a) + square_of<T>(b)) + (square_of<T>(c) + square_of<T>(d));
    } else {
      for (long long v = v0 + threadIdx.x; v < v1; v += kClipThreads) sum += one(v);
    }
  });
  const float total = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// Walks each CTA's range backwards: what the first launch read last is still in the L2.  A factor of one leaves the gradients alone.  333M fp32
// values: 454 us, 5.9 TB/s.
template <int kMax>
__global__ void __launch_bounds__(kClipThreads)
clip_scale_kernel(const __grid_constant__ GradTable<kMax> table, const float* __restrict__ partial, int num_partial, float max_norm,
                  float* __restrict__ norm_out) {
  float sum = 0.f;
  for (int i = threadIdx.x; i < num_partial; i += kClipThreads) sum += partial[i];
  const float norm = sqrtf(block_sum(sum));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) *norm_out = norm;
  const float ratio = max_norm / (norm + 1e-6f);
  const float factor = ratio > 1.f ? 1.f : ratio;  // a NaN stays one
  if (factor == 1.f) return;
  for_each_chunk<kMax, true>(table, [&](auto tag, uintptr_t base, long long v0, long long v1, long long head, long long total) {
    using T = decltype(tag);
    constexpr int kPer = 16 / sizeof(T);
    uint4* vecs = reinterpret_cast<uint4*>(base);
    T* elems = reinterpret_cast<T*>(base);
    auto scaled = [&](uint4 u) {
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int k = 0; k < kPer; ++k) e[k] = from_float<T>(to_float(e[k]) * factor);
      return u;
    };
    if (v1 - v0 == kChunkVecs && v0 * kPer >= head && v1 * kPer <= total) {
      uint4* p = vecs + v0 + threadIdx.x;
      const uint4 a = p[0], b = p[kClipThreads], c = p[2 * kClipThreads], d = p[3 * kClipThreads];
      p[0] = scaled(a);
      p[kClipThreads] = scaled(b);
      p[2 * kClipThreads] = scaled(c);
      p[3 * kClipThreads] = scaled(d);
    } else {
      for (long long v = v0 + threadIdx.x; v < v1; v += kClipThreads) {
        if (v * kPer >= head && (v + 1) * kPer <= total) {
          vecs[v] = scaled(vecs[v]);
        } else {
          for (int k = 0; k < kPer; ++k) {
            const long long e = v * kPer + k;
            if (e >= head && e < total) elems[e] = from_float<T>(to_float(elems[e]) * factor);
          }
        }
      }
    }
  });
}

constexpr int kTableSizes[3] = {32, 180, 1500};
static_assert(sizeof(GradTable<1500>) + 64 <= 32764, "kernel parameters take at most 32764 bytes");
static_assert(sizeof(GradTable<180>) + 64 <= 4096, "the middle size stays below 4 KB");

struct GradSpan {
  uintptr_t ptr;
  long long numel;
  int kind;
};

std::vector<GradSpan> spans_of(const std::vector<torch::Tensor>& grads) {
  std::vector<GradSpan> spans;
  spans.reserve(grads.size());
  for (const auto& g : grads) {
    const auto st = g.scalar_type();
    TORCH_CHECK(g.is_cuda() && g.device() == grads[0].device(), "clip: gradients are CUDA tensors on one device");
    TORCH_CHECK(st == torch::kFloat32 || st == torch::kBFloat16 || st == torch::kFloat16, "clip: gradients are fp32, bf16 or fp16");
    TORCH_CHECK(g.is_non_overlapping_and_dense(), "clip: gradients fill their memory without gaps or overlaps");
    if (g.numel() == 0) continue;
    spans.push_back({reinterpret_cast<uintptr_t>(g.data_ptr()), static_cast<long long>(g.numel()),
                     st == torch::kFloat32 ? 0 : st == torch::kBFloat16 ? 1 : 2});
  }
  return spans;
}

void check_disjoint(std::vector<GradSpan> spans) {
  std::sort(spans.begin(), spans.end(), [](const GradSpan& a, const GradSpan& b) { return a.ptr < b.ptr; });
  for (size_t i = 1; i < spans.size(); ++i) {
    const auto& p = spans[i - 1];
    TORCH_CHECK_VALUE(p.ptr + static_cast<uintptr_t>(p.numel) * (p.kind == 0 ? 4 : 2) <= spans[i].ptr,
                      "clip: two gradients share memory; each value can be scaled once only");
  }
}

template <int kMax>
GradTable<kMax> fill(const GradSpan* spans, int count) {
  GradTable<kMax> t;
  t.count = count;
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    t.ptr[i] = spans[i].ptr;
    t.numel[i] = spans[i].numel;
    t.kind[i] = static_cast<unsigned char>(spans[i].kind);
    t.first_chunk[i] = static_cast<int>(chunks);
    const int size = spans[i].kind == 0 ? 4 : 2;
    const long long bytes = static_cast<long long>(spans[i].ptr & 15) + spans[i].numel * size;
    chunks += (bytes + kChunkBytes - 1) / kChunkBytes;
  }
  TORCH_CHECK(chunks < (1LL << 31), "clip: gradients too large");
  t.first_chunk[count] = static_cast<int>(chunks);
  return t;
}

// Calls launch(table, grid, batch) for the gradients in tables of the smallest size that holds them.
template <typename Launch>
void in_tables(const std::vector<GradSpan>& spans, Launch&& launch) {
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int n = static_cast<int>(spans.size());
  for (int at = 0, batch = 0; at < n; ++batch) {
    const int left = n - at;
    auto go = [&](auto size) {
      constexpr int kMax = decltype(size)::value;
      const int count = std::min(left, kMax);
      const auto table = fill<kMax>(spans.data() + at, count);
      launch(table, std::min(4 * sms, table.first_chunk[count]), batch);
      at += count;
    };
    if (left <= kTableSizes[0]) go(std::integral_constant<int, kTableSizes[0]>{});
    else if (left <= kTableSizes[1]) go(std::integral_constant<int, kTableSizes[1]>{});
    else go(std::integral_constant<int, kTableSizes[2]>{});
  }
}

}  // namespace

// Sums of squares of the gradients, to be added up: fp32 [k].
torch::Tensor grad_sumsq(const std::vector<torch::Tensor>& grads, bool disjoint) {
  TORCH_CHECK(!grads.empty(), "clip: no gradients");
  c10::cuda::CUDAGuard guard(grads[0].device());
  const auto spans = spans_of(grads);
  if (disjoint) check_disjoint(spans);
  const auto f32 = grads[0].options().dtype(torch::kFloat32);
  if (spans.empty()) return torch::zeros({1}, f32);
  int total = 0;
  in_tables(spans, [&](const auto&, int grid, int) { total += grid; });
  auto partial = torch::empty({total}, f32);
  auto st = at::cuda::getCurrentCUDAStream();
  int at = 0;
  in_tables(spans, [&](const auto& table, int grid, int) {
    grad_sumsq_kernel<<<grid, kClipThreads, 0, st>>>(table, partial.data_ptr<float>() + at);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    at += grid;
  });
  return partial;
}

// Scales the gradients by min(1, max_norm / (norm + 1e-6)) where norm^2 is the sum over `partial`; returns the norm.
torch::Tensor clip_scale(const std::vector<torch::Tensor>& grads, const torch::Tensor& partial, double max_norm) {
  TORCH_CHECK(!grads.empty(), "clip: no gradients");
  TORCH_CHECK(partial.device() == grads[0].device() && partial.scalar_type() == torch::kFloat32 && partial.is_contiguous() && partial.numel() > 0,
              "clip: sums are fp32 on the gradients' device");
  c10::cuda::CUDAGuard guard(grads[0].device());
  const auto spans = spans_of(grads);
  auto norm = torch::empty({}, partial.options());
  if (spans.empty()) return norm.copy_(partial.sum().sqrt());
  auto st = at::cuda::getCurrentCUDAStream();
  in_tables(spans, [&](const auto& table, int grid, int batch) {
    clip_scale_kernel<<<grid, kClipThreads, 0, st>>>(table, partial.data_ptr<float>(), static_cast<int>(partial.numel()),
                                                     static_cast<float>(max_norm), batch == 0 ? norm.data_ptr<float>() : nullptr);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  for (const auto& g : grads)  // written in place: whoever saved one for a backward pass has to learn of it
    if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
  return norm;
}

// The whole call for the usual case, without a pass over the gradients in Python: every gradient on one sm_100 device, of these
// types, filling its memory.  None otherwise, and where there is no gradient.
std::optional<torch::Tensor> clip_parameters(const std::vector<torch::Tensor>& parameters, double max_norm) {
  std::vector<torch::Tensor> grads;
  std::unordered_set<const void*> seen;
  grads.reserve(parameters.size());
  for (const auto& p : parameters) {
    if (!p.defined() || !p.is_leaf()) return std::nullopt;
    const auto& g = p.grad();
    if (!g.defined() || !seen.insert(p.unsafeGetTensorImpl()).second) continue;
    const auto st = g.scalar_type();
    if (g.unsafeGetTensorImpl()->is_python_dispatch() || g.layout() != torch::kStrided || !g.is_cuda() ||
        (st != torch::kFloat32 && st != torch::kBFloat16 && st != torch::kFloat16) || !g.is_non_overlapping_and_dense() ||
        (!grads.empty() && g.device() != grads[0].device()))
      return std::nullopt;
    grads.push_back(g);
  }
  if (grads.empty() || at::cuda::getDeviceProperties(grads[0].device().index())->major != 10) return std::nullopt;
  return clip_scale(grads, grad_sumsq(grads, true), max_norm);
}

void register_clip_ops(pybind11::module_& m) {
  m.def("grad_sumsq", &grad_sumsq);
  m.def("clip_scale", &clip_scale);
  m.def("clip_parameters", &clip_parameters);
}

}  // namespace ob200
