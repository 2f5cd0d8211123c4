// Residual addition + RMSNorm.
//
//   add_norm_fwd   h = x + r (rounded to r's type), y = h * rsqrt(mean h^2 + eps) * w, in fp32 or bf16, or in e4m3 with an fp32 scale
//                  per 128 columns; also 1 / rms per row for the backward pass
//   add_norm_bwd   dh + rs * (dy w - z mean(dy w z)) with z = h rs, written in the types of x and of r, and dw = sum over rows of dy z
//
// A row belongs to `tpr` threads (a multiple of 32), each with eight neighbouring columns out of every 8 * tpr: a warp reads 512 or 1024
// bytes in a row, sixteen lanes hold one group of 128 columns, and a thread keeps its columns from row to row, so that the
// backward pass adds dw in registers.  Both are bound by HBM: 16384 x 2048, bf16 x and an fp32 residual, 76 us (5.3 TB/s) forward and 111 us (4.8
// TB/s) backward, which reads h again.  Rows off the 16-byte grid are loaded value by value and take 1.5 times as long.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "fp8_format.cuh"

namespace ob200 {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kMaxNormWidth = 16384;
enum NormOut { kOutF32 = 0, kOutBf16 = 1, kOutFp8 = 2 };

// Sum over the threads of a row, for every row of the CTA.  `parts` has a word per warp; all threads of the CTA take part.
__device__ __forceinline__ float row_sum(float v, float* parts, int warps_per_row) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps_per_row == 1) return v;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) parts[warp] = v;
  __syncthreads();
  const int first = warp / warps_per_row * warps_per_row;
  float s = 0.f;
  for (int w = 0; w < warps_per_row; ++w) s += parts[first + w];
  __syncthreads();
  return s;
}

template <bool kVec>
__device__ __forceinline__ void load_weight(const void* w, bool w_bf16, int col, int C, float (&v)[8]) {
  if (w_bf16) load8<kVec>(static_cast<const bf16*>(w), col, C, v);
  else load8<kVec>(static_cast<const float*>(w), col, C, v);
}

struct NormFwdArgs {
  const void *x, *r, *w;
  void *h, *y;
  float *rstd, *scale;
  long long rows;
  int C, tpr, out, ld_fp8;
  bool w_bf16;
  float eps;
};

template <typename X, typename R, int kVecs, int kThreads, bool kVec>
__global__ void __launch_bounds__(kThreads) add_norm_fwd_kernel(const NormFwdArgs a) {
  __shared__ float parts[32];
  const int t = threadIdx.x % a.tpr, C = a.C;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / a.tpr) + threadIdx.x / a.tpr;
  const bool live = row < a.rows;  // every thread takes part in the sums
  const long long at = (live ? row : 0) * C;
  float h[kVecs][8];
  float sq = 0.f;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int col = (v * a.tpr + t) * 8;
    load8<kVec>(static_cast<const X*>(a.x) + at, col, C, h[v]);
    if (a.r != nullptr) {
      float r[8];
      load8<kVec>(static_cast<const R*>(a.r) + at, col, C, r);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        h[v][k] += r[k];
        if constexpr (sizeof(R) == 2) h[v][k] = __bfloat162float(__float2bfloat16_rn(h[v][k]));
      }
      if (live) store8<kVec>(static_cast<R*>(a.h) + at, col, C, h[v]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sq = fmaf(h[v][k], h[v][k], sq);
  }
  const float rs = rsqrtf(row_sum(sq, parts, a.tpr / 32) / static_cast<float>(C) + a.eps);
  if (live && t == 0 && a.rstd != nullptr) a.rstd[row] = rs;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int col = (v * a.tpr + t) * 8;
    float w[8];
    load_weight<kVec>(a.w, a.w_bf16, col, C, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[v][k] = h[v][k] * rs * w[k];
    if (a.out == kOutFp8) {
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, magnitude_bits(h[v][k]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const GroupScale g = group_scale(top);
      if (live && col < C) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.y) + row * a.ld_fp8 + col) = e4m3x8(h[v], g.factor);  // the pitch is a multiple of 16
        if ((t & 15) == 0) a.scale[static_cast<long long>(col / kFp8Group) * a.rows + row] = g.scale;
      }
    } else if (live) {
      if (a.out == kOutBf16) store8<kVec>(static_cast<bf16*>(a.y) + at, col, C, h[v]);
      else store8<kVec>(static_cast<float*>(a.y) + at, col, C, h[v]);
    }
  }
}

struct NormBwdArgs {
  const void *dy, *dh, *h, *w;
  const float* rstd;
  void *dx, *dr;
  float* partial;
  long long rows;
  int C, tpr;
  bool dy_bf16, w_bf16;
};

// Persistent: a CTA takes every gridDim-th set of rows and leaves one row of dw in partial[cta].
template <typename X, typename R, int kVecs, int kThreads, bool kVec>
__global__ void __launch_bounds__(kThreads) add_norm_bwd_kernel(const NormBwdArgs a) {
  __shared__ float parts[32];
  extern __shared__ float sums[];  // [rows of the CTA - 1][C]
  const int t = threadIdx.x % a.tpr, own = threadIdx.x / a.tpr, C = a.C;
  const int per_cta = blockDim.x / a.tpr;
  float dw[kVecs][8];
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[v][k] = 0.f;
  for (long long row0 = static_cast<long long>(blockIdx.x) * per_cta; row0 < a.rows; row0 += static_cast<long long>(gridDim.x) * per_cta) {
    const long long row = row0 + own;
    const bool live = row < a.rows;
    const long long at = (live ? row : 0) * C;
    const float rs = live ? a.rstd[row] : 0.f;
    float z[kVecs][8], g[kVecs][8];
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int col = (v * a.tpr + t) * 8;
      float w[8];
      load8<kVec>(static_cast<const R*>(a.h) + at, col, C, z[v]);
      if (a.dy_bf16) load8<kVec>(static_cast<const bf16*>(a.dy) + at, col, C, g[v]);
      else load8<kVec>(static_cast<const float*>(a.dy) + at, col, C, g[v]);
      load_weight<kVec>(a.w, a.w_bf16, col, C, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        z[v][k] *= rs;
        if (live) dw[v][k] = fmaf(g[v][k], z[v][k], dw[v][k]);
        g[v][k] *= w[k];
        dot = fmaf(g[v][k], z[v][k], dot);
      }
    }
    const float mean = row_sum(dot, parts, a.tpr / 32) / static_cast<float>(C);
    if (!live) continue;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int col = (v * a.tpr + t) * 8;
      float o[8];
      if (a.dh != nullptr) load8<kVec>(static_cast<const R*>(a.dh) + at, col, C, o);
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = (a.dh != nullptr ? o[k] : 0.f) + rs * (g[v][k] - z[v][k] * mean);
      store8<kVec>(static_cast<X*>(a.dx) + at, col, C, o);
      if (a.dr != nullptr) store8<kVec>(static_cast<R*>(a.dr) + at, col, C, o);
    }
  }
  if (own > 0) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) store8<false>(sums + static_cast<long long>(own - 1) * C, (v * a.tpr + t) * 8, C, dw[v]);
  }
  __syncthreads();
  if (own > 0) return;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int col = (v * a.tpr + t) * 8;
    for (int r = 0; r + 1 < per_cta; ++r) {
      float s[8];
      load8<false>(sums + static_cast<long long>(r) * C, col, C, s);
#pragma unroll
      for (int k = 0; k < 8; ++k) dw[v][k] += s[k];
    }
    store8<false>(a.partial + static_cast<long long>(blockIdx.x) * C, col, C, dw[v]);
  }
}

// out[c] = sum over r of partial[r][c]: 32 columns per CTA, eight warps take every eighth row, then the eight sums in order.
template <typename T>
__global__ void __launch_bounds__(256) sum_partial_kernel(const float* __restrict__ partial, T* __restrict__ out, int rows, int C) {
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < C)
    for (int r = warp; r < rows; r += 8) s += partial[static_cast<long long>(r) * C + c];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < C) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += sums[w][lane];
    if constexpr (sizeof(T) == 4) out[c] = t;
    else out[c] = __float2bfloat16_rn(t);
  }
}

struct NormShape {
  int tpr, vecs, per_cta;
};

// Threads per row: one per eight columns up to 4096, one per sixteen beyond; rows share a CTA of about 256 threads.  The backward pass keeps
// to eight up to 8192: it holds three arrays per column, and with sixteen columns a thread only 512 threads fit on an SM (4096 x 8192: 136 us
// instead of 156).  The forward pass is faster with two CTAs of 512 than with one of 1024 (76 us instead of 117).
NormShape norm_shape(int64_t C, bool backward) {
  const int packs = static_cast<int>((C + 7) / 8);
  const int vecs = packs <= (backward ? 1024 : 512) ? 1 : 2;
  const int tpr = std::max(32, (packs + 32 * vecs - 1) / (32 * vecs) * 32);
  return {tpr, vecs, std::max(1, 256 / tpr)};
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool is_bf16(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16; }
bool fp32_or_bf16(const torch::Tensor& t) { return t.scalar_type() == torch::kFloat32 || is_bf16(t); }

void check_rows(const torch::Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1 && x.is_contiguous() && fp32_or_bf16(x), "add_norm: ", what, " is a contiguous fp32 or bf16 CUDA tensor");
  TORCH_CHECK(x.size(-1) > 0 && x.size(-1) <= kMaxNormWidth, "add_norm: rows have 1 to ", kMaxNormWidth, " columns");
}
void check_like(const torch::Tensor& t, const torch::Tensor& x, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device() && t.is_contiguous() && fp32_or_bf16(t) && t.sizes() == x.sizes(), "add_norm: ", what, " is fp32 or bf16, of x's shape");
}
void check_weight(const torch::Tensor& w, const torch::Tensor& x) {
  TORCH_CHECK(w.device() == x.device() && w.dim() == 1 && w.is_contiguous() && fp32_or_bf16(w) && w.numel() == x.size(-1), "add_norm: the weight is fp32 or bf16 [C]");
}

template <typename F>
void with_types(bool x_bf16, bool r_bf16, F&& f) {
  if (x_bf16 && r_bf16) f(bf16{}, bf16{});
  else if (x_bf16) f(bf16{}, float{});
  else f(float{}, float{});
}
template <int kVecsOf, int kThreadsOf>
struct Shape {
  static constexpr int kVecs = kVecsOf, kThreads = kThreadsOf;
};
template <typename F>
void with_shape(const NormShape& s, bool vec, F&& f) {
  auto go = [&](auto shape) {
    if (vec) f(shape, std::true_type{});
    else f(shape, std::false_type{});
  };
  if (s.vecs == 1 && s.tpr <= 512) go(Shape<1, 512>{});
  else if (s.vecs == 1) go(Shape<1, 1024>{});
  else if (s.tpr <= 512) go(Shape<2, 512>{});
  else go(Shape<2, 1024>{});
}

}  // namespace

// x, r [..., C] (r may be absent; fp32 x with bf16 r is not offered) -> (y, scale, h, rstd).  out: 0 fp32, 1 bf16, 2 e4m3 (uint8, rows at a
// pitch of a multiple of 16 bytes) with scale [groups, rows].  h is empty where r is absent (it is x then).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> add_norm_fwd(const torch::Tensor& x, const std::optional<torch::Tensor>& r,
                                                                                    const torch::Tensor& w, double eps, int64_t out, bool want_rstd) {
  check_rows(x, "x");
  check_weight(w, x);
  if (r.has_value()) check_like(*r, x, "the residual");
  TORCH_CHECK(!r.has_value() || is_bf16(x) || !is_bf16(*r), "add_norm: an fp32 x needs an fp32 residual");
  TORCH_CHECK(out >= 0 && out <= 2, "add_norm: output format");
  const int64_t C = x.size(-1), rows = x.numel() / C;
  c10::cuda::CUDAGuard guard(x.device());
  const auto opt = x.options();
  const int64_t pitch = (C + 15) / 16 * 16, groups = (C + kFp8Group - 1) / kFp8Group;
  auto y = out == kOutFp8 ? torch::empty({rows, pitch}, opt.dtype(torch::kUInt8)) : torch::empty(x.sizes(), opt.dtype(out == kOutBf16 ? torch::kBFloat16 : torch::kFloat32));
  auto scale = torch::empty({out == kOutFp8 ? groups : 0, rows}, opt.dtype(torch::kFloat32));
  auto h = r.has_value() ? torch::empty_like(*r) : torch::empty({0}, opt);
  auto rstd = torch::empty({want_rstd ? rows : 0}, opt.dtype(torch::kFloat32));
  if (rows == 0) return {y, scale, h, rstd};
  const NormShape s = norm_shape(C, false);
  const bool vec = C % 8 == 0 && aligned16(w.data_ptr()) && aligned16(x.data_ptr()) && (!r.has_value() || aligned16(r->data_ptr()));
  const NormFwdArgs args{x.data_ptr(), r.has_value() ? r->data_ptr() : nullptr, w.data_ptr(), r.has_value() ? h.data_ptr() : nullptr, y.data_ptr(),
                         want_rstd ? rstd.data_ptr<float>() : nullptr, scale.data_ptr<float>(), rows, static_cast<int>(C), s.tpr, static_cast<int>(out),
                         static_cast<int>(pitch), is_bf16(w), static_cast<float>(eps)};
  const int64_t grid = (rows + s.per_cta - 1) / s.per_cta;
  TORCH_CHECK(grid < (1LL << 31), "add_norm: too many rows");
  auto st = at::cuda::getCurrentCUDAStream();
  with_types(is_bf16(x), r.has_value() ? is_bf16(*r) : is_bf16(x), [&](auto xt, auto rt) {
    with_shape(s, vec, [&](auto shape, auto kvec) {
      add_norm_fwd_kernel<decltype(xt), decltype(rt), decltype(shape)::kVecs, decltype(shape)::kThreads, decltype(kvec)::value>
          <<<static_cast<unsigned>(grid), s.tpr * s.per_cta, 0, st>>>(args);
    });
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {y, scale, h, rstd};
}

// -> (dx in x's type, dr in h's type or empty, dw in the weight's type)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> add_norm_bwd(const torch::Tensor& dy, const std::optional<torch::Tensor>& dh, const torch::Tensor& h,
                                                                     const torch::Tensor& w, const torch::Tensor& rstd, bool dx_bf16, bool want_dr) {
  check_rows(h, "h");
  check_weight(w, h);
  check_like(dy, h, "dy");
  if (dh.has_value()) {
    check_like(*dh, h, "dh");
    TORCH_CHECK(dh->scalar_type() == h.scalar_type(), "add_norm: dh has h's type");
  }
  const int64_t C = h.size(-1), rows = h.numel() / C;
  TORCH_CHECK(rstd.device() == h.device() && rstd.scalar_type() == torch::kFloat32 && rstd.is_contiguous() && rstd.numel() == rows, "add_norm: rstd fp32 [rows]");
  TORCH_CHECK(dx_bf16 || !is_bf16(h), "add_norm: an fp32 x has an fp32 h");
  c10::cuda::CUDAGuard guard(h.device());
  auto dx = torch::empty(h.sizes(), h.options().dtype(dx_bf16 ? torch::kBFloat16 : torch::kFloat32));
  auto dr = want_dr ? torch::empty_like(h) : torch::empty({0}, h.options());
  auto dw = torch::empty({C}, w.options());
  if (rows == 0) return {dx, dr, dw.zero_()};
  const NormShape s = norm_shape(C, true);
  const bool vec = C % 8 == 0 && aligned16(w.data_ptr()) && aligned16(h.data_ptr()) && aligned16(dy.data_ptr()) && (!dh.has_value() || aligned16(dh->data_ptr()));
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int threads = s.tpr * s.per_cta;
  const int64_t sets = (rows + s.per_cta - 1) / s.per_cta;
  const int grid = static_cast<int>(std::min<int64_t>(sets, static_cast<int64_t>(sms) * std::max(1, 1024 / threads)));
  auto partial = torch::empty({grid, C}, h.options().dtype(torch::kFloat32));
  const NormBwdArgs args{dy.data_ptr(), dh.has_value() ? dh->data_ptr() : nullptr, h.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dx.data_ptr(),
                         want_dr ? dr.data_ptr() : nullptr, partial.data_ptr<float>(), rows, static_cast<int>(C), s.tpr, is_bf16(dy), is_bf16(w)};
  const size_t smem = static_cast<size_t>(s.per_cta - 1) * C * 4;  // below 8 KB: rows share a CTA up to 1024 columns
  auto st = at::cuda::getCurrentCUDAStream();
  with_types(dx_bf16, is_bf16(h), [&](auto xt, auto rt) {
    with_shape(s, vec, [&](auto shape, auto kvec) {
      add_norm_bwd_kernel<decltype(xt), decltype(rt), decltype(shape)::kVecs, decltype(shape)::kThreads, decltype(kvec)::value><<<grid, threads, smem, st>>>(args);
    });
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  const unsigned sum_grid = static_cast<unsigned>((C + 31) / 32);
  if (is_bf16(w)) sum_partial_kernel<bf16><<<sum_grid, 256, 0, st>>>(partial.data_ptr<float>(), static_cast<bf16*>(dw.data_ptr()), grid, static_cast<int>(C));
  else sum_partial_kernel<float><<<sum_grid, 256, 0, st>>>(partial.data_ptr<float>(), dw.data_ptr<float>(), grid, static_cast<int>(C));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dx, dr, dw};
}

void register_residual_norm_ops(pybind11::module_& m) {
  m.def("add_norm_fwd", &add_norm_fwd);
  m.def("add_norm_bwd", &add_norm_bwd);
}

}  // namespace ob200
