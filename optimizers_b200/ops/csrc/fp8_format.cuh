// The 8-bit format of the decoder's products: e4m3 values with one fp32 scale per group.
//
// For the largest magnitude a of a group (at least 1e-30, so that its reciprocal stays finite) the scale is a / 448 and a value x
// is held as e4m3(x * (448 / a)); each of these is rounded to fp32, the last step to nearest even.  Magnitudes are compared as
// integers: the bit pattern of a NaN is above that of infinity, so a NaN in a group makes its scale, and all products of the group, NaN;
// an infinity makes the scale infinite and the products NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <cstdint>
#include <type_traits>

namespace ob200 {

constexpr int kFp8Group = 128;

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct GroupScale {
  float factor;  // 448 / a
  float scale;   // a / 448
};

__device__ __forceinline__ GroupScale group_scale(uint32_t top_bits) {
  const float a = __uint_as_float(max(top_bits, __float_as_uint(1e-30f)));
  return {__fdiv_rn(448.f, a), __fdiv_rn(a, 448.f)};
}

// Four values as e4m3 bytes, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float factor) {
  return make_uint2(e4m3x4(__fmul_rn(v[0], factor), __fmul_rn(v[1], factor), __fmul_rn(v[2], factor), __fmul_rn(v[3], factor)),
                    e4m3x4(__fmul_rn(v[4], factor), __fmul_rn(v[5], factor), __fmul_rn(v[6], factor), __fmul_rn(v[7], factor)));
}

// Eight consecutive values from column `col` of a row of `cols`: one or two 16-byte loads where kVec (then cols % 8 == 0 and the
// row is 16-byte aligned), else one by one; columns that do not exist are 0.
template <bool kVec, typename T>
__device__ __forceinline__ void load8(const T* row, int col, int cols, float (&v)[8]) {
  if constexpr (kVec) {
    if (col >= cols) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.f;
    } else if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + col), b = *reinterpret_cast<const float4*>(row + col + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(row + col);
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 t = __bfloat1622float2(h[k]);
        v[2 * k] = t.x;
        v[2 * k + 1] = t.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (sizeof(T) == 4) v[k] = col + k < cols ? row[col + k] : 0.f;
      else v[k] = col + k < cols ? __bfloat162float(row[col + k]) : 0.f;
    }
  }
}

template <bool kVec, typename T>
__device__ __forceinline__ void store8(T* row, int col, int cols, const float (&v)[8]) {
  if constexpr (kVec) {
    if (col >= cols) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + col) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(row + col + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 u;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
      *reinterpret_cast<uint4*>(row + col) = u;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (col + k >= cols) continue;
      if constexpr (sizeof(T) == 4) row[col + k] = v[k];
      else row[col + k] = __float2bfloat16_rn(v[k]);
    }
  }
}

}  // namespace ob200
