// Pieces shared by the kernels over a paged key/value cache.
//
// Pages `k`, `v` [pages, page_size, kv_heads, D] hold the stream type, or e4m3 beside one
// power of two a token and head (`k_scale`, `v_scale` [pages, kv_heads, page_size], e8m0:
// code c stands for 2^(c - 127), 255 for NaN). A power of two costs e4m3 nothing but its
// smallest values, and multiplying by it rounds nothing where the stream type has the product:
// there, what attention computes with and what is read back are the same numbers in every path.
// f16 alone has products that it rounds (its subnormals) where keys and values are widened; the
// few-row kernel takes them as they are. Products beyond a type's largest number: `in_range`.
#pragma once

#include <cuda_fp8.h>
#include <float.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged_split.cuh"

namespace svodb {
namespace paged {

__device__ __forceinline__ Row row_of(const int32_t* start, const int32_t* lens, int64_t b, int64_t t, int64_t capacity) {
  Row r;
  r.start = start != nullptr ? start[b] : 0;
  int64_t n = t;
  if (lens != nullptr) {
    const int64_t l = lens[b];
    n = l < 0 ? 0 : (l < t ? l : t);
  }
  r.bad = n > 0 && (r.start < 0 || r.start + n > capacity);
  r.n = r.bad ? 0 : (int)n;
  return r;
}

// The e8m0 code of 2^e, the least power of two with amax <= 448 * 2^e: 448 = 1.75 * 2^8, so
// the exponent of amax less 8, and one more where its significand is above 1.75. Zeros, and
// rows too small for the least code, have code 0 (2^-127); a row that is not finite has the NaN code.
__device__ __forceinline__ uint32_t scale_code(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits >= 0x7f800000u) return 255u;
  const int code = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return code < 0 ? 0u : (uint32_t)code;
}
// 2^(code - 127): code 0 is below the normal numbers, code 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t code) {
  return code == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(code == 0u ? 0x00400000u : code << 23);
}
// 2^(127 - code) for the codes `scale_code` gives to finite rows (0 .. 247): 2^127 at most.
__device__ __forceinline__ float scale_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t u) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)u, __NV_E4M3);
  return __half22float2(__half2(h));
}

// A page's value in the stream type's range. e4m3 rounds the topmost values of a type past its
// largest number (f16: 63488 and more to 256 * 2^8 = 65536), which then stands for them: a row
// that was finite reads back finite, half a step off at most. NaN stays.
template <typename T>
constexpr float kLargest = std::is_same<T, __half>::value ? 65504.f : std::is_same<T, float>::value ? FLT_MAX : 0x1.fep127f;
template <typename T>
__device__ __forceinline__ float in_range(float x) {
  return fabsf(x) > kLargest<T> ? copysignf(kLargest<T>, x) : x;
}

// The same for a pair on its way into the type, in the conversion itself.
template <typename T>
__device__ __forceinline__ uint32_t pack_in_range(float lo, float hi) {
  uint32_t u;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  return u;
}

// n / d for 0 <= n < 2^31 without a division: (floor(n m / 2^32) + n) >> shift with
// m = floor(2^32 (2^shift - d) / d) + 1, 2^shift >= d (Granlund and Montgomery's method).
struct Divider {
  uint32_t d, m, shift;
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> shift; }
};
inline Divider divider(uint32_t d) {
  Divider v{d, 0, 0};
  while ((1ull << v.shift) < d) ++v.shift;
  v.m = (uint32_t)(((1ull << 32) * ((1ull << v.shift) - d)) / d + 1);
  return v;
}

}  // namespace paged
}  // namespace svodb
