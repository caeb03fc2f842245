// Wave-level pieces shared by the attention kernels (device code).
#pragma once

#include "common.h"

namespace yapd {

__device__ __forceinline__ u32x4_t load16(const uint16_t* p) {
  return *reinterpret_cast<const u32x4_t*>(p);
}

// K/V pages are streamed once per step: non-temporal loads keep them from
// evicting the q / K / V lines the QKV GEMM has just written, whose
// write-back would otherwise land in the middle of this stream (measured
// 195 -> 179 us per layer right after the QKV GEMM).
__device__ __forceinline__ u32x4_t load16_stream(const uint16_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
}

// Lane l combined with lane l ^ 16 (l ^ 32): v_permlane16_swap (32_swap) of a
// value with itself returns the two halves of every exchanged pair, so the
// max or sum of its two results is the pair's in both lanes -- a VALU
// exchange instead of an LDS permute.
__device__ __forceinline__ float2 swap16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 swap32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor16_32(float v) {
  const float2 a = swap16(v);
  const float2 b = swap32(fmaxf(a.x, a.y));
  return fmaxf(b.x, b.y);
}
__device__ __forceinline__ float sum_xor16_32(float v) {
  const float2 a = swap16(v);
  const float2 b = swap32(a.x + a.y);
  return b.x + b.y;
}

}  // namespace yapd
