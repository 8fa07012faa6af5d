// Device helpers of the 8-bit KV cache kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv8.h"
#include "sm100_async.cuh"

namespace qb {
namespace kv8 {

template <int kType>
struct TypeOf;
template <>
struct TypeOf<0> {
  using T = float;
};
template <>
struct TypeOf<1> {
  using T = __half;
};
template <>
struct TypeOf<2> {
  using T = __nv_bfloat16;
};

template <typename T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<__nv_bfloat16> = true;

__device__ __forceinline__ void bad_index() { atomicOr(&g_kernel_error, kErrBadIndex); }

// Four consecutive values as they lie in memory, and as fp32. The entry points check the alignment (16 or 8 bytes).
__device__ __forceinline__ float4 raw4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
template <typename T>
__device__ __forceinline__ uint2 raw4(const T* p) {
  return __ldg(reinterpret_cast<const uint2*>(p));
}
template <typename T>
__device__ __forceinline__ float4 expand(float4 b) {
  return b;
}
template <typename T>
__device__ __forceinline__ float4 expand(uint2 b) {
  if (sizeof(T) == 2 && !kIsBf16<T>) {
    const float2 lo = __half22float2(reinterpret_cast<const __half2&>(b.x));
    const float2 hi = __half22float2(reinterpret_cast<const __half2&>(b.y));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
  }
  return make_float4(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                     __uint_as_float(b.y & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  return expand<T>(raw4(p));
}

// The rounding to the caller's type: the one rounding of a value that was computed in fp32.
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__half* p, float4 v) {
  uint2 b;
  reinterpret_cast<__half2&>(b.x) = __floats2half2_rn(v.x, v.y);
  reinterpret_cast<__half2&>(b.y) = __floats2half2_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = b;
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  uint2 b;
  reinterpret_cast<__nv_bfloat162&>(b.x) = __floats2bfloat162_rn(v.x, v.y);
  reinterpret_cast<__nv_bfloat162&>(b.y) = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = b;
}

// The same for values that are not read again soon: evicted first, the cache keeps what is (reading 8 x 4096 rows back:
// 17.6 us without, 16.9 us with).
__device__ __forceinline__ void stream4(float* p, float4 v) { __stcs(reinterpret_cast<float4*>(p), v); }
template <typename T>
__device__ __forceinline__ void stream4(T* p, float4 v) {
  __align__(8) T four[4];
  store4(four, v);
  __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(four));
}

}  // namespace kv8
}  // namespace qb
