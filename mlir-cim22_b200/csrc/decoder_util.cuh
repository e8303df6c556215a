// decoder_util.cuh - what the decoder-block kernels (block norm, 8-bit
// key/value cache, attention over it) share: the activation types and vector
// access to rows whose start need not lie on a vector boundary.
#pragma once

#include "cim_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace cim {

inline bool float_type(int32_t t) {
  return t == CIM22_FLOAT32 || t == CIM22_BFLOAT16 || t == CIM22_FLOAT16;
}
inline int64_t float_size(int32_t t) { return t == CIM22_FLOAT32 ? 4 : 2; }

#if defined(__CUDACC__)
namespace {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Rounded to nearest even, half a step of T at most.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// Elements of a 16-byte vector.
template <typename T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <typename T> union Pack {
  uint4 raw;
  T at[kVec<T>];
  __device__ Pack() : raw(make_uint4(0, 0, 0, 0)) {}
};

// Elements e .. e + kVec - 1 of a row of `count` elements (those outside it
// read as zero): one 16-byte load where they lie on such a boundary.
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T *row, int64_t e, int64_t count) {
  Pack<T> p;
  const T *at = row + e;
  if (e >= 0 && e + kVec<T> <= count && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
    p.raw = __ldg(reinterpret_cast<const uint4 *>(at));
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (e + i >= 0 && e + i < count)
        p.at[i] = at[i];
  }
  return p;
}

template <typename T>
__device__ __forceinline__ void store_pack(T *row, int64_t e, int64_t count, const Pack<T> &p) {
  T *at = row + e;
  if (e >= 0 && e + kVec<T> <= count && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
    *reinterpret_cast<uint4 *>(at) = p.raw;
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (e + i >= 0 && e + i < count)
        at[i] = p.at[i];
  }
}

} // namespace
#endif

} // namespace cim
