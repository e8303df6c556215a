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

// A vector as f32, and back (each element rounded to nearest even).
__device__ __forceinline__ void unpack(const Pack<float> &p, float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = p.at[i];
}
__device__ __forceinline__ void unpack(const Pack<__nv_bfloat16> &p, float (&x)[8]) {
  const uint32_t w[4] = {p.raw.x, p.raw.y, p.raw.z, p.raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const Pack<__half> &p, float (&x)[8]) {
  const uint32_t w[4] = {p.raw.x, p.raw.y, p.raw.z, p.raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void pack(const float (&x)[4], Pack<float> &p) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p.at[i] = x[i];
}
__device__ __forceinline__ void pack(const float (&x)[8], Pack<__nv_bfloat16> &p) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  p.raw = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(const float (&x)[8], Pack<__half> &p) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  p.raw = make_uint4(w[0], w[1], w[2], w[3]);
}

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
