// kv_attention.h - what the attention kernels over the 8-bit cache share.
#pragma once

#include "kv_util.cuh"

#include <atomic>

namespace cim {

struct KvAttendArgs {
  KvView v;
  const void *q;
  int64_t q_row_stride, q_head_stride;
  bool q_aligned; // every row starts on a 16-byte boundary
  void *out;
  float *lse;
  float scale_log2; // softmax scale * log2(e)
  int q_heads, group, causal, window;
  int splits;     // parts of the key axis,
  int cluster;    // so many neighbouring ones joined within the kernel
  float *part_o;   // [splits / cluster][rows * q_heads][dim], relative to 2^m,
  float2 *part_ml; // [splits / cluster][rows * q_heads] (m, l), when not one
  // For prompts of f32 queries, or null: what each stream has taken out of its
  // accumulators, [splits][2][kv_heads][64 or 128][rows * group].
  float *carry;
  int32_t *status;
};

// The tensor-memory kernel for prompts (kv_attention_tc.cu).
cudaError_t kv_prompt_launch(const KvAttendArgs &a, int type, bool share, int tiles,
                             cudaStream_t stream);

// Allows a kernel its dynamic shared memory, once for each device.
class DynamicSmem {
public:
  template <typename K> cudaError_t allow(K kernel, size_t bytes) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && done_.load() >> device & 1))
      return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(bytes));
    if (e == cudaSuccess && device < 64)
      done_.fetch_or(uint64_t{1} << device);
    return e;
  }

private:
  std::atomic<uint64_t> done_{0};
};

#if defined(__CUDACC__)
namespace {

// Softmax over values held as codes with a scale for each block. With
// t = score * log2(e) + log2(value scale of the key's block), m a running
// reference near max t, p = 2^(t - m):
//   out = sum_j p_j * code_j / l,   l = sum_j p_j / value_scale_j,
// so the products take the codes alone (exact in f16), p needs no range
// beyond its own maximum, and one multiply a block scales l.
// l does need more. Value scales reach from 2^-87 (a block of zeros) to 2^121,
// and where they lie far apart a key of much weight has a p below f32's range,
// although its part of l, 2^(score - m), is within it. Blocks whose scale is
// below 2^-kApart times the largest one met therefore carry 0 in place of 1 /
// value_scale, and their weights are computed by themselves, relative to their
// own largest. What p loses of the others weighs at most 2^(kApart - 126) of the
// largest weight a key. (A block of zeros beside values of up to 16 is not that
// far apart.)
// Value scales below kKvLeastScale count as it (the writer's least one).
constexpr float kApart = 84.0f;
constexpr float kKvLeastScale = 0x1p-87f;
// p is kept at most 2^kTop when the reference is set and may grow to 2^kGrowth
// before it is set again: the largest is then a power of two, which f16 does not
// round (with whole references one key of much weight in 200,000 was, and
// outputs were off by 3.8e-4, not 2.0e-4, of which 2.0e-4 are their own). f16 (largest 65504, steps of 2^-24) then
// holds every p to within 2^-11 of itself or 2^-31 of the largest; with two
// parts (f32 queries), which set it again sooner, to within 2^-22 or 2^-38.
// kNone: the reference of a row that has seen no key.
constexpr float kNone = -1e30f;
// One part costs f16 outputs some accuracy, since l takes the probabilities
// unrounded: 2.7e-4 against 64 bits, not 2.1e-4, where many keys share the weight
// (chunks of 1,024, window 4,096); bf16 outputs none (1.7e-3 both). Two parts
// would double the second product.
template <int kParts> constexpr float kTop = kParts == 2 ? 13.0f : 6.0f;
template <int kParts> constexpr float kGrowth = kParts == 2 ? 15.0f : 14.0f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// l * 2^(a - b) of a sum of weights. Between far references 2^(a - b) alone may
// lie below f32's range, and a - b rounds: their whole and broken parts are
// then subtracted apart. Near ones take the factor that the outputs take.
__device__ __forceinline__ float weigh(float l, float a, float b) {
  if (fabsf(a - b) < 16.0f)
    return l * exp2_approx(a - b);
  const float d = rintf(a) - rintf(b);
  l *= exp2_approx((a - rintf(a)) - (b - rintf(b)));
  return d > -100.0f ? l * exp2_approx(d) : l * 0x1p-100f * exp2_approx(d + 100.0f);
}

__device__ __forceinline__ float nan_max(float a, float b) { // a NaN stays
  return b > a || b != b ? b : a;
}

// The first key within the window of a row at position p, which may lie far
// before the sequence's start: p - window need not fit 32 bits.
__device__ __forceinline__ int window_start(int window, int p) {
  return window > 0 && p >= window ? p - window + 1 : 0;
}

// The range of keys [lo, hi) that rows at positions p0 .. p1 can see.
__device__ __forceinline__ void key_range(const KvAttendArgs &a, int length, int p0, int p1,
                                          int &lo, int &hi) {
  hi = a.causal ? min(length, p1 + 1) : length;
  lo = window_start(a.window, p0);
  if (hi < lo)
    hi = lo;
}

__device__ __forceinline__ bool sees(const KvAttendArgs &a, int length, int p, int key) {
  return key < length && (!a.causal || key <= p) && key >= window_start(a.window, p);
}

// Power-of-two factor 2^(141 - E) that brings a row whose largest magnitude
// has biased exponent E to [2^14, 2^15), so that its f16 parts keep every
// element to within 2^-39 of the largest, and the factor's inverse.
__device__ __forceinline__ void row_factor(float amax, float &factor, float &inverse) {
  const int e = min(max((__float_as_int(amax) >> 23) & 255, 15), 254);
  factor = amax == 0.0f ? 1.0f : __int_as_float((268 - e) << 23);
  inverse = amax == 0.0f ? 1.0f : __int_as_float((e - 14) << 23);
}

// Four int8 codes as two f16 pairs, exactly: code + 128 as the low byte of
// 1024 + u, less 1152.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
  w ^= 0x80808080u;
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), bias);
  const __half2 y = __hsub2(*reinterpret_cast<__half2 *>(&b), bias);
  lo = *reinterpret_cast<const uint32_t *>(&x);
  hi = *reinterpret_cast<const uint32_t *>(&y);
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float2 unpack_half(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

} // namespace
#endif

} // namespace cim
