// kv_cache.cu - the 8-bit key/value cache: quantising packed rows into paged
// blocks as they are written, and reading rows back as values.
//
// A CTA owns one touched block of one kv head and side (key or value), so a
// block's scale has a single writer and needs no atomics: it holds the
// block's new values in registers, reduces their largest magnitude, settles
// the scale and stores the codes. The block's earlier codes are loaded only
// when the scale grew.
//
// Bound for prompts by HBM (values in, one byte a value out) and as much by the
// issue of instructions (88% and 81% of the slots): 57,560 tokens of 8 heads of
// 128 in bf16 81 us to write, 4.4 TB/s, and 71 to read back, 5.0 (128 threads a
// block, for fewer warps to set up, 136 and 74). Single tokens are bound by
// latency (length, page, scale and value loads in a row: 64 sequences, 8 heads,
// 3.4 us).
#include "kv_util.cuh"

#include <algorithm>

namespace cim {
namespace {

constexpr int kThreads = 256;

// rint(x * inverse) within +-127; NaN gives 0.
__device__ __forceinline__ int quantise(float x, float inverse) {
  const float q = fminf(fmaxf(rintf(__fmul_rn(x, inverse)), -127.0f), 127.0f);
  return x == x ? static_cast<int>(q) : 0;
}

// The largest magnitude's bits so far, with a vector's (an infinity or NaN is
// above every finite value's), in the words that max_bits takes them from.
__device__ __forceinline__ uint32_t max_bits(uint32_t top, const Pack<float> &p) {
  top = max(max(top, p.raw.x & 0x7fffffffu), p.raw.y & 0x7fffffffu);
  return max(max(top, p.raw.z & 0x7fffffffu), p.raw.w & 0x7fffffffu);
}
template <typename T> __device__ __forceinline__ uint32_t max_bits(uint32_t top, const Pack<T> &p) {
  top = __vimax3_u16x2(top, p.raw.x & 0x7fff7fffu, p.raw.y & 0x7fff7fffu);
  return __vimax3_u16x2(top, p.raw.z & 0x7fff7fffu, p.raw.w & 0x7fff7fffu);
}
template <typename T> __device__ __forceinline__ float magnitude(uint32_t top) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(top);
  } else {
    const uint16_t most = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    return to_f32(*reinterpret_cast<const T *>(&most));
  }
}

// Codes of four values that the scale covers: |x * inverse| is below 127.5, so
// 1.5 * 2^23 more is rounded to an integer whose low byte is the code.
__device__ __forceinline__ uint32_t quantise4(const float *x, float inverse) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inverse), 12582912.0f));
  return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}

// Four codes as f32: code + 128 as the low byte of 2^23 + u.
__device__ __forceinline__ void code_values(uint32_t codes, float *y) {
  codes ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    y[i] = __uint_as_float(__byte_perm(codes, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
}

template <typename T> struct Codes; // kVec<T> codes
template <> struct Codes<float> {
  using type = uint32_t;
};
template <> struct Codes<__nv_bfloat16> {
  using type = uint2;
};
template <> struct Codes<__half> {
  using type = uint2;
};

struct Rows {
  const void *at;
  int64_t row_stride, head_stride;
};

template <typename T, int kPer>
__global__ void __launch_bounds__(kThreads)
    kv_write_kernel(const KvView v, const Rows keys, const Rows values, const FastDiv parts,
                    int32_t *status) {
  constexpr int V = kVec<T>;
  using C = typename Codes<T>::type;
  __shared__ float top[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  // Neighbouring CTAs take the heads and sides of one block: their rows are
  // neighbours in memory.
  const int b = blockIdx.y, planes = 2 * v.heads, touch = blockIdx.x / planes;
  const int plane = blockIdx.x - touch * planes, head = plane >> 1, side = plane & 1;
  const KvSequence s = kv_sequence(v, b);
  if (!s.ok) {
    if (threadIdx.x == 0 && blockIdx.x == 0)
      atomicOr(status, CIM22_STATUS_CACHE_INDEX);
    return;
  }
  const int begin = max(0, s.length - s.n);
  const int ordinal = (begin >> v.block_log2) + touch;
  const int64_t base = static_cast<int64_t>(ordinal) << v.block_log2;
  if (begin >= s.length || base >= s.length)
    return;
  const int lo = static_cast<int>(max(static_cast<int64_t>(begin), base) - base);
  const int hi = static_cast<int>(min(static_cast<int64_t>(s.length) - base,
                                      static_cast<int64_t>(1) << v.block_log2));
  // Row of the block's token 0 (may lie before the sequence's rows; only
  // tokens lo .. hi - 1 are followed).
  const int64_t row = s.row0 + base - (static_cast<int64_t>(s.length) - s.n);
  const T *rows = side ? static_cast<const T *>(values.at) + head * values.head_stride
                       : static_cast<const T *>(keys.at) + head * keys.head_stride;
  const int64_t stride = side ? values.row_stride : keys.row_stride;
  const int chunks = (hi - lo) * parts.d;

  Pack<T> x[kPer];
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int c = p * blockDim.x + threadIdx.x;
    if (c < chunks) {
      const int i = fdiv(c, parts);
      x[p] = load_pack(rows + (row + lo + i) * stride, (c - i * parts.d) * V, v.dim);
    }
  }
  // The page is looked up while the values are on their way.
  const int page = kv_page(v, b, ordinal);
  if (page < 0) {
    if (threadIdx.x == 0)
      atomicOr(status, CIM22_STATUS_CACHE_INDEX);
    return;
  }
  float *scale_at = v.scales + (static_cast<int64_t>(page) * v.heads + head) * 2 + side;
  const float old = lo > 0 ? *scale_at : 0.0f;
  uint32_t bits = 0;
#pragma unroll
  for (int p = 0; p < kPer; ++p)
    bits = max_bits(bits, x[p]);
  float amax = magnitude<T>(bits);
  // Also orders every thread's read of the old scale before the new store.
  const bool wild = __syncthreads_or(!(amax < INFINITY));
  if (wild) { // the largest of the finite ones
    amax = 0.0f;
#pragma unroll
    for (int p = 0; p < kPer; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float m = fabsf(to_f32(x[p].at[i]));
        amax = m < INFINITY ? fmaxf(amax, m) : amax;
      }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0)
    top[threadIdx.x >> 5] = amax;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w)
    amax = fmaxf(amax, top[w]);
  const float scale = fmaxf(old, __fmul_rn(fmaxf(amax, kKvFloor), kKvInv127));
  const float inverse = __frcp_rn(scale);
  if (threadIdx.x == 0) {
    *scale_at = scale;
    if (wild)
      atomicOr(status, CIM22_STATUS_CACHE_NOT_FINITE);
  }
  int8_t *codes = kv_codes(v, page, head, side);
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int c = p * blockDim.x + threadIdx.x;
    if (c < chunks) {
      union {
        C raw;
        int8_t at[V];
        uint32_t words[V / 4];
      } q;
      float y[V];
      unpack(x[p], y);
      if (wild) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          q.at[i] = static_cast<int8_t>(quantise(y[i], inverse));
      } else {
#pragma unroll
        for (int i = 0; i < V; i += 4)
          q.words[i / 4] = quantise4(y + i, inverse);
      }
      *reinterpret_cast<C *>(codes + lo * v.dim + c * V) = q.raw;
    }
  }
  if (scale > old && lo > 0) {
    uint4 *earlier = reinterpret_cast<uint4 *>(codes);
    for (int c = threadIdx.x; c < lo * v.dim / 16; c += blockDim.x) {
      union {
        uint4 raw;
        int8_t at[16];
      } q;
      q.raw = earlier[c];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        q.at[i] = static_cast<int8_t>(quantise(__fmul_rn(static_cast<float>(q.at[i]), old), inverse));
      earlier[c] = q.raw;
    }
  }
}

// Rows of one plane, dim elements each, shared by `ctas` CTAs. Out of line: few
// calls have such rows, and within the kernel it took 10 registers more.
template <typename T>
__device__ __noinline__ void zero_rows(T *rows, int count, int dim, int64_t stride, int cta, int ctas) {
  const Pack<T> none;
  const int parts = dim / kVec<T>;
  for (int64_t c = static_cast<int64_t>(cta) * kThreads + threadIdx.x;
       c < static_cast<int64_t>(count) * parts; c += static_cast<int64_t>(ctas) * kThreads) {
    const int64_t i = c / parts;
    store_pack(rows + i * stride, (c - i * parts) * kVec<T>, dim, none);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    kv_read_kernel(const KvView v, T *__restrict__ k, T *__restrict__ values, const FastDiv parts,
                   int32_t *status) {
  constexpr int V = kVec<T>;
  using C = typename Codes<T>::type;
  pdl_launch_dependents();
  pdl_wait();
  // Neighbouring CTAs take the heads and sides of one block: their rows are
  // neighbours in memory.
  const int b = blockIdx.y, planes = 2 * v.heads, touch = blockIdx.x / planes;
  const int plane = blockIdx.x - touch * planes, head = plane >> 1, side = plane & 1;
  T *out = side ? values : k;
  const KvSequence s = kv_sequence(v, b);
  if (!s.ok) {
    if (threadIdx.x == 0 && blockIdx.x == 0)
      atomicOr(status, CIM22_STATUS_CACHE_INDEX);
    return;
  }
  if (!out)
    return;
  const int64_t stride = static_cast<int64_t>(v.heads) * v.dim;
  const int before = s.n - s.length; // rows before the sequence's start
  if (before > 0)                    // are zeros; the plane's CTAs share them
    zero_rows(out + s.row0 * stride + head * v.dim, before, v.dim, stride, touch,
              gridDim.x / planes);
  const int begin = max(0, s.length - s.n);
  const int ordinal = (begin >> v.block_log2) + touch;
  const int64_t base = static_cast<int64_t>(ordinal) << v.block_log2;
  if (begin >= s.length || base >= s.length)
    return;
  const int page = kv_page(v, b, ordinal);
  if (page < 0) {
    if (threadIdx.x == 0)
      atomicOr(status, CIM22_STATUS_CACHE_INDEX);
    return;
  }
  const int lo = static_cast<int>(max(static_cast<int64_t>(begin), base) - base);
  const int hi = static_cast<int>(min(static_cast<int64_t>(s.length) - base,
                                      static_cast<int64_t>(1) << v.block_log2));
  const int64_t row = s.row0 + base - (static_cast<int64_t>(s.length) - s.n);
  const float scale = v.scales[(static_cast<int64_t>(page) * v.heads + head) * 2 + side];
  const int8_t *codes = kv_codes(v, page, head, side) + lo * v.dim;
  const int chunks = (hi - lo) * parts.d;
  T *to = out + (row + lo) * stride + head * v.dim;
  const bool aligned = (reinterpret_cast<uintptr_t>(to) & 15) == 0; // rows are whole vectors
  constexpr int kUnroll = 4;
  for (int c0 = threadIdx.x; c0 < chunks; c0 += kUnroll * kThreads) {
    union {
      C raw;
      uint32_t words[V / 4];
    } q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (c0 + u * kThreads < chunks)
        q[u].raw = *reinterpret_cast<const C *>(codes + (c0 + u * kThreads) * V);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int c = c0 + u * kThreads;
      if (c < chunks) {
        const int i = fdiv(c, parts);
        float y[V];
#pragma unroll
        for (int j = 0; j < V; j += 4)
          code_values(q[u].words[j / 4], y + j);
#pragma unroll
        for (int j = 0; j < V; ++j)
          y[j] = __fmul_rn(y[j], scale);
        Pack<T> o;
        pack(y, o);
        T *at = to + i * stride + (c - i * parts.d) * V;
        if (aligned)
          *reinterpret_cast<uint4 *>(at) = o.raw;
        else
          store_pack(at, 0, V, o);
      }
    }
  }
}

// CTAs for the heads and sides of the blocks that a sequence's rows can touch.
int64_t planes_touched(const KvView &v) {
  const int block = 1 << v.block_log2;
  const int64_t most = std::min<int64_t>(v.most, static_cast<int64_t>(v.table_width) * block);
  const int64_t touched = std::min<int64_t>((most + 2 * block - 2) / block, v.table_width);
  return std::max<int64_t>(1, touched) * v.heads * 2;
}

bool too_many(const char *what, const KvView &v) {
  if (planes_touched(v) <= 0x7fffffff)
    return false;
  set_last_error(std::string(what) + ": too many rows a sequence for one call");
  return true;
}

template <typename T>
cudaError_t launch_write(const KvView &v, const Rows &keys, const Rows &values, int32_t *status,
                         cudaStream_t stream) {
  const int parts = v.dim / kVec<T>;
  const int chunks = std::min(v.most, 1 << v.block_log2) * parts;
  const int threads = std::min<int>(kThreads, std::max<int>(128, static_cast<int>(round_up(chunks, 32))));
  const int per = (chunks + threads - 1) / threads;
  const auto kernel = per <= 1 ? kv_write_kernel<T, 1>
                      : per <= 2 ? kv_write_kernel<T, 2>
                      : per <= 4 ? kv_write_kernel<T, 4>
                      : per <= 8 ? kv_write_kernel<T, 8>
                                 : kv_write_kernel<T, 128 * 128 / kVec<T> / kThreads>;
  return launch_pdl(kernel, dim3(static_cast<unsigned>(planes_touched(v)), v.batch), dim3(threads), 0, stream, v,
                    keys, values, make_fastdiv(parts), status);
}

template <typename T>
cudaError_t launch_read(const KvView &v, void *k, void *values, int32_t *status,
                        cudaStream_t stream) {
  return launch_pdl(kv_read_kernel<T>, dim3(static_cast<unsigned>(planes_touched(v)), v.batch), dim3(kThreads), 0,
                    stream, v, static_cast<T *>(k), static_cast<T *>(values),
                    make_fastdiv(v.dim / kVec<T>), status);
}

} // namespace
} // namespace cim

using namespace cim;

extern "C" {

int cim22_cuda_kv_write(const cim22_kv_cache *cache, const cim22_kv_sequences *sequences,
                        int32_t type, const void *k, int64_t k_row_stride, int64_t k_head_stride,
                        const void *v, int64_t v_row_stride, int64_t v_head_stride,
                        int32_t *status, void *stream) {
  const int bad = CIM22_STATUS_BAD_ARGUMENT;
  KvView view;
  if (!kv_view("cim22_cuda_kv_write", cache, sequences, view))
    return bad;
  if (!float_type(type) || !status || (view.rows > 0 && (!k || !v))) {
    set_last_error("cim22_cuda_kv_write: null rows or status, or unknown type");
    return bad;
  }
  if (k_row_stride < 0 || v_row_stride < 0 || k_head_stride < 0 || v_head_stride < 0) {
    set_last_error("cim22_cuda_kv_write: strides must not be negative");
    return bad;
  }
  if (view.batch == 0 || view.rows == 0)
    return 0;
  if (too_many("cim22_cuda_kv_write", view))
    return bad;
  const Rows keys{k, k_row_stride, k_head_stride}, values{v, v_row_stride, v_head_stride};
  const auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = type == CIM22_FLOAT32    ? launch_write<float>(view, keys, values, status, s)
                        : type == CIM22_BFLOAT16 ? launch_write<__nv_bfloat16>(view, keys, values, status, s)
                                                 : launch_write<__half>(view, keys, values, status, s);
  return cuda_ok(e, "kv_write") ? 0 : bad;
}

int cim22_cuda_kv_read(const cim22_kv_cache *cache, const cim22_kv_sequences *sequences,
                       int32_t type, void *k, void *v, int32_t *status, void *stream) {
  const int bad = CIM22_STATUS_BAD_ARGUMENT;
  KvView view;
  if (!kv_view("cim22_cuda_kv_read", cache, sequences, view))
    return bad;
  if (!float_type(type) || !status) {
    set_last_error("cim22_cuda_kv_read: null status or unknown type");
    return bad;
  }
  if (view.batch == 0 || view.rows == 0 || (!k && !v))
    return 0;
  if (too_many("cim22_cuda_kv_read", view))
    return bad;
  const auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = type == CIM22_FLOAT32    ? launch_read<float>(view, k, v, status, s)
                        : type == CIM22_BFLOAT16 ? launch_read<__nv_bfloat16>(view, k, v, status, s)
                                                 : launch_read<__half>(view, k, v, status, s);
  return cuda_ok(e, "kv_read") ? 0 : bad;
}

} // extern "C"
