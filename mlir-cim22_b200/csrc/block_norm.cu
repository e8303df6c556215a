// block_norm.cu - the norms before and after a decoder block with the block's
// gate and residual add between them, one pass over the data:
//
//   h = residual_scale * residual + act(gate) * post(x)      (stored as T)
//   y = pre(h)                                               (stored as T)
//
// post / pre: RMS norm v / sqrt(mean(v^2) + eps) * w (+ b) or layer norm
// (v - mean) / sqrt(mean((v - mean)^2) + eps) * w (+ b), over the row. All
// arithmetic is f32; pre reads h before it is rounded to T, so y carries one
// rounding only.
//
// Bound by HBM (x and residual read once, h and y written once): a row stays
// in registers between the reductions, kPer 16-byte vectors a thread, W warps
// a row.
#include "decoder_util.cuh"

#include <algorithm>
#include <atomic>

namespace cim {
namespace {

struct NormArg {
  int kind; // CIM22_NORM_*
  float eps;
  const void *weight, *bias;
  int type; // of weight and bias
};

struct BlockNormArgs {
  const void *x, *residual, *gate;
  void *h, *y;
  int64_t rows, dim, x_stride, residual_stride, gate_stride, h_stride, y_stride;
  int64_t gate_rows; // consecutive rows that share a gate row
  int type, gate_type, gate_columns, gate_act;
  float residual_scale;
  NormArg post, pre;
  int warps_log2; // warps a row, log2
};

__device__ __forceinline__ float gate_fn(float g, int act) {
  if (act == CIM22_GATE_SIGMOID)
    return 1.0f / (1.0f + expf(-g));
  if (act == CIM22_GATE_TANH)
    return tanhf(g);
  return g;
}

// Sum over the W warps of a row; `slot` alternates so that one barrier a
// reduction is enough.
__device__ __forceinline__ float row_sum(float v, int warps_log2, float *buffer, int &slot) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps_log2 == 0)
    return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *part = buffer + 32 * slot;
  slot ^= 1;
  if (lane == 0)
    part[warp] = v;
  __syncthreads();
  const int w = 1 << warps_log2;
  v = lane < w ? part[(warp & ~(w - 1)) + lane] : 0.0f;
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rows off vector boundaries, several to a CTA where they are narrow. A warp's
// loads and stores take 32 neighbouring elements (lanes that each took their
// own eight spread every weight load over eight lines: 3,001 x 1,001 f16, 31 us
// against 19). Bound by the issue of 2-byte accesses: 20,000 x 1,001 f16 with a
// gate value an element 98 us, 2.05 TB/s.
template <typename T, int kPer, int kMax>
__global__ void __launch_bounds__(kMax) block_norm_kernel(const BlockNormArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float buffer[64];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w = 1 << a.warps_log2, part = warp & (w - 1);
  const int64_t row_at = static_cast<int64_t>(blockIdx.x) * ((blockDim.x >> 5) >> a.warps_log2) +
                         (warp >> a.warps_log2);
  const bool live = row_at < a.rows;
  const int64_t row = live ? row_at : a.rows - 1; // every thread reaches the barriers
  const int dim = static_cast<int>(a.dim);
  const float inverse = 1.0f / static_cast<float>(dim);
  int slot = 0;
  // The thread's element i of its p-th group.
  auto at = [&](int p, int i) { return ((p * w + part) * V + i) * 32 + lane; };
  auto load = [&](const T *from, int p, float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      x[i] = at(p, i) < dim ? to_f32(from[at(p, i)]) : 0.0f;
  };
  auto load_weights = [&](const void *from, int type, int p, float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = at(p, i);
      x[i] = 0.0f;
      if (e < dim)
        x[i] = type == CIM22_FLOAT32 ? static_cast<const float *>(from)[e]
                                     : to_f32(static_cast<const T *>(from)[e]);
    }
  };

  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  float v[kPer][V], res[kPer][V];
#pragma unroll
  for (int p = 0; p < kPer; ++p)
    load(x, p, v[p]);
  if (a.residual) {
    const T *residual = static_cast<const T *>(a.residual) + row * a.residual_stride;
#pragma unroll
    for (int p = 0; p < kPer; ++p)
      load(residual, p, res[p]);
  }

  // A gate row of x's type is on its way while post reduces.
  T gates[kPer][V];
  const bool early = a.gate && a.gate_columns != 1 && a.gate_type == a.type;
  if (early) {
    const T *gate = static_cast<const T *>(a.gate) + (a.gate_rows ? row / a.gate_rows * a.gate_stride : 0);
#pragma unroll
    for (int p = 0; p < kPer; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at(p, i) < dim)
          gates[p][i] = gate[at(p, i)];
  }

  auto normalise = [&](const NormArg &n) {
    float mean = 0.0f, s = 0.0f;
    if (n.kind == CIM22_NORM_LAYER) {
#pragma unroll
      for (int p = 0; p < kPer; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i)
          s += v[p][i]; // zero outside the row
      mean = row_sum(s, a.warps_log2, buffer, slot) * inverse;
      s = 0.0f;
    }
#pragma unroll
    for (int p = 0; p < kPer; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[p][i] = at(p, i) < dim ? v[p][i] - mean : 0.0f;
        s = fmaf(v[p][i], v[p][i], s);
      }
    const float scale = rsqrtf(row_sum(s, a.warps_log2, buffer, slot) * inverse + n.eps);
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      float g[V];
      if (n.weight) {
        load_weights(n.weight, n.type, p, g);
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] *= scale * g[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] *= scale;
      }
      if (n.bias) {
        load_weights(n.bias, n.type, p, g);
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] += g[i];
      }
    }
  };

  if (a.post.kind != CIM22_NORM_NONE)
    normalise(a.post);
  if (a.gate) {
    const int64_t from = a.gate_rows ? row / a.gate_rows * a.gate_stride : 0;
    const char *gate = static_cast<const char *>(a.gate) + from * (a.gate_type == CIM22_FLOAT32 ? 4 : 2);
    if (a.gate_columns == 1) {
      const float g = gate_fn(a.gate_type == CIM22_FLOAT32 ? *reinterpret_cast<const float *>(gate)
                                                           : to_f32(*reinterpret_cast<const T *>(gate)),
                              a.gate_act);
#pragma unroll
      for (int p = 0; p < kPer; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] *= g;
    } else {
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        float g[V];
        if (early) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            g[i] = at(p, i) < dim ? to_f32(gates[p][i]) : 0.0f;
        } else {
          load_weights(gate, a.gate_type, p, g);
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] *= gate_fn(g[i], a.gate_act);
      }
    }
  }
  if (a.residual) {
#pragma unroll
    for (int p = 0; p < kPer; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i)
        v[p][i] = fmaf(a.residual_scale, res[p][i], v[p][i]);
  }
  auto put = [&](void *out, int64_t stride) {
    if (!live)
      return;
    T *to = static_cast<T *>(out) + row * stride;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at(p, i) < dim)
          to[at(p, i)] = from_f32<T>(v[p][i]);
    }
  };
  if (a.h)
    put(a.h, a.h_stride);
  if (a.y) {
    if (a.pre.kind != CIM22_NORM_NONE)
      normalise(a.pre);
    put(a.y, a.y_stride);
  }
}

// A row's parameters, 16-byte aligned.
template <int N> __device__ __forceinline__ void load_whole(const void *base, int type, int64_t e, float (&out)[N]) {
  if (type == CIM22_FLOAT32) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
      const float4 p = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(base) + e + c));
      out[c] = p.x;
      out[c + 1] = p.y;
      out[c + 2] = p.z;
      out[c + 3] = p.w;
    }
  } else if constexpr (N == 8) {
    Pack<__nv_bfloat16> p;
    p.raw = __ldg(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(base) + e));
    if (type == CIM22_BFLOAT16) {
      unpack(p, out);
    } else {
      Pack<__half> h;
      h.raw = p.raw;
      unpack(h, out);
    }
  }
}

// Read once: past the L1 cache, which keeps the weights.
__device__ __forceinline__ uint4 load_stream(const void *at) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(at)
               : "memory");
  return v;
}

// Rows of whole, aligned vectors: every ordinary width. Each CTA
// keeps to its columns over many rows, so that it loads the weights once (kHold:
// into registers) and has the next row's streams on their way while it reduces
// this one. Measured on 32,768 x 4096 bf16 (two norms, a gate value a row): 237
// us, 4.5 TB/s, against 410 us of a CTA for each few rows, which tests every element's
// place and reads the weights each time (262,144 x 512: 195 and 265, x 64: 85
// and 178). What bounds it is the latency of a
// row's two reductions at 16 resident warps: with the weights left in memory 24
// warps fit and take 283 us, 512 threads a row 310 us.
template <typename T, int kPer, bool kHold, int kMax>
__global__ void __launch_bounds__(kMax) block_norm_rows_kernel(const BlockNormArgs a, const FastDiv gate_rows) {
  constexpr int V = kVec<T>;
  __shared__ float buffer[64];
  pdl_launch_dependents();
  pdl_wait();
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float inverse = 1.0f / static_cast<float>(a.dim);
  int slot = 0;
  int around = 0; // warps rounded up to a power of two, less one
  while (around < warps - 1)
    around = 2 * around + 1;
  int64_t at[kPer];
  bool in[kPer];
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    at[p] = static_cast<int64_t>(p * blockDim.x + threadIdx.x) * V;
    in[p] = at[p] < a.dim;
  }
  float post_w[kHold ? kPer : 1][V], pre_w[kHold ? kPer : 1][V];
  if constexpr (kHold) {
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        post_w[p][i] = pre_w[p][i] = 1.0f;
      if (in[p] && a.post.weight)
        load_whole<V>(a.post.weight, a.post.type, at[p], post_w[p]);
      if (in[p] && a.pre.weight)
        load_whole<V>(a.pre.weight, a.pre.type, at[p], pre_w[p]);
    }
  }
  auto block_sum = [&](float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
      v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1)
      return v;
    float *part = buffer + 32 * slot;
    slot ^= 1;
    if (lane == 0)
      part[warp] = v;
    __syncthreads();
    v = (lane & around) < warps ? part[lane & around] : 0.0f;
    for (int o = (around + 1) >> 1; o; o >>= 1)
      v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  // A gate value or gate row of each row comes with the row's other streams.
  const bool gate_value = a.gate && a.gate_columns == 1;
  const bool gate_stream = a.gate && !gate_value && a.gate_rows && a.type == a.gate_type;
  Pack<T> raw[kPer], res[kPer], gates[kPer];
  float gate_next = 0.0f;
  auto fetch = [&](int64_t row) {
    if (gate_value || gate_stream) {
      const int64_t from = a.gate_rows ? fdiv(static_cast<int>(row), gate_rows) * a.gate_stride : 0;
      if (gate_stream) {
#pragma unroll
        for (int p = 0; p < kPer; ++p)
          if (in[p])
            gates[p].raw = load_stream(static_cast<const T *>(a.gate) + from + at[p]);
      } else {
        gate_next = a.gate_type == CIM22_FLOAT32 ? static_cast<const float *>(a.gate)[from]
                                                 : to_f32(static_cast<const T *>(a.gate)[from]);
      }
    }
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *residual = static_cast<const T *>(a.residual) + row * a.residual_stride;
#pragma unroll
    for (int p = 0; p < kPer; ++p)
      if (in[p]) {
        raw[p].raw = load_stream(x + at[p]);
        if (a.residual)
          res[p].raw = load_stream(residual + at[p]);
      }
  };
  int64_t row = blockIdx.x;
  if (row < a.rows)
    fetch(row);
  for (; row < a.rows; row += gridDim.x) {
    float v[kPer][V];
    Pack<T> held[kPer], gate_held[kPer];
    const float gate_now = gate_next;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      held[p] = res[p];
      gate_held[p] = gates[p];
      unpack(raw[p], v[p]); // zero outside the row
    }
    if (row + gridDim.x < a.rows)
      fetch(row + gridDim.x);
    auto normalise = [&](const NormArg &n, const float (&held_w)[kHold ? kPer : 1][V]) {
      float mean = 0.0f, s = 0.0f;
      if (n.kind == CIM22_NORM_LAYER) {
#pragma unroll
        for (int p = 0; p < kPer; ++p)
#pragma unroll
          for (int i = 0; i < V; ++i)
            s += v[p][i];
        mean = block_sum(s) * inverse;
        s = 0.0f;
      }
      if (n.kind == CIM22_NORM_LAYER) {
#pragma unroll
        for (int p = 0; p < kPer; ++p)
#pragma unroll
          for (int i = 0; i < V; ++i)
            v[p][i] = in[p] ? v[p][i] - mean : 0.0f;
      }
#pragma unroll
      for (int p = 0; p < kPer; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i)
          s = fmaf(v[p][i], v[p][i], s);
      const float scale = rsqrtf(block_sum(s) * inverse + n.eps);
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        float g[V];
        if constexpr (kHold) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            v[p][i] *= scale * held_w[p][i];
        } else if (n.weight) {
          if (in[p])
            load_whole<V>(n.weight, n.type, at[p], g);
#pragma unroll
          for (int i = 0; i < V; ++i)
            v[p][i] = in[p] ? v[p][i] * (scale * g[i]) : 0.0f;
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i)
            v[p][i] *= scale;
        }
        if (n.bias && in[p]) {
          load_whole<V>(n.bias, n.type, at[p], g);
#pragma unroll
          for (int i = 0; i < V; ++i)
            v[p][i] += g[i];
        }
      }
    };
    if (a.post.kind != CIM22_NORM_NONE)
      normalise(a.post, post_w);
    if (gate_value) {
      const float g = gate_fn(gate_now, a.gate_act);
#pragma unroll
      for (int p = 0; p < kPer; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] *= g;
    } else if (a.gate) {
      const int64_t from =
          a.gate_rows && !gate_stream ? fdiv(static_cast<int>(row), gate_rows) * a.gate_stride : 0;
      const char *gate = static_cast<const char *>(a.gate) + from * (a.gate_type == CIM22_FLOAT32 ? 4 : 2);
#pragma unroll
      for (int p = 0; p < kPer; ++p)
        if (in[p]) {
          float g[V];
          if (gate_stream)
            unpack(gate_held[p], g);
          else
            load_whole<V>(gate, a.gate_type, at[p], g);
#pragma unroll
          for (int i = 0; i < V; ++i)
            v[p][i] *= gate_fn(g[i], a.gate_act);
        }
    }
    if (a.residual) {
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        float r[V];
        unpack(held[p], r);
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] = fmaf(a.residual_scale, r[i], v[p][i]);
      }
    }
    auto put = [&](void *out, int64_t stride) {
      T *to = static_cast<T *>(out) + row * stride;
#pragma unroll
      for (int p = 0; p < kPer; ++p)
        if (in[p]) {
          Pack<T> o;
          pack(v[p], o);
          *reinterpret_cast<uint4 *>(to + at[p]) = o.raw;
        }
    };
    if (a.h)
      put(a.h, a.h_stride);
    if (a.y) {
      if (a.pre.kind != CIM22_NORM_NONE)
        normalise(a.pre, pre_w);
      put(a.y, a.y_stride);
    }
  }
}

// Whether every row, parameter and gate row consists of aligned vectors.
template <typename T> bool whole_vectors(const BlockNormArgs &a) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.residual) |
                   reinterpret_cast<uintptr_t>(a.h) | reinterpret_cast<uintptr_t>(a.y) |
                   reinterpret_cast<uintptr_t>(a.post.weight) | reinterpret_cast<uintptr_t>(a.post.bias) |
                   reinterpret_cast<uintptr_t>(a.pre.weight) | reinterpret_cast<uintptr_t>(a.pre.bias);
  uint64_t strides = a.dim;
  if (a.rows > 1)
    strides |= a.x_stride | (a.residual ? a.residual_stride : 0) | (a.h ? a.h_stride : 0) |
               (a.y ? a.y_stride : 0);
  if (a.gate && a.gate_columns != 1) {
    bits |= reinterpret_cast<uintptr_t>(a.gate);
    strides |= a.gate_stride;
  }
  return bits % 16 == 0 && strides % kVec<T> == 0;
}

template <typename T, int kPer, bool kHold, int kMax>
cudaError_t launch_rows(const BlockNormArgs &a, int threads, cudaStream_t stream) {
  const auto kernel = block_norm_rows_kernel<T, kPer, kHold, kMax>;
  // CTAs an SM for each block size, asked for once (every device is a B200).
  static std::atomic<int> known[kMax / 32 + 1];
  int resident = known[threads / 32].load(std::memory_order_relaxed);
  if (resident == 0) {
    if (const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, threads, 0);
        e != cudaSuccess)
      return e;
    known[threads / 32].store(resident, std::memory_order_relaxed);
  }
  const int64_t grid = std::min<int64_t>(a.rows, 148 * std::max(1, resident));
  return launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(threads), 0, stream, a,
                    make_fastdiv(static_cast<uint32_t>(std::max<int64_t>(1, a.gate_rows))));
}

template <typename T>
cudaError_t launch_block_norm(BlockNormArgs a, cudaStream_t stream) {
  constexpr int V = kVec<T>;
  const int64_t vectors = (a.dim + V - 1) / V;
  if (whole_vectors<T>(a)) {
    if (vectors <= 256)
      return launch_rows<T, 1, true, 256>(a, static_cast<int>(round_up(vectors, 32)), stream);
    if (vectors <= 512)
      return launch_rows<T, 2, true, 256>(a, 256, stream);
    if (vectors <= 1024) // (512 x 4096 f32, two layer norms: 13.9 us; 256 threads 18.4)
      return launch_rows<T, 2, true, 512>(a, 512, stream);
    if constexpr (V == 8) {
      return launch_rows<T, 4, false, 512>(a, 512, stream);
    } else {
      if (vectors <= 2048)
        return launch_rows<T, 4, true, 512>(a, 512, stream);
      return launch_rows<T, 8, false, 512>(a, 512, stream);
    }
  }
  // Groups of V elements a thread and warps a row: two groups, and four only
  // where the row needs them (20,000 x 1,001 f16: 98 us; four 137, one 106).
  const int per = vectors <= 32 ? 1 : vectors <= (V == 8 ? 1024 : 2048) ? 2 : 4;
  int log2w = 0;
  while ((int64_t{32} * per << log2w) < vectors)
    ++log2w;
  a.warps_log2 = log2w;
  const int warps = std::max(8, 1 << log2w);
  const int64_t grid = (a.rows + (warps >> log2w) - 1) / (warps >> log2w);
  constexpr int kWidest = V == 8 ? 512 : 1024; // threads of the widest row
  const auto kernel = per == 1     ? block_norm_kernel<T, 1, 256>
                      : per == 4   ? block_norm_kernel<T, 4, kWidest>
                      : warps <= 8 ? block_norm_kernel<T, 2, 256>
                                   : block_norm_kernel<T, 2, kWidest>;
  return launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(warps * 32), 0, stream, a);
}

bool refuse(const char *why) {
  set_last_error(std::string("cim22_cuda_block_norm: ") + why);
  return false;
}

bool norm_arg(const cim22_norm *n, int32_t type, NormArg &out) {
  out = NormArg{CIM22_NORM_NONE, 0.0f, nullptr, nullptr, type};
  if (!n)
    return true;
  if (n->kind != CIM22_NORM_RMS && n->kind != CIM22_NORM_LAYER)
    return refuse("norm kind must be CIM22_NORM_RMS or CIM22_NORM_LAYER");
  if (n->type != CIM22_FLOAT32 && n->type != type)
    return refuse("norm weights must be f32 or the activations' type");
  if (!(n->eps >= 0.0f))
    return refuse("norm eps must not be negative");
  out = NormArg{n->kind, n->eps, n->weight, n->bias, n->type};
  return true;
}

} // namespace
} // namespace cim

extern "C" int cim22_cuda_block_norm(const cim22_block_norm *d, void *stream) {
  using namespace cim;
  const int bad = CIM22_STATUS_BAD_ARGUMENT;
  if (!d)
    return refuse("null description"), bad;
  if (!float_type(d->type))
    return refuse("unknown activation type"), bad;
  if (d->rows < 0 || d->dim < 1 || d->dim > CIM22_BLOCK_NORM_MAX_DIM || d->rows > 0x7fffffff)
    return refuse("rows or dim out of range"), bad;
  if (d->rows > 0 && (!d->x || (!d->h && !d->y)))
    return refuse("null x, or neither h nor y"), bad;
  if ((d->rows > 1) && (d->x_stride < d->dim || (d->residual && d->residual_stride < d->dim) ||
                        (d->h && d->h_stride < d->dim) || (d->y && d->y_stride < d->dim)))
    return refuse("row strides must be at least dim"), bad;
  if (d->gate) {
    if (d->gate_type != CIM22_FLOAT32 && d->gate_type != d->type)
      return refuse("gate must be f32 or the activations' type"), bad;
    if (d->gate_columns != 1 && d->gate_columns != d->dim)
      return refuse("gate must have 1 or dim columns"), bad;
    if (d->gate_rows < 0 || d->gate_activation < 0 || d->gate_activation > CIM22_GATE_TANH)
      return refuse("gate rows or activation out of range"), bad;
  }
  BlockNormArgs a{};
  if (!norm_arg(d->post, d->type, a.post) || !norm_arg(d->pre, d->type, a.pre))
    return bad;
  if (d->rows == 0)
    return 0;
  a.x = d->x;
  a.residual = d->residual;
  a.gate = d->gate;
  a.h = d->h;
  a.y = d->y;
  a.rows = d->rows;
  a.dim = d->dim;
  a.x_stride = d->x_stride;
  a.residual_stride = d->residual_stride;
  a.gate_stride = d->gate_stride;
  a.h_stride = d->h_stride;
  a.y_stride = d->y_stride;
  a.gate_rows = std::min(d->gate_rows, d->rows); // as much as any more; divided by in 32 bits
  a.type = d->type;
  a.gate_type = d->gate_type;
  a.gate_columns = static_cast<int>(d->gate_columns == d->dim ? 0 : 1);
  a.gate_act = d->gate_activation;
  a.residual_scale = d->residual_scale;
  const auto s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d->type == CIM22_FLOAT32)
    e = launch_block_norm<float>(a, s);
  else if (d->type == CIM22_BFLOAT16)
    e = launch_block_norm<__nv_bfloat16>(a, s);
  else
    e = launch_block_norm<__half>(a, s);
  return cuda_ok(e, "block_norm") ? 0 : bad;
}
