// kv_attention.cu - attention of few query rows over the 8-bit cache, and the
// dispatch between it and the tensor-memory kernel for prompts.
//
// Decode reads every cached code once: bound by HBM. A tile is the 16 rows of
// an m16n8k16 product (query tokens x the heads that share a kv head), a work
// item a 16-token group of one kv head, which lies in one page, so its two
// scales are constants. Warps take groups in turn and need nothing from each
// other until the end: each lane copies (cp.async) exactly the bytes it later
// feeds the product with into its own shared-memory slots, six groups deep,
// so the ring has no barriers and no bank conflicts:
//   keys    lane (g, c) holds token g's codes 16c .. 16c + 15 of each 64: the
//           contraction runs over head_dim in the order that makes these its
//           B fragments, and the queries are laid out to match;
//   values  lane (g, c) holds codes 16g .. 16g + 15 (D = 128) of tokens 2c,
//           2c + 1, 8 + 2c, 9 + 2c: byte permutes make the fragments, and the
//           output columns come out as 32 neighbouring elements a lane.
// Codes are exact in f16. Queries are scaled by a power of two a row and held
// as one f16 part (bf16 and f16 inputs lose nothing within 2^-39 of the row's
// largest) or two (f32: 22 bits); so are the probabilities.
#include "kv_attention.h"

#include <algorithm>

namespace cim {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 6;

template <int kCh> constexpr int kStageBytes = 16 * 2 * 64 * kCh; // one group of one warp

__device__ __forceinline__ uint32_t smem_at(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, bool valid) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(valid ? 16 : 0)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src),
                 "r"(valid ? 8 : 0)
                 : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One row's final (or partial) output element range.
template <typename T, int kCount>
__device__ __forceinline__ void put_row(T *out, int d, int dim, const float (&v)[kCount]) {
#pragma unroll
  for (int i = 0; i < kCount; i += kVec<T>) {
    Pack<T> o;
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j)
      o.at[j] = from_f32<T>(v[i + j]);
    store_pack(out, d + i, dim, o);
  }
}

template <typename T, int kCh, int kParts>
__global__ void __launch_bounds__(kThreads, 2) kv_decode_kernel(const KvAttendArgs a) {
  constexpr int kTiles = 8 * kCh;     // output tiles: element 8 * kCh * g + j of the head
  constexpr int kLane = 8 * kCh;      // value bytes a lane holds of a token
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float row_m[kWarps][16], row_l[kWarps][16], row_e[kWarps][16];
  pdl_launch_dependents();
  pdl_wait();
  const KvView &v = a.v;
  const int b = blockIdx.z, split = blockIdx.x;
  const int head = blockIdx.y % v.heads, f0 = blockIdx.y / v.heads * 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const KvSequence s = kv_sequence(v, b);
  if (!s.ok) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0)
      atomicOr(a.status, CIM22_STATUS_CACHE_INDEX);
    return;
  }
  const int rows = s.n * a.group;
  if (f0 >= rows)
    return;
  const int offset = s.length - s.n; // position of the sequence's row 0
  const int last = min(f0 + 15, rows - 1);
  int lo, hi;
  key_range(a, s.length, offset + f0 / a.group, offset + last / a.group, lo, hi);
  const int first_group = lo >> 4, groups = ((hi + 15) >> 4) - first_group;
  const int each = (groups + a.splits - 1) / a.splits;
  const int begin = first_group + min(groups, split * each);
  const int end = first_group + min(groups, (split + 1) * each);

  // Query rows g and g + 8 as A fragments.
  uint32_t qa[kParts][kCh * 4][4];
  float coef[2];
  int pos[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int f = f0 + g + 8 * r;
    const bool live = f < rows;
    const int i = live ? f / a.group : 0;
    pos[r] = live ? offset + i : -0x40000000; // a row past the tile sees nothing that counts
    const T *q = static_cast<const T *>(a.q) + (s.row0 + i) * a.q_row_stride +
                 (head * a.group + (live ? f - i * a.group : 0)) * a.q_head_stride;
    float x[kCh * 16];
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < kCh * 16; e += kVec<T>) {
      Pack<T> p;
      if (live)
        p = load_pack(q, (e / 16) * 64 + 16 * c + e % 16, v.dim);
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j) {
        x[e + j] = to_f32(p.at[j]);
        const float m = fabsf(x[e + j]);
        amax = nan_max(amax, m);
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) {
      const float m = __shfl_xor_sync(0xffffffffu, amax, o);
      amax = nan_max(amax, m);
    }
    float factor, inverse;
    row_factor(amax, factor, inverse);
    // A row with NaN or infinity gives NaN wherever it sees a key.
    coef[r] = amax < INFINITY ? inverse * a.scale_log2 : NAN;
#pragma unroll
    for (int e = 0; e < kCh * 16; e += 2) {
      const float y0 = x[e] * factor, y1 = x[e + 1] * factor;
      const uint32_t h = pack_half(y0, y1);
      // Elements 4s .. 4s + 3 of a lane are columns 2c, 2c + 1, 2c + 8, 2c + 9.
      qa[0][e / 4][(e & 2) + r] = h;
      if constexpr (kParts == 2) {
        const float2 back = unpack_half(h);
        qa[1][e / 4][(e & 2) + r] = pack_half(y0 - back.x, y1 - back.y);
      }
    }
  }

  float o[kTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
    o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  // l sums the probabilities as the product takes them, so that their rounding
  // leaves the weights' sum at one; full sums them unrounded for the logarithm.
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, full[2] = {0.0f, 0.0f};

  const uint32_t ring = smem_at(smem) + warp * kStages * kStageBytes<kCh>;
  const int count = end > begin + warp ? (end - begin - warp + kWarps - 1) / kWarps : 0;
  // Lane i of a batch of 32 holds what the warp needs of its i-th group.
  int batch_page = -1, next_page = -1;
  float batch_k = 0.0f, batch_log = 0.0f, batch_inv = 0.0f;
  auto pages_of = [&](int j0) {
    const int j = j0 + lane;
    int page = -1;
    if (j < count) {
      const int64_t group = begin + warp + static_cast<int64_t>(j) * kWarps;
      page = kv_page(v, b, static_cast<int>(group >> (v.block_log2 - 4)));
      if (page < 0)
        atomicOr(a.status, CIM22_STATUS_CACHE_INDEX);
    }
    return page;
  };
  auto issue = [&](int j) { // every lane copies its bytes of group j
    if (j < count) {
      const int page = __shfl_sync(0xffffffffu, (j & 32) == 0 ? batch_page : next_page, j & 31);
      const int64_t group = begin + warp + static_cast<int64_t>(j) * kWarps;
      const int token = static_cast<int>(group & ((1 << (v.block_log2 - 4)) - 1)) << 4;
      const int8_t *k = kv_codes(v, max(page, 0), head, 0) + token * v.dim;
      const int8_t *values = k + (static_cast<int64_t>(v.dim) << v.block_log2);
      const uint32_t slot = ring + (j % kStages) * kStageBytes<kCh>;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int ch = 0; ch < kCh; ++ch) {
          const int d = 64 * ch + 16 * c;
          const bool in = page >= 0 && d < v.dim;
          copy_async<16>(slot + (u * kCh + ch) * 512 + lane * 16,
                         in ? k + (8 * u + g) * v.dim + d : v.codes, in);
        }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int d = kLane * g;
        const bool in = page >= 0 && d < v.dim;
        copy_async<kLane>(slot + 2 * kCh * 512 + t * 32 * kLane + lane * kLane,
                          in ? values + ((t & 1) + 2 * c + 8 * (t >> 1)) * v.dim + d : v.codes, in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // The pages of groups [64 i, 64 i + 32) are in batch_page, of the next 32 in
  // next_page; each is refilled when its last group has been issued.
  batch_page = pages_of(0);
  next_page = pages_of(32);
#pragma unroll 1
  for (int j = 0; j < kStages - 1; ++j)
    issue(j);
#pragma unroll 1
  for (int j = 0; j < count; ++j) {
    if ((j & 31) == 0) { // scales of groups j .. j + 31 (their pages are still held)
      const int page = (j & 32) == 0 ? batch_page : next_page;
      batch_k = batch_log = 0.0f;
      batch_inv = 1.0f;
      if (page >= 0) {
        const float2 sc = *reinterpret_cast<const float2 *>(
            v.scales + (static_cast<int64_t>(page) * v.heads + head) * 2);
        const float sv = fmaxf(sc.y, kKvLeastScale);
        batch_k = sc.x;
        batch_log = log2f(sv);
        batch_inv = 1.0f / sv;
      }
    }
    const bool usable = __shfl_sync(0xffffffffu, (j & 32) == 0 ? batch_page : next_page, j & 31) >= 0;
    issue(j + kStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    const uint32_t slot = ring + (j % kStages) * kStageBytes<kCh>;
    const float sk = __shfl_sync(0xffffffffu, batch_k, j & 31);
    const float log_sv = __shfl_sync(0xffffffffu, batch_log, j & 31);
    const float inv_sv = __shfl_sync(0xffffffffu, batch_inv, j & 31);
    if ((j & 31) == 31) { // this batch's pages are no longer needed
      const int refill = pages_of(j + 33);
      if ((j & 32) == 0)
        batch_page = refill;
      else
        next_page = refill;
    }

    float sc[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u][0] = sc[u][1] = sc[u][2] = sc[u][3] = 0.0f;
#pragma unroll
      for (int ch = 0; ch < kCh; ++ch) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(slot + (u * kCh + ch) * 512 + lane * 16)
                     : "memory");
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t b0, b1;
          codes_to_half(w[x], b0, b1);
          mma_f16(sc[u], qa[0][ch * 4 + x], b0, b1);
          if constexpr (kParts == 2)
            mma_f16(sc[u], qa[1][ch * 4 + x], b0, b1);
        }
      }
    }
    // Exponents relative to the rows' references.
    const int key0 = static_cast<int>((begin + warp + static_cast<int64_t>(j) * kWarps) << 4);
    const bool whole = usable && key0 + 15 < s.length &&
                       (!a.causal || key0 + 15 <= offset + f0 / a.group) &&
                       (a.window <= 0 || key0 > offset + last / a.group - a.window);
    uint32_t hidden = 0; // bit 4 u + e
    if (!whole) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!usable || !sees(a, s.length, pos[e >> 1], key0 + 8 * u + 2 * c + (e & 1)))
            hidden |= 1u << (4 * u + e);
    }
    float arg[2][4];
    auto arguments = [&](int r) {
      const float factor = coef[r] * sk, shift = log_sv - (m[r] == -INFINITY ? 0.0f : m[r]);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e)
          arg[u][e] = hidden >> (4 * u + e) & 1 ? -INFINITY : fmaf(sc[u][e], factor, shift);
    };
    bool grown = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      arguments(r);
      const float limit = m[r] == -INFINITY ? -INFINITY : kGrowth<kParts>;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e)
          grown |= !(arg[u][e] <= limit); // NaN too
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = arg[0][2 * r];
        top = nan_max(top, arg[0][2 * r + 1]);
        top = nan_max(top, arg[1][2 * r]);
        top = nan_max(top, arg[1][2 * r + 1]);
#pragma unroll
        for (int x = 1; x < 4; x *= 2)
          top = nan_max(top, __shfl_xor_sync(0xffffffffu, top, x));
        if (top != -INFINITY && (m[r] == -INFINITY || !(top <= kTop<kParts>))) {
          const float to = (m[r] == -INFINITY ? 0.0f : m[r]) + top - kTop<kParts>;
          const float shrink = exp2_approx(m[r] - to); // 0 for the first
          m[r] = to;
          l[r] *= shrink;
          full[r] *= shrink;
#pragma unroll
          for (int j2 = 0; j2 < kTiles; ++j2) {
            o[j2][2 * r] *= shrink;
            o[j2][2 * r + 1] *= shrink;
          }
          arguments(r);
        }
      }
    }
    uint32_t pa[kParts][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float p0 = exp2_approx(arg[u][2 * r]), p1 = exp2_approx(arg[u][2 * r + 1]);
        const uint32_t h = pack_half(p0, p1);
        const float2 back = unpack_half(h);
        pa[0][2 * u + r] = h;
        if constexpr (kParts == 2) {
          pa[1][2 * u + r] = pack_half(p0 - back.x, p1 - back.y);
          l[r] = fmaf(p0 + p1, inv_sv, l[r]);
        } else {
          l[r] = fmaf(back.x + back.y, inv_sv, l[r]);
          full[r] = fmaf(p0 + p1, inv_sv, full[r]);
        }
      }
    // Values: pairs of tokens at one element.
    uint32_t w[4][2 * kCh];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t at = slot + 2 * kCh * 512 + t * 32 * kLane + lane * kLane;
      if constexpr (kCh == 2)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[t][0]), "=r"(w[t][1]), "=r"(w[t][2]), "=r"(w[t][3])
                     : "r"(at)
                     : "memory");
      else
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                     : "=r"(w[t][0]), "=r"(w[t][1])
                     : "r"(at)
                     : "memory");
    }
#pragma unroll
    for (int x = 0; x < 2 * kCh; ++x) {
      uint32_t h[2][4]; // token pair, element
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        codes_to_half(__byte_perm(w[2 * t][x], w[2 * t + 1][x], 0x5140), h[t][0], h[t][1]);
        codes_to_half(__byte_perm(w[2 * t][x], w[2 * t + 1][x], 0x7362), h[t][2], h[t][3]);
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if constexpr (kParts == 2) {
          // The product's own accumulation does not round to nearest: over
          // many groups in one accumulator that cost f32 outputs half their
          // accuracy (1.2e-6 against 0.7e-6 relative at 1500 keys), so each
          // group's products are added to the sum here.
          float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_f16(part, pa[1], h[0][y], h[1][y]);
          mma_f16(part, pa[0], h[0][y], h[1][y]);
#pragma unroll
          for (int z = 0; z < 4; ++z)
            o[4 * x + y][z] += part[z];
        } else {
          mma_f16(o[4 * x + y], pa[0], h[0][y], h[1][y]);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int x = 1; x < 4; x *= 2) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
      full[r] += __shfl_xor_sync(0xffffffffu, full[r], x);
    }

  // Join the warps: rows [warp][16][64 * kCh] in the ring's memory.
  __syncthreads();
  float *joined = reinterpret_cast<float *>(smem);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = g + 8 * r;
    if (c == 0) {
      row_m[warp][row] = m[r];
      row_l[warp][row] = l[r];
      row_e[warp][row] = kParts == 2 ? l[r] : full[r];
    }
    float *to = joined + (warp * 16 + row) * 64 * kCh;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      to[kTiles * (2 * c) + j] = o[j][2 * r];
      to[kTiles * (2 * c + 1) + j] = o[j][2 * r + 1];
    }
  }
  __syncthreads();
  const int row = threadIdx.x >> 3, d = (threadIdx.x & 7) * kTiles;
  const int f = f0 + row;
  if (f >= rows)
    return;
  float top = -INFINITY;
#pragma unroll
  for (int x = 0; x < kWarps; ++x)
    top = nan_max(top, row_m[x][row]);
  float sum = 0.0f, plain = 0.0f, acc[kTiles];
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
    acc[j] = 0.0f;
#pragma unroll
  for (int x = 0; x < kWarps; ++x) {
    const float share = row_m[x][row] == -INFINITY ? 0.0f : exp2_approx(row_m[x][row] - top);
    sum = fmaf(row_l[x][row], share, sum);
    plain = fmaf(row_e[x][row], share, plain);
    if (share != 0.0f) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
        acc[j] = fmaf(joined[(x * 16 + row) * 64 * kCh + d + j], share, acc[j]);
    }
  }
  const int i = f / a.group;
  const int64_t at = (s.row0 + i) * a.q_heads + head * a.group + (f - i * a.group);
  if (a.splits > 1) {
    const int64_t slot = static_cast<int64_t>(split) * v.rows * a.q_heads + at;
    if ((threadIdx.x & 7) == 0)
      a.part_ml[slot] = make_float4(top, sum, plain, 0.0f);
    put_row(a.part_o + slot * v.dim, d, v.dim, acc);
    return;
  }
  const bool some = top > -INFINITY || top != top;
  const float share = some ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
    acc[j] *= share;
  put_row(static_cast<T *>(a.out) + at * v.dim, d, v.dim, acc);
  if (a.lse && (threadIdx.x & 7) == 0)
    a.lse[at] = some ? (top + log2f(plain)) * 0.69314718055994531f : -INFINITY;
}

// Joins the parts of the key axis: a warp a row and head.
template <typename T>
__global__ void __launch_bounds__(128) kv_join_kernel(const KvAttendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const KvView &v = a.v;
  const int b = blockIdx.z, lane = threadIdx.x & 31;
  const KvSequence s = kv_sequence(v, b);
  const int64_t f = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (!s.ok || f >= static_cast<int64_t>(s.n) * a.q_heads)
    return;
  const int64_t at = s.row0 * a.q_heads + f, step = v.rows * a.q_heads;
  float top = -INFINITY;
  for (int x = 0; x < a.splits; ++x) {
    const float m = a.part_ml[x * step + at].x;
    top = nan_max(top, m);
  }
  float sum = 0.0f, plain = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int x = 0; x < a.splits; ++x) {
    const float4 ml = a.part_ml[x * step + at];
    const float share = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - top);
    if (share == 0.0f)
      continue;
    sum = fmaf(ml.y, share, sum);
    plain = fmaf(ml.z, share, plain);
    if (4 * lane < v.dim) {
      const float4 p = *reinterpret_cast<const float4 *>(a.part_o + (x * step + at) * v.dim + 4 * lane);
      acc[0] = fmaf(p.x, share, acc[0]);
      acc[1] = fmaf(p.y, share, acc[1]);
      acc[2] = fmaf(p.z, share, acc[2]);
      acc[3] = fmaf(p.w, share, acc[3]);
    }
  }
  const bool some = top > -INFINITY || top != top;
  const float share = some ? 1.0f / sum : 0.0f;
  if (4 * lane < v.dim) {
    T *out = static_cast<T *>(a.out) + at * v.dim + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      out[j] = from_f32<T>(acc[j] * share);
  }
  if (a.lse && lane == 0)
    a.lse[at] = some ? (top + log2f(plain)) * 0.69314718055994531f : -INFINITY;
}

// Parts of the key axis: enough work items for two resident CTAs an SM, each
// part at least 256 keys.
int decode_splits(const KvView &v, int64_t tiles, int64_t longest) {
  const int64_t items = std::max<int64_t>(1, tiles * v.heads * v.batch);
  const int64_t want = (2 * 148 + items - 1) / items;
  return static_cast<int>(std::max<int64_t>(1, std::min({want, (longest + 255) / 256, int64_t{64}})));
}

struct Plan {
  bool prompt; // by the tensor-memory kernel
  bool share;  // with one query tile a CTA
  int splits;
  int64_t tiles;
  size_t bytes; // of the partial results
};

// Up to kDecodeRows query rows a sequence and kv head go to the decode kernel.
constexpr int64_t kDecodeRows = 32;

Plan attend_plan(const KvView &v, const cim22_kv_attention &t) {
  Plan p;
  const int64_t group = t.q_heads / v.heads;
  const int64_t rows = std::min<int64_t>(v.most, v.rows) * group;
  const int64_t held = static_cast<int64_t>(v.table_width) << v.block_log2;
  const int64_t longest = std::max<int64_t>(1, std::min(t.longest, held));
  p.prompt = rows > kDecodeRows;
  p.share = p.prompt && (t.type == CIM22_FLOAT32 || rows <= 128);
  if (!p.prompt) {
    p.tiles = (rows + 15) / 16;
    p.splits = decode_splits(v, p.tiles, longest);
  } else {
    p.tiles = (rows + (p.share ? 127 : 255)) / (p.share ? 128 : 256);
    const int64_t items = p.tiles * v.heads * v.batch;
    p.splits = static_cast<int>(std::max<int64_t>(1, std::min({148 / std::max<int64_t>(1, items), (longest + 1023) / 1024, int64_t{64}})));
  }
  p.bytes = p.splits == 1 ? 0
                          : static_cast<size_t>(p.splits) * v.rows * t.q_heads *
                                (static_cast<size_t>(v.dim) * 4 + 16);
  return p;
}

bool attend_args(const char *what, const KvView &v, const cim22_kv_attention *t) {
  const auto refuse = [&](const char *why) {
    set_last_error(std::string(what) + ": " + why);
    return false;
  };
  if (!t)
    return refuse("null attention");
  if (!float_type(t->type))
    return refuse("unknown type");
  if (t->q_heads < 1 || t->q_heads % v.heads)
    return refuse("q_heads must be a multiple of kv_heads");
  if (t->window < 0 || t->longest < 0)
    return refuse("window and longest must not be negative");
  if (t->q_row_stride < 0 || t->q_head_stride < 0)
    return refuse("strides must not be negative");
  if (!(t->scale == t->scale) || t->scale - t->scale != 0.0f)
    return refuse("scale must be finite");
  if (static_cast<int64_t>(v.most) * (t->q_heads / v.heads) > 0x3fffffff)
    return refuse("too many query rows");
  return true;
}

template <typename T, int kCh, int kParts>
cudaError_t launch_decode(const KvAttendArgs &a, int64_t tiles, cudaStream_t stream) {
  constexpr size_t bytes = static_cast<size_t>(kWarps) * kStages * kStageBytes<kCh>;
  const auto kernel = kv_decode_kernel<T, kCh, kParts>;
  static DynamicSmem allowed;
  if (const cudaError_t e = allowed.allow(kernel, bytes); e != cudaSuccess)
    return e;
  return launch_pdl(kernel, dim3(a.splits, static_cast<unsigned>(tiles * a.v.heads), a.v.batch),
                    dim3(kThreads), bytes, stream, a);
}

template <typename T, int kParts>
cudaError_t launch_attend(const KvAttendArgs &a, int type, const Plan &plan, cudaStream_t stream) {
  cudaError_t e = plan.prompt ? kv_prompt_launch(a, type, plan.share, static_cast<int>(plan.tiles), stream)
                  : a.v.dim > 64 ? launch_decode<T, 2, kParts>(a, plan.tiles, stream)
                                 : launch_decode<T, 1, kParts>(a, plan.tiles, stream);
  if (e == cudaSuccess && a.splits > 1) {
    const int64_t rows = std::min<int64_t>(a.v.most, a.v.rows) * a.q_heads;
    e = launch_pdl(kv_join_kernel<T>, dim3(static_cast<unsigned>((rows + 3) / 4), 1, a.v.batch),
                   dim3(128), 0, stream, a);
  }
  return e;
}

} // namespace
} // namespace cim

using namespace cim;

extern "C" {

size_t cim22_cuda_kv_attend_workspace(const cim22_kv_cache *cache,
                                      const cim22_kv_sequences *sequences,
                                      const cim22_kv_attention *attention) {
  KvView v;
  if (!kv_view("cim22_cuda_kv_attend_workspace", cache, sequences, v) ||
      !attend_args("cim22_cuda_kv_attend_workspace", v, attention))
    return 0;
  return attend_plan(v, *attention).bytes;
}

int cim22_cuda_kv_attend(const cim22_kv_cache *cache, const cim22_kv_sequences *sequences,
                         const cim22_kv_attention *attention, void *workspace,
                         size_t workspace_bytes, int32_t *status, void *stream) {
  const int bad = CIM22_STATUS_BAD_ARGUMENT;
  const char *what = "cim22_cuda_kv_attend";
  KvView v;
  if (!kv_view(what, cache, sequences, v) || !attend_args(what, v, attention))
    return bad;
  if (!status || (v.rows > 0 && (!attention->q || !attention->out))) {
    set_last_error("cim22_cuda_kv_attend: null q, out or status");
    return bad;
  }
  if (v.batch == 0 || v.rows == 0)
    return 0;
  const Plan plan = attend_plan(v, *attention);
  if (plan.bytes > workspace_bytes || (plan.bytes && !workspace) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_last_error("cim22_cuda_kv_attend: workspace too small or not 16-byte aligned");
    return bad;
  }
  if (plan.tiles * v.heads > 65535) {
    set_last_error("cim22_cuda_kv_attend: too many query rows");
    return bad;
  }
  KvAttendArgs a{};
  a.v = v;
  a.q = attention->q;
  a.q_row_stride = attention->q_row_stride;
  a.q_head_stride = attention->q_head_stride;
  a.out = attention->out;
  a.lse = attention->lse;
  a.scale_log2 = attention->scale * 1.4426950408889634f;
  a.q_heads = attention->q_heads;
  a.group = attention->q_heads / v.heads;
  a.causal = attention->causal != 0;
  a.window = attention->window;
  a.splits = plan.splits;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = plan.bytes ? reinterpret_cast<float4 *>(a.part_o + static_cast<size_t>(plan.splits) * v.rows * a.q_heads * v.dim)
                         : nullptr;
  a.status = status;
  const auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      attention->type == CIM22_FLOAT32    ? launch_attend<float, 2>(a, attention->type, plan, s)
      : attention->type == CIM22_BFLOAT16 ? launch_attend<__nv_bfloat16, 1>(a, attention->type, plan, s)
                                          : launch_attend<__half, 1>(a, attention->type, plan, s);
  return cuda_ok(e, "kv_attend") ? 0 : bad;
}

} // extern "C"
