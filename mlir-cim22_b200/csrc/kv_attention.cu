// kv_attention.cu - attention of few query rows over the 8-bit cache, and the
// dispatch between it and the tensor-memory kernel for prompts.
//
// Decode reads every cached code once: bound by HBM (64 sequences of 286,000
// tokens in all, 8 kv heads of 128, bf16: 112 us, 5.2 TB/s; one of 200,000, 4 kv
// heads, 47 us, 4.4 TB/s with its filling and joining). The products are taken
// transposed, S^T = K Q^T and O^T = V^T P^T (m16n8k16), so that 16 tokens or
// 16 elements of the head fill the 16 rows and a tile needs only 8 query rows
// (query tokens x the heads that share a kv head). A work item is a 16-token
// group of one kv head, which lies in one page, so its two scales are
// constants. Warps take groups in turn and need nothing from each other until
// the end: each has its own ring of swizzled shared-memory tiles that one bulk
// tensor copy a group fills (per-lane asynchronous copies of the same bytes
// stopped at 3.4 TB/s, whatever was done with them).
//   keys    lane (g, c) takes codes 16c .. 16c + 15 of each 64 of tokens t(g)
//           and 8 + t(g): the contraction runs over head_dim in the order that
//           makes these its A fragments, and the queries are laid out to match;
//   values  lane (g, c) takes 16 codes (D = 128) of tokens t(2c), t(2c + 1) and
//           those plus 8: byte permutes make the A fragments, and neighbouring
//           rows of the result are neighbouring elements.
// t and the elements that a lane takes are chosen so that eight neighbouring
// lanes read eight different 16-byte banks of the swizzled rows.
// Codes are exact in f16. Queries are scaled by a power of two a row and held
// as one f16 part (bf16 and f16 inputs lose nothing within 2^-39 of the row's
// largest) or two (f32: 22 bits); so are the probabilities.
#include "gemm_tc.h"
#include "kv_attention.h"
#include "tma_util.cuh"

#include <algorithm>

namespace cim {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;

// CTAs an SM by the registers that query tiles and parts take, the groups that
// a warp then has in its ring, and how many it takes at a time.
template <int kParts, int kQ> constexpr int kResident = kParts * kQ == 4 ? 2 : 3;
template <int kCh> constexpr int kGroupBytes = 16 * 2 * 64 * kCh;
template <int kCh, int kParts, int kQ> constexpr int kRing = 24 / (kResident<kParts, kQ> * kCh);
template <int kParts, int kQ> constexpr int kTake = kParts * kQ == 1 ? 2 : 1;

__device__ __forceinline__ uint32_t smem_at(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// The 8 x 8 matrix of 16-bit values that a warp's registers hold, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A float of the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float peer_load(const float *mine, int rank, int cluster) {
  if (cluster == 1)
    return *mine;
  float x;
  asm volatile("{\n .reg .b32 at;\n mapa.shared::cluster.u32 at, %1, %2;\n"
               " ld.shared::cluster.f32 %0, [at];\n}\n"
               : "=f"(x)
               : "r"(smem_at(mine)), "r"(rank)
               : "memory");
  return x;
}

// kE neighbouring ones.
template <int kE>
__device__ __forceinline__ void peer_load(const float *mine, int rank, int cluster, float (&x)[kE]) {
  if (cluster == 1) {
#pragma unroll
    for (int e = 0; e < kE; ++e)
      x[e] = mine[e];
  } else if constexpr (kE == 4) {
    asm volatile("{\n .reg .b32 at;\n mapa.shared::cluster.u32 at, %4, %5;\n"
                 " ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [at];\n}\n"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                 : "r"(smem_at(mine)), "r"(rank)
                 : "memory");
  } else {
    asm volatile("{\n .reg .b32 at;\n mapa.shared::cluster.u32 at, %2, %3;\n"
                 " ld.shared::cluster.v2.f32 {%0, %1}, [at];\n}\n"
                 : "=f"(x[0]), "=f"(x[1])
                 : "r"(smem_at(mine)), "r"(rank)
                 : "memory");
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T, int kCh, int kParts, int kQ>
__global__ void __launch_bounds__(kThreads, kResident<kParts, kQ>)
    kv_decode_kernel(const KvAttendArgs a, const __grid_constant__ CUtensorMap codes) {
  constexpr int kTiles = 4 * kCh;  // 16-element tiles of the head
  constexpr int kLane = 8 * kCh;   // value bytes a lane holds of a token
  constexpr int kG = kTake<kParts, kQ>; // groups a round
  constexpr int kRounds = kRing<kCh, kParts, kQ> / kG; // rounds in the ring
  constexpr int kBytes = kGroupBytes<kCh>;
  constexpr int kRows = 8 * kQ;
  extern __shared__ uint8_t raw[];
  uint8_t *smem = raw + ((1024u - (smem_at(raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[kWarps][kRounds];
  __shared__ float row_m[kWarps][kRows], row_l[kWarps][kRows];
  __shared__ float4 constants[kWarps][32];
  pdl_launch_dependents();
  pdl_wait();
  const KvView &v = a.v;
  const int b = blockIdx.z, split = blockIdx.x;
  const int head = blockIdx.y % v.heads, f0 = blockIdx.y / v.heads * kRows;
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
  const int last = min(f0 + kRows, rows) - 1;
  const int pos_first = offset + f0 / a.group, pos_last = offset + last / a.group;
  int lo, hi;
  key_range(a, s.length, pos_first, pos_last, lo, hi);
  const int first_group = lo >> 4, groups = ((hi + 15) >> 4) - first_group;
  const int each = (groups + a.splits - 1) / a.splits;
  const int begin = first_group + min(groups, split * each) + kG * warp;
  const int end = first_group + min(groups, (split + 1) * each);
  // The warp's i-th group is begin + (i / kG) * kG * kWarps + i % kG; the last
  // round may run past `end` (its groups are then hidden).
  const int count = end > begin ? (end - begin + kG * kWarps - 1) / (kG * kWarps) : 0; // rounds

  uint8_t *ring = smem + warp * kRounds * kG * kBytes;
  if (lane == 0)
    for (int i = 0; i < kRounds; ++i)
      barrier_init(&full[warp][i], 1);
  __syncwarp();
  const int per_page = v.block_log2 - 4; // log2 of the groups a page holds
  // Lane i of a batch of 32 groups holds the page of the warp's i-th group; -1
  // where there is none.
  auto pages_of = [&](int i0) {
    const int i = i0 + lane;
    const int group = begin + i / kG * (kG * kWarps) + i % kG;
    int page = -1;
    if (i < count * kG && group < end) {
      page = kv_page(v, b, group >> per_page);
      if (page < 0)
        atomicOr(a.status, CIM22_STATUS_CACHE_INDEX);
    }
    return page;
  };
  // Query row f0 + 8 t + g, the lane's 16 elements of each 64: on their way
  // before the copies of the codes are.
  Pack<T> query[kQ][kCh * 16 / kVec<T>];
#pragma unroll
  for (int t = 0; t < kQ; ++t) {
    const int f = f0 + 8 * t + g;
    if (f < rows) {
      const int i = f / a.group;
      const T *q = static_cast<const T *>(a.q) + (s.row0 + i) * a.q_row_stride +
                   (head * a.group + f - i * a.group) * a.q_head_stride;
#pragma unroll
      for (int e = 0; e < kCh * 16; e += kVec<T>) {
        const int d = (e / 16) * 64 + 16 * c + e % 16;
        if (d < v.dim) { // head_dim is a multiple of 16
          if (a.q_aligned) {
            query[t][e / kVec<T>].raw = __ldg(reinterpret_cast<const uint4 *>(q + d));
          } else {
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j)
              query[t][e / kVec<T>].at[j] = q[d + j];
          }
        }
      }
    }
  }
  int batch_page = pages_of(0), next_page = -1;
  // One copy a group: 16 tokens of keys and of values (elements past head_dim
  // arrive as zeros). Groups without a page keep what the slot held (any codes
  // are finite, and they are hidden below).
  auto issue = [&](int j, int round) {
    if (j < count) {
      int page[kG], bytes = 0;
#pragma unroll
      for (int u = 0; u < kG; ++u) {
        const int i = j * kG + u;
        page[u] = __shfl_sync(0xffffffffu, (i & 32) == 0 ? batch_page : next_page, i & 31);
        bytes += page[u] >= 0 ? kBytes : 0;
      }
      if (lane == 0) {
        barrier_expect_tx(&full[warp][round], bytes);
#pragma unroll
        for (int u = 0; u < kG; ++u)
          if (page[u] >= 0)
            tma_load_4d(ring + (round * kG + u) * kBytes, &codes, &full[warp][round], 0,
                        ((begin + j * (kG * kWarps) + u) & ((1 << per_page) - 1)) << 4, 2 * head,
                        page[u]);
      }
    }
  };
  next_page = pages_of(32); // (the first rounds take batch_page alone)
#pragma unroll 1
  for (int j = 0; j < kRounds - 1; ++j)
    issue(j, j);

  // Token of row g, and where the lane's bytes of a group lie (comment above).
  const int token = kCh == 2 ? (g >> 1) | (g & 1) << 2 : g;
  const int chunk = kCh == 2 ? token : g; // the lane's 8 * kCh value elements
  const uint32_t k_at = smem_at(ring) + token * 64 * kCh +
                        ((c ^ (kCh == 2 ? token : g >> 1)) << 4);
  const uint32_t v_at = smem_at(ring) + 16 * 64 * kCh +
                        (kCh == 2 ? c * 128 + ((chunk ^ c) << 4)
                                  : 2 * c * 64 + (((g >> 1) ^ c) << 4) + (g & 1) * 8);

  // Query rows f0 + 8 t + g as B fragments (lane (g, c) holds the elements
  // whose codes lane (., c) holds); results come out for rows 2c and 2c + 1.
  uint32_t qb[kQ][kParts][kCh * 4][2];
  float coef[kQ][2];
  int pos[kQ][2];
#pragma unroll
  for (int t = 0; t < kQ; ++t) {
    float x[kCh * 16];
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < kCh * 16; ++e) {
      x[e] = to_f32(query[t][e / kVec<T>].at[e % kVec<T>]);
      amax = nan_max(amax, fabsf(x[e]));
    }
#pragma unroll
    for (int o = 1; o < 4; o *= 2)
      amax = nan_max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float factor, inverse;
    row_factor(amax, factor, inverse);
    // A row with NaN or infinity gives NaN wherever it sees a key.
    const bool wild = !(amax < INFINITY);
    const float mine = wild ? NAN : inverse * a.scale_log2;
#pragma unroll
    for (int e = 0; e < kCh * 16; e += 2) {
      const float y0 = wild ? 0.0f : x[e] * factor, y1 = wild ? 0.0f : x[e + 1] * factor;
      const uint32_t h = pack_half(y0, y1);
      const float2 back = unpack_half(h);
      // Elements 4x .. 4x + 3 of a lane are columns 2c, 2c + 1, 2c + 8, 2c + 9.
      qb[t][0][e / 4][(e & 2) / 2] = h;
      if constexpr (kParts == 2)
        qb[t][1][e / 4][(e & 2) / 2] = pack_half(y0 - back.x, y1 - back.y);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      coef[t][r] = __shfl_sync(0xffffffffu, mine, (2 * c + r) * 4);
      const int fr = f0 + 8 * t + 2 * c + r;
      pos[t][r] = fr < rows ? offset + fr / a.group : -0x40000000;
    }
  }

  float o[kQ][kTiles][4];
  // l sums the lane's own tokens. It takes the probabilities unrounded: where
  // value scales differ, what f16 keeps of a small one is not its weight.
  float m[kQ][2], l[kQ][2];
#pragma unroll
  for (int t = 0; t < kQ; ++t) {
    m[t][0] = m[t][1] = kNone;
    l[t][0] = l[t][1] = 0.0f;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
      o[t][j][0] = o[t][j][1] = o[t][j][2] = o[t][j][3] = 0.0f;
  }
  float widest = -INFINITY; // log2 of the largest value scale met
  // The pages of groups [64 i, 64 i + 32) are in batch_page, of the next 32 in
  // next_page; each is refilled when its last group has been taken.
  int round = 0, parity = 0, issued = min(count, kRounds - 1);
  bool ok = true;
#pragma unroll 1
  for (int j = 0; j < count; ++j) {
    const int i0 = j * kG;
    if ((i0 & 31) == 0) { // scales of groups i0 .. i0 + 31 (their pages are still held)
      const int page = (i0 & 32) == 0 ? batch_page : next_page;
      float4 k = make_float4(0.0f, 0.0f, 1.0f, 0.0f); // hidden
      if (page >= 0) {
        const float2 sc = *reinterpret_cast<const float2 *>(
            v.scales + (static_cast<int64_t>(page) * v.heads + head) * 2);
        const float sv = fmaxf(sc.y, kKvLeastScale);
        k = make_float4(sc.x, log2f(sv), 1.0f / sv, 1.0f);
        widest = fmaxf(widest, k.y);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1)
        widest = fmaxf(widest, __shfl_xor_sync(0xffffffffu, widest, o));
      if (k.w != 0.0f && k.y < widest - kApart)
        k.z = 0.0f;
      __syncwarp();
      constants[warp][lane] = k;
    }
    __syncwarp(); // every lane is done with the slot that is filled next
    issue(j + kRounds - 1, round == 0 ? kRounds - 1 : round - 1);
    issued = min(count, j + kRounds);
    if (((i0 + kG) & 31) == 0) { // this batch's pages are no longer needed
      const int refill = pages_of(i0 + kG + 32);
      if ((i0 & 32) == 0)
        batch_page = refill;
      else
        next_page = refill;
    }
    ok = __all_sync(0xffffffffu, barrier_wait(&full[warp][round], parity));
    if (!ok) {
      // Leave only when the copies in flight have landed, or never will.
      for (int x = j; x < issued; ++x)
        barrier_wait(&full[warp][x % kRounds], (x / kRounds) & 1);
      break;
    }
    const uint32_t slot = round * kG * kBytes;
    round = round + 1 == kRounds ? 0 : round + 1;
    parity ^= round == 0;
    float4 k[kG];
#pragma unroll
    for (int u = 0; u < kG; ++u)
      k[u] = constants[warp][(i0 + u) & 31];

    float sc[kG][kQ][4];
#pragma unroll
    for (int u = 0; u < kG; ++u)
#pragma unroll
      for (int t = 0; t < kQ; ++t) {
        sc[u][t][0] = sc[u][t][1] = sc[u][t][2] = sc[u][t][3] = 0.0f;
      }
#pragma unroll
    for (int ch = 0; ch < kCh; ++ch) {
      uint32_t w[kG][2][4];
#pragma unroll
      for (int u = 0; u < kG; ++u)
#pragma unroll
        for (int z = 0; z < 2; ++z)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[u][z][0]), "=r"(w[u][z][1]), "=r"(w[u][z][2]), "=r"(w[u][z][3])
                       : "r"((k_at ^ (64 * ch)) + slot + u * kBytes + z * 8 * 64 * kCh)
                       : "memory");
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int u = 0; u < kG; ++u) {
          uint32_t f[4];
          codes_to_half(w[u][0][x], f[0], f[2]);
          codes_to_half(w[u][1][x], f[1], f[3]);
#pragma unroll
          for (int t = 0; t < kQ; ++t) {
            if constexpr (kParts == 2)
              mma_f16(sc[u][t], f, qb[t][1][ch * 4 + x][0], qb[t][1][ch * 4 + x][1]);
            mma_f16(sc[u][t], f, qb[t][0][ch * 4 + x][0], qb[t][0][ch * 4 + x][1]);
          }
        }
    }
    // Exponents relative to the rows' references: element e of sc is token
    // t(g) + 8 (e / 2) of its group and row 2c + (e % 2).
    const int key0 = (begin + j * (kG * kWarps)) << 4;
    bool whole = key0 + 16 * kG - 1 < s.length &&
                 (!a.causal || key0 + 16 * kG - 1 <= pos_first) &&
                 key0 >= window_start(a.window, pos_last);
#pragma unroll
    for (int u = 0; u < kG; ++u)
      whole &= k[u].w != 0.0f;
    bool beside = false; // the same for the warp
#pragma unroll
    for (int u = 0; u < kG; ++u)
      beside |= k[u].z == 0.0f;
    uint32_t pb[kG][kQ][kParts][2];
#pragma unroll
    for (int t = 0; t < kQ; ++t) {
      uint32_t hidden = 0;
      if (!whole) {
#pragma unroll
        for (int u = 0; u < kG; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[u].w == 0.0f || !sees(a, s.length, pos[t][e & 1], key0 + 16 * u + token + 8 * (e >> 1)))
              hidden |= 1u << (4 * u + e);
      }
      float arg[kG][4];
      auto arguments = [&] {
#pragma unroll
        for (int u = 0; u < kG; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float slope = coef[t][r] * k[u].x, shift = k[u].y - m[t][r];
            arg[u][r] = fmaf(sc[u][t][r], slope, shift);
            arg[u][r + 2] = fmaf(sc[u][t][r + 2], slope, shift);
          }
        if (!whole) {
#pragma unroll
          for (int u = 0; u < kG; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              arg[u][e] = hidden >> (4 * u + e) & 1 ? -INFINITY : arg[u][e];
        }
      };
      arguments();
      float most = -INFINITY;
#pragma unroll
      for (int u = 0; u < kG; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          most = fmaxf(most, arg[u][e]);
      if (__any_sync(0xffffffffu, most > kGrowth<kParts>)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = -INFINITY;
#pragma unroll
          for (int u = 0; u < kG; ++u)
#pragma unroll
            for (int e = r; e < 4; e += 2)
              if (!(hidden >> (4 * u + e) & 1))
                top = fmaxf(top, fmaf(sc[u][t][e], coef[t][r] * k[u].x, k[u].y));
#pragma unroll
          for (int x = 4; x < 32; x *= 2)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const float to = top - kTop<kParts>;
          if (to > m[t][r]) {
            const float shrink = exp2_approx(m[t][r] - to); // 0 for the first
            l[t][r] = weigh(l[t][r], m[t][r], to);
            m[t][r] = to;
#pragma unroll
            for (int j2 = 0; j2 < kTiles; ++j2) {
              o[t][j2][r] *= shrink;
              o[t][j2][r + 2] *= shrink;
            }
          }
        }
        arguments();
      }
      if (beside) { // weights of groups far below the largest value scale
#pragma unroll
        for (int u = 0; u < kG; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float slope = coef[t][r] * k[u].x;
            const bool hide0 = hidden >> (4 * u + r) & 1, hide1 = hidden >> (4 * u + r + 2) & 1;
            const float best = fmaxf(hide0 ? -INFINITY : sc[u][t][r] * slope,
                                     hide1 ? -INFINITY : sc[u][t][r + 2] * slope);
            if (k[u].z == 0.0f && best > -INFINITY) {
              const float e = ceilf(best);
              l[t][r] += weigh((hide0 ? 0.0f : exp2_approx(fmaf(sc[u][t][r], slope, -e))) +
                                   (hide1 ? 0.0f : exp2_approx(fmaf(sc[u][t][r + 2], slope, -e))),
                               e, m[t][r]);
            }
          }
      }
#pragma unroll
      for (int u = 0; u < kG; ++u) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p[e] = exp2_approx(arg[u][e]);
        l[t][0] = fmaf(p[0] + p[2], k[u].z, l[t][0]);
        l[t][1] = fmaf(p[1] + p[3], k[u].z, l[t][1]);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const uint32_t h = pack_half(p[2 * z], p[2 * z + 1]);
          pb[u][t][0][z] = transpose8(h);
          if constexpr (kParts == 2) {
            const float2 back = unpack_half(h);
            pb[u][t][1][z] = transpose8(pack_half(p[2 * z] - back.x, p[2 * z + 1] - back.y));
          }
        }
      }
    }
    // Values: pairs of tokens at one element.
#pragma unroll
    for (int u = 0; u < kG; ++u) {
      uint32_t w[4][2 * kCh];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if constexpr (kCh == 2)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[t][0]), "=r"(w[t][1]), "=r"(w[t][2]), "=r"(w[t][3])
                       : "r"((v_at ^ (64 * (t & 1))) + slot + u * kBytes +
                             ((t & 1) * 4 + (t >> 1) * 8) * 128)
                       : "memory");
        else
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                       : "=r"(w[t][0]), "=r"(w[t][1])
                       : "r"(v_at + slot + u * kBytes + ((t & 1) + (t >> 1) * 8) * 64)
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
        for (int y = 0; y < 2; ++y) { // rows g and g + 8 are elements 4x + 2y and the next
          const uint32_t f[4] = {h[0][2 * y], h[0][2 * y + 1], h[1][2 * y], h[1][2 * y + 1]};
#pragma unroll
          for (int t = 0; t < kQ; ++t) {
            if constexpr (kParts == 2) {
              // The product's own accumulation does not round to nearest: over
              // many groups in one accumulator that cost f32 outputs half their
              // accuracy (1.2e-6 against 0.7e-6 relative at 1500 keys), so each
              // group's products are added to the sum here.
              float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_f16(part, f, pb[u][t][1][0], pb[u][t][1][1]);
              mma_f16(part, f, pb[u][t][0][0], pb[u][t][0][1]);
#pragma unroll
              for (int z = 0; z < 4; ++z)
                o[t][2 * x + y][z] += part[z];
            } else {
              mma_f16(o[t][2 * x + y], f, pb[u][t][0][0], pb[u][t][0][1]);
            }
          }
        }
      }
    }
  }
  if (!ok && lane == 0)
    atomicOr(a.status, CIM22_STATUS_TIMEOUT);

  // Join the warps of the cluster's CTAs, which hold parts of one key axis:
  // rows [warp][kRows][64 * kCh] in the rings' memory, each CTA finishing every
  // cl-th row from all of them.
  __syncthreads();
  float *joined = reinterpret_cast<float *>(smem);
#pragma unroll
  for (int t = 0; t < kQ; ++t)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = 8 * t + 2 * c + r;
#pragma unroll
      for (int x = 4; x < 32; x *= 2)
        l[t][r] += __shfl_xor_sync(0xffffffffu, l[t][r], x);
      if (g == 0) {
        row_m[warp][row] = m[t][r];
        row_l[warp][row] = l[t][r];
      }
      float2 *to = reinterpret_cast<float2 *>(joined + (warp * kRows + row) * 64 * kCh + kLane * chunk);
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
        to[j] = make_float2(o[t][j][r], o[t][j][r + 2]);
    }
  const int cl = a.cluster, rank = split % cl;
  if (cl > 1)
    cluster_sync();
  else
    __syncthreads();
  // A warp a row, 2 * kCh neighbouring elements a lane.
  constexpr int kE = 2 * kCh;
  const int d = kE * lane;
#pragma unroll 1
  for (int row = rank + cl * warp; row < kRows; row += cl * kWarps) {
    const int f = f0 + row;
    if (f >= rows)
      break;
    // Lane 4 p + x weighs what warp x of CTA p holds.
    const bool there = lane >> 2 < cl;
    const float mine = there ? peer_load(&row_m[lane & 3][row], lane >> 2, cl) : kNone;
    float sum = there ? peer_load(&row_l[lane & 3][row], lane >> 2, cl) : 0.0f;
    float top = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1)
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float share = exp2_approx(mine - top);
    sum = weigh(sum, mine, top);
#pragma unroll
    for (int o = 16; o; o >>= 1)
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float acc[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e)
      acc[e] = 0.0f;
#pragma unroll 2
    for (int p = 0; p < cl; ++p) {
      float part[kWarps][kE];
#pragma unroll
      for (int x = 0; x < kWarps; ++x)
        peer_load(&joined[(x * kRows + row) * 64 * kCh + d], p, cl, part[x]);
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float w = __shfl_sync(0xffffffffu, share, 4 * p + x);
#pragma unroll
        for (int e = 0; e < kE; ++e)
          acc[e] = fmaf(part[x][e], w, acc[e]);
      }
    }
    if (d >= v.dim)
      continue;
    const int i = f / a.group;
    const int64_t at = (s.row0 + i) * a.q_heads + head * a.group + (f - i * a.group);
    if (a.splits > cl) {
      const int64_t to = static_cast<int64_t>(split / cl) * v.rows * a.q_heads + at;
      if (d == 0)
        a.part_ml[to] = make_float2(top, sum);
#pragma unroll
      for (int e = 0; e < kE; ++e)
        a.part_o[to * v.dim + d + e] = acc[e];
    } else {
      const bool some = top > kNone || sum != sum;
      const float scale = some ? 1.0f / sum : 0.0f;
      T *out = static_cast<T *>(a.out) + at * v.dim + d;
#pragma unroll
      for (int e = 0; e < kE; ++e)
        out[e] = from_f32<T>(acc[e] * scale);
      if (a.lse && d == 0)
        a.lse[at] = some ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
    }
  }
  if (cl > 1)
    cluster_sync(); // no CTA leaves while others read its memory
}

// Joins the parts of the key axis. kWarps 4: a CTA a row and head, its warps
// take parts in turn; 1, for up to 8 parts: a warp a row (2 parts of 8,192 rows:
// 10 us less; one row of 32 parts 2 us more).
template <typename T, int kWarps>
__global__ void __launch_bounds__(128) kv_join_kernel(const KvAttendArgs a) {
  __shared__ float2 warp_ml[4];
  __shared__ float4 warp_o[4][32];
  pdl_launch_dependents();
  pdl_wait();
  const KvView &v = a.v;
  const int b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const KvSequence s = kv_sequence(v, b);
  const int64_t f = kWarps == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + warp : blockIdx.x;
  if (!s.ok || f >= static_cast<int64_t>(s.n) * a.q_heads)
    return;
  const int64_t at = s.row0 * a.q_heads + f, step = v.rows * a.q_heads;
  float m = kNone, sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int kAhead = 4;
  const int parts = a.splits / a.cluster;
  for (int x0 = kWarps == 1 ? 0 : warp; x0 < parts; x0 += kWarps * kAhead) {
    float2 ml[kAhead];
    float4 p[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t x = x0 + kWarps * u;
      ml[u] = make_float2(kNone, 0.0f);
      p[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (x < parts) {
        ml[u] = a.part_ml[x * step + at];
        if (4 * lane < v.dim)
          p[u] = *reinterpret_cast<const float4 *>(a.part_o + (x * step + at) * v.dim + 4 * lane);
      }
    }
    float to = m;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      to = fmaxf(to, ml[u].x);
    const float shrink = exp2_approx(m - to);
    sum = weigh(sum, m, to);
    m = to;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc[e] *= shrink;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float share = exp2_approx(ml[u].x - m);
      sum += weigh(ml[u].y, ml[u].x, m);
      acc[0] = fmaf(p[u].x, share, acc[0]);
      acc[1] = fmaf(p[u].y, share, acc[1]);
      acc[2] = fmaf(p[u].z, share, acc[2]);
      acc[3] = fmaf(p[u].w, share, acc[3]);
    }
  }
  float top = m;
  if constexpr (kWarps > 1) {
    if (lane == 0)
      warp_ml[warp] = make_float2(m, sum);
    warp_o[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (warp > 0)
      return;
    top = kNone;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      top = fmaxf(top, warp_ml[x].x);
    sum = acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float2 ml = warp_ml[x];
      const float4 p = warp_o[x][lane];
      const float share = exp2_approx(ml.x - top);
      sum += weigh(ml.y, ml.x, top);
      acc[0] = fmaf(p.x, share, acc[0]);
      acc[1] = fmaf(p.y, share, acc[1]);
      acc[2] = fmaf(p.z, share, acc[2]);
      acc[3] = fmaf(p.w, share, acc[3]);
    }
  }
  const bool some = top > kNone || sum != sum;
  const float share = some ? 1.0f / sum : 0.0f;
  if (4 * lane < v.dim) {
    const float o[4] = {acc[0] * share, acc[1] * share, acc[2] * share, acc[3] * share};
    T *out = static_cast<T *>(a.out) + at * v.dim + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      out[j] = from_f32<T>(o[j]);
  }
  if (a.lse && lane == 0)
    a.lse[at] = some ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
}

// Parts of the key axis: as many as keep all work items resident at once (one
// more would start a second round of CTAs), each of at least 128 keys. Items
// that fill every place by themselves are halved once, which evens out
// sequences of unequal length (64 of 1,000-8,191 tokens, 8 kv heads: 141 -> 131
// us); fewer are left whole (32 of 4,000 in f32: 76 us, halved 94). Parts are joined within the kernel as clusters:
// all of them up to four, up to eight at a time where every CTA has an SM to
// itself, else in pairs (larger clusters leave places on the SMs empty: one
// sequence of 200,000 tokens 60 -> 76 us with eight), and the rest by
// kv_join_kernel.
void decode_parts(const KvView &v, int64_t tiles, int64_t longest, int resident, int &splits,
                  int &cluster) {
  const int64_t items = std::max<int64_t>(1, tiles * v.heads * v.batch), slots = 148 * resident;
  const int64_t want = 2 * items > slots
                           ? std::min<int64_t>(items >= slots && items < 4 * slots ? 2 : 1, longest / 512)
                           : std::min<int64_t>(slots / items, (longest + 127) / 128);
  splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, 256)));
  if (splits <= 4 || (splits <= 8 && items * splits <= 148))
    cluster = splits;
  else
    cluster = items * splits <= 148 ? 8 : 2;
  splits = splits / cluster * cluster;
}

// The same for prompts, where a CTA fills an SM: the number that takes the least
// time, counted in tiles of 128 keys (2.8 us, 2.1 with head_dim 64). A round of
// CTAs lasts as long as its tiles and some five more for filling and emptying;
// joining takes two and the parts' way through memory. (3 sequences of 6,000,
// window 4,096, 700 new tokens, 24 heads of 64: 216 CTAs 223 us, halved 199; one
// of 1,000, 8 heads of 128: 49 us, in 4 parts 39.)
int prompt_parts(const KvView &v, int64_t tiles, int64_t tile_rows, int64_t group, int64_t longest,
                 int64_t window) {
  const int64_t items =
      v.heads * std::min<int64_t>(tiles * v.batch, v.rows * group / tile_rows + v.batch);
  const int64_t span =
      ((window ? std::min(longest, window + tile_rows / group) : longest) + 127) / 128;
  const double join = static_cast<double>(items * tile_rows * v.dim) * 8.0 / 12.5e6;
  int64_t best = 1;
  double least = 0.0;
  for (int64_t parts = 1; parts <= std::min<int64_t>(64, span); ++parts) {
    const int64_t rounds = (items * parts + 147) / 148;
    if (parts > 1 && rounds > 6)
      break;
    const double cost =
        static_cast<double>(rounds) * static_cast<double>((span + parts - 1) / parts + 5) +
        (parts > 1 ? 2.0 + join * static_cast<double>(parts) : 0.0);
    if (parts == 1 || cost < (best == 1 ? 0.96 : 1.0) * least) {
      least = cost;
      best = parts;
    }
  }
  return static_cast<int>(best);
}

struct Plan {
  bool prompt; // by the tensor-memory kernel
  bool share;  // with one query tile a CTA
  bool few;    // decode tiles of 8 query rows, not 16
  int splits;  // parts of the key axis,
  int cluster; // so many of them joined within the kernel
  int64_t tiles;
  size_t bytes; // of the workspace: the parts' results, then
  size_t carry; // what f32 prompts carry from tile to tile (0: nothing)
};

// Up to kDecodeRows query rows a sequence and kv head go to the decode kernel
// (decode | prompt, head_dim 128, bf16, 8 kv heads, L2 flushed: 32 sequences of
// 4,096 with 32 rows 145 | 197 us, 48 rows 195 | 199, 64 rows 244 | 197; one of
// 32,768 46 | 63, 58 | 65, 75 | 65). So do more rows where all of its tiles of 16
// have a place at once and come to kDecodeWork keys: the prompt kernel takes some
// 15 us to fill and empty (one sequence of 1,000 with 256 rows 25 | 33 us, 4 with
// 64 rows 27 | 28; twice that work, one of 4,000 with 128 rows 36 | 30; more tiles
// than places, 16 of 300 with 64 rows, 37 | 27).
constexpr int64_t kDecodeRows = 32, kDecodeWork = 1 << 17;

// Rows that a launch is sized for: one at least, since a sequence with more rows
// than the bound is reported by the kernels.
int64_t most_rows(const KvView &v) { return std::max<int64_t>(1, std::min<int64_t>(v.most, v.rows)); }

Plan attend_plan(const KvView &v, const cim22_kv_attention &t) {
  Plan p{};
  const int64_t group = t.q_heads / v.heads;
  const int64_t rows = most_rows(v) * group;
  const int64_t held = static_cast<int64_t>(v.table_width) << v.block_log2;
  const int64_t longest = std::max<int64_t>(1, std::min(t.longest, held));
  const int64_t tiles16 = (rows + 15) / 16 * v.heads * v.batch;
  const int resident = t.type == CIM22_FLOAT32 && rows > 8 ? 2 : 3;
  p.prompt =
      rows > kDecodeRows && (tiles16 > 148 * resident || tiles16 * longest > kDecodeWork);
  // One query tile a CTA up to 128 rows: 32 sequences of 4,096 with 64 rows 199
  // us, as two half-empty tiles 285; 192 rows the other way round, 363 and 260.
  p.share = p.prompt && (t.type == CIM22_FLOAT32 || rows <= 128);
  if (!p.prompt) {
    p.few = rows <= 8;
    p.tiles = (rows + (p.few ? 7 : 15)) / (p.few ? 8 : 16);
    decode_parts(v, p.tiles, longest, resident, p.splits, p.cluster);
  } else {
    p.tiles = (rows + (p.share ? 127 : 255)) / (p.share ? 128 : 256);
    p.cluster = 1;
    p.splits = prompt_parts(v, p.tiles, p.share ? 128 : 256, group, longest, t.window);
  }
  const int parts = p.splits / p.cluster;
  p.bytes = parts == 1 ? 0
                       : static_cast<size_t>(parts) * v.rows * t.q_heads *
                             (static_cast<size_t>(v.dim) * 4 + 8);
  // More than two tiles of 128 keys for each of a CTA's two streams, by what the
  // table can hold: `longest` may be any value, and without this the sums of
  // a longer sequence would lose accuracy (4.8e-6 over 8,192 keys).
  if (p.prompt && t.type == CIM22_FLOAT32 && (held + p.splits - 1) / p.splits > 512) {
    p.bytes = (p.bytes + 15) / 16 * 16;
    p.carry = static_cast<size_t>(p.splits) * 2 * v.rows * t.q_heads * (v.dim > 64 ? 128 : 64) * 4;
    p.bytes += p.carry;
  }
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
  if (most_rows(v) * (t->q_heads / v.heads) > 0x3fffffff)
    return refuse("too many query rows");
  return true;
}

template <typename T, int kCh, int kParts, int kQ>
cudaError_t launch_decode(const KvAttendArgs &a, int64_t tiles, cudaStream_t stream) {
  constexpr size_t bytes =
      static_cast<size_t>(kWarps) * kRing<kCh, kParts, kQ> * kGroupBytes<kCh> + 1024;
  const auto kernel = kv_decode_kernel<T, kCh, kParts, kQ>;
  static DynamicSmem allowed;
  if (const cudaError_t e = allowed.allow(kernel, bytes); e != cudaSuccess)
    return e;
  CUtensorMap codes;
  if (!tc::encode_kv_groups(&codes, a.v.codes, a.v.dim, 1 << a.v.block_log2, 2 * a.v.heads,
                            a.v.pages, 64 * kCh))
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits, static_cast<unsigned>(tiles * a.v.heads), a.v.batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, codes);
}

template <typename T, int kParts, int kQ>
cudaError_t launch_decode(const KvAttendArgs &a, int64_t tiles, cudaStream_t stream) {
  return a.v.dim > 64 ? launch_decode<T, 2, kParts, kQ>(a, tiles, stream)
                      : launch_decode<T, 1, kParts, kQ>(a, tiles, stream);
}

template <typename T, int kParts>
cudaError_t launch_attend(const KvAttendArgs &a, int type, const Plan &plan, cudaStream_t stream) {
  cudaError_t e =
      plan.prompt ? kv_prompt_launch(a, type, plan.share, static_cast<int>(plan.tiles), stream)
      : plan.few  ? launch_decode<T, kParts, 1>(a, plan.tiles, stream)
                  : launch_decode<T, kParts, 2>(a, plan.tiles, stream);
  if (e == cudaSuccess && a.splits > a.cluster) {
    const int64_t rows = most_rows(a.v) * a.q_heads;
    e = a.splits / a.cluster <= 8
            ? launch_pdl(kv_join_kernel<T, 1>, dim3(static_cast<unsigned>((rows + 3) / 4), 1, a.v.batch),
                         dim3(128), 0, stream, a)
            : launch_pdl(kv_join_kernel<T, 4>, dim3(static_cast<unsigned>(rows), 1, a.v.batch),
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
  if (plan.tiles * v.heads > 0x7fffffff) { // (decode's fit its axis by the choice above)
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
  a.q_aligned = (reinterpret_cast<uintptr_t>(a.q) |
                 (a.q_row_stride | a.q_head_stride) * float_size(attention->type)) % 16 == 0;
  a.causal = attention->causal != 0;
  a.window = attention->window;
  a.splits = plan.splits;
  a.cluster = plan.cluster;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = plan.splits > plan.cluster ? reinterpret_cast<float2 *>(a.part_o + static_cast<size_t>(plan.splits / plan.cluster) * v.rows * a.q_heads * v.dim)
                         : nullptr;
  a.carry = plan.carry ? reinterpret_cast<float *>(static_cast<char *>(workspace) + (plan.bytes - plan.carry))
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
