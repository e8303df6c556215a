// kv_attention_tc.cu - attention of prompts and chunks over the 8-bit cache on
// the tensor cores (tcgen05, operands and accumulators in TMEM).
//
// Bound by the tensor cores, shared memory and the exponentials, about equally:
// 128 rows x 128 keys (head_dim 128) take 2 x 512 cycles of f16 products, whose
// operands fill shared memory's 128 bytes a cycle, and 1,024 of the
// special-function units. A CTA therefore runs two streams of 128 query rows,
// so that one's products cover the other's softmax (a prompt of 8,192, 32 heads
// of 128 on 8, bf16: 0.65 ms, 844 TFLOP/s, in ten calls, 0.69 ms, 797, once the
// clock falls at the power limit; 3 chunks of 1,024 each in a window of 4,096, 24
// heads of 64: 171 us, 451, and of 1,024 and less 194 us, 240):
//   warps 0-7, 8-15 softmax of stream 0 and 1: two threads a row, one for each
//                   64 keys of a tile, scores from TMEM, probabilities back over
//                   them as the f16 A operand (one thread a row left too few
//                   warps to keep the special-function units busy)
//   warps 16-19     converters: 64 tokens of keys, then of values, at a time,
//                   int8 codes (16 bytes a load, exact in f16) into
//                   128-byte-swizzled tiles of 128 tokens, two each
//   warp 20         issues the products: S = Q K^T, then O += P V
//   warp 21         looks up the pages and scales of the tokens to come
// (Two buffers of 64 keys a stream, which let products run ahead, were slower:
// a product of 64 keys still reads all of its query tile. So were all 128
// scores of a row in registers, with or without more registers for these
// warps, and warps of their own for keys and for values: 0.66 ms. The queries
// read by the softmax warps alone, while the converters start, took 0.71.)
// Query rows are the tokens of a sequence times the heads that share a kv
// head, so a tile of keys is converted once for up to 256 rows. The codes'
// scales stay out of the products: a group of 16 tokens lies in one page, and
// its key scale multiplies the scores, its value scale goes into the exponent
// (kv_attention.h).
// kShare: both streams take the same 128 rows and alternate tiles of keys, and
// their results are joined at the end. It serves few rows, and f32 queries,
// whose rows are two f16 parts and need the second tile's shared memory.
#include "kv_attention.h"
#include "kv_convert.h"

#include <algorithm>
#include <type_traits>

namespace cim {
namespace {

constexpr int kThreads = 768, kM = 128, kTile = 128; // query rows a stream, keys a tile
constexpr int kSub = 64, kIndex = 8; // tokens converted at a time, and indexed ahead
constexpr int kPanel = 128 * 128;    // bytes: 128 rows of 64 f16
// The products' accumulation does not round to nearest: f32 outputs lost half
// their accuracy to it over 1,500 keys (1.25e-6 relative; 4.8e-6 over 8,192). With
// two parts a stream's sum is therefore taken out of the accumulators every
// kFlush tiles and added to what it carries in memory, rounding to nearest
// (0.7e-6 over 1,800 keys; 5 prompts of up to 1,500, 16 heads of 80 on 4: 129 ->
// 161 us, now 166).
constexpr int kFlush = 2;
constexpr uint64_t kWaitLimit = 2000000000ull; // ns

template <int kCh> struct alignas(1024) PromptSmem {
  uint8_t q[2][kCh * kPanel]; // query tiles, or the two parts of one
  uint8_t kv[2][2][kCh * kPanel]; // keys and values of tile j at j % 2
  // Of the groups of 16 tokens of part j (64 tokens) at j % kIndex: key scale, log2 and inverse of the
  // value scale, and where the keys begin in units of a group's keys (-1: none).
  float4 scale[kIndex][kSub / 16];
  float coef[2 * kM];            // what turns a row's product into an exponent
  float join[2][kM], sums[2][2][kM];
  float tops[2][2][2][kM];       // [tile % 2][stream][half]
  uint64_t kv_full[2][4], kv_empty[2][2]; // of parts and of tiles
  uint64_t index_full[kIndex], index_empty[kIndex];
  uint64_t s_full[2], p_full[2], o_full[2], done;
  uint32_t tmem;
  int failed;
  uint2 range[16]; // least and largest value scale (bits) that each softmax warp found
};

__device__ __forceinline__ uint32_t smem_at(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(bar)), "r"(count));
}

__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(bar)) : "memory");
}

// Waits for the phase of the given parity, for at most kWaitLimit of the
// global timer; gives up sooner when another role has. The first try is all
// that most waits need; what follows is kept out of line and short, since the
// waiting warps' polls compete with the working ones for issue slots.
__device__ __forceinline__ bool bar_try(uint32_t at, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
               " selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(done)
               : "r"(at), "r"(parity)
               : "memory");
  return done;
}

__device__ __noinline__ bool bar_wait_long(uint32_t at, uint32_t parity, int *failed) {
  uint64_t start = 0;
  while (!bar_try(at, parity)) {
    uint64_t now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (start == 0)
      start = now;
    if (now - start > kWaitLimit || *reinterpret_cast<volatile int *>(failed)) {
      *reinterpret_cast<volatile int *>(failed) = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, int *failed) {
  const uint32_t at = smem_at(bar);
  return bar_try(at, parity) || bar_wait_long(at, parity, failed);
}

// Matrix descriptors, 128-byte swizzle. K-major (queries, keys): rows of 128
// bytes in 1024-byte atoms. MN-major (values): a row holds 64 elements of one
// token; 64-element panels kPanel apart, 8-token atoms 1024 bytes apart. The
// low word counts the address in 16 bytes, so a step within a tile is an
// addition to it; the high word is a constant.
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k_major(uint32_t at) { return (at & 0x3ffff) >> 4; }
__device__ __forceinline__ uint32_t desc_mn_major(uint32_t at) {
  return desc_k_major(at) | (kPanel >> 4) << 16;
}

// kind::f16 with f16 A and B and f32 accumulators (format 1 at bit 4); B is
// MN-major with bit 16.
constexpr uint32_t idesc_f16(int m, int n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n"
               " mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
               "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
               : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n"
               " mov.b64 b, {%2, %5};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d),
               "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
               : "memory");
}

// One thread of a converged warp.
__device__ __forceinline__ bool elect() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(yes));
  return yes != 0;
}

__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_at(bar))
      : "memory");
}

__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, "
               "%9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
               "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
                 "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                 "=r"(r[30]), "=r"(r[31])
               : "r"(at)
               : "memory");
}

// 16 columns without waiting: tmem_loaded() orders the registers' use.
__device__ __forceinline__ void tmem_load_start(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, "
               "%9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at)
               : "memory");
}

__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// a * b + c and a + b of pairs, each half rounding as the scalar operation.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Score to exponent: a positive slope (of nearly nothing where the row or the
// scale is zero) leaves what is hidden at -infinity.
__device__ __forceinline__ float score_slope(float coef, float key_scale) {
  const float slope = coef * key_scale;
  return slope < 1e-37f ? 1e-37f : slope;
}

// In the order written: all of a tile's at once would not leave registers for
// its scores.
__device__ __forceinline__ float4 load_scale(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(at)
               : "memory");
}

__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// 2^x of a pair on the FMA units, which are idle while the special-function
// units work at their limit: n = rint(x) by adding 1.5 * 2^23, a polynomial in
// f = x - n of [-0.5, 0.5] (least largest relative error, fitted by reweighted
// least squares: 2.7e-6), n added to the exponent bits. Below 2^-120 it stays
// there, hidden keys included: in f16 that is 0, and to l it adds at most
// 2^(kApart - 126) of the row's largest weight a key.
__device__ __forceinline__ float2 exp2_pair(float2 x) {
  x.x = fmaxf(x.x, -120.0f);
  x.y = fmaxf(x.y, -120.0f);
  const float2 magic = make_float2(12582912.0f, 12582912.0f);
  const float2 r = add2(x, magic);
  const float2 n = add2(r, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 p = fma2(f, make_float2(9.5701022e-3f, 9.5701022e-3f), make_float2(5.5917863e-2f, 5.5917863e-2f));
  p = fma2(p, f, make_float2(0.24024744f, 0.24024744f));
  p = fma2(p, f, make_float2(0.69312179f, 0.69312179f));
  p = fma2(p, f, make_float2(0.99999928f, 0.99999928f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(r.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(r.y) << 23)));
}

__device__ __forceinline__ void tmem_stored() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// The weights, relative to 2^m, of a row's keys in groups far below the largest
// value scale, of 64 keys whose scores lie at `scores` in TMEM. The row sees keys
// from .. to - 1 of them.
__device__ __noinline__ float apart_weights(uint32_t scores, uint32_t scales, float far, int from,
                                            int to, float coef, float m) {
  float l = 0.0f;
  for (int g = 0; g < kSub / 16; ++g) {
    const float4 sc = load_scale(scales + 16 * g);
    if (!(sc.y < far) || sc.y == -INFINITY) // the same for the warp
      continue;
    const float slope = score_slope(coef, sc.x);
    for (int c = 16 * g; c < 16 * (g + 1); c += 8) {
      uint32_t y[8];
      tmem_load8(scores + c, y);
      float best = -INFINITY, w = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i >= from && c + i < to)
          best = fmaxf(best, __uint_as_float(y[i]));
      if (best > -INFINITY) {
        const float e = ceilf(best * slope);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i >= from && c + i < to)
            w += exp2_approx(fmaf(__uint_as_float(y[i]), slope, -e));
        l += weigh(w, e, m);
      }
    }
  }
  return l;
}

// kCount neighbouring elements of a query row as f32, zero from `dim` on.
template <typename T, int kCount>
__device__ __forceinline__ void load_few(const T *row, int d, int dim, bool aligned,
                                         float (&x)[kCount]) {
  constexpr int kBytes = kCount * static_cast<int>(sizeof(T));
  union {
    uint32_t raw[kBytes / 4];
    T at[kCount];
  } p;
#pragma unroll
  for (int i = 0; i < kBytes / 4; ++i)
    p.raw[i] = 0;
  if (d < dim) { // head_dim is a multiple of 16: all or nothing
    if (!aligned) {
#pragma unroll
      for (int i = 0; i < kCount; ++i)
        p.at[i] = row[d + i];
    } else if constexpr (kBytes == 16) {
      *reinterpret_cast<uint4 *>(p.raw) = __ldg(reinterpret_cast<const uint4 *>(row + d));
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2 *>(p.raw) = __ldg(reinterpret_cast<const uint2 *>(row + d));
    } else {
      p.raw[0] = __ldg(reinterpret_cast<const uint32_t *>(row + d));
    }
  }
#pragma unroll
  for (int i = 0; i < kCount; ++i)
    x[i] = to_f32(p.at[i]);
}

template <typename T, int kCh, int kParts, bool kShare>
__global__ void __launch_bounds__(kThreads, 1) kv_prompt_kernel(const KvAttendArgs a, int tiles) {
  static_assert(kParts == 1 || kShare, "two query tiles of two parts do not fit");
  extern __shared__ uint8_t raw[];
  PromptSmem<kCh> &sm =
      *reinterpret_cast<PromptSmem<kCh> *>(raw + ((1024u - (smem_at(raw) & 1023u)) & 1023u));
  const KvView &v = a.v;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kRows = kShare ? kM : 2 * kM; // query rows of this CTA
  constexpr int kD = 64 * kCh;
  if (threadIdx.x == 0) {
    for (int side = 0; side < 2; ++side) {
      for (int i = 0; i < 4; ++i)
        bar_init(&sm.kv_full[side][i], 128);
      for (int i = 0; i < 2; ++i)
        bar_init(&sm.kv_empty[side][i], 1);
    }
    for (int i = 0; i < kIndex; ++i) {
      bar_init(&sm.index_full[i], 1);
      // The converters' warps, and those of the streams that take the part.
      bar_init(&sm.index_empty[i], 4 + (kShare ? 4 : 8));
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&sm.s_full[i], 1);
      bar_init(&sm.p_full[i], 256);
      bar_init(&sm.o_full[i], 1);
    }
    bar_init(&sm.done, 1);
    sm.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.z, split = blockIdx.y;
  const int head = blockIdx.x % v.heads;
  // The last tiles of a causal prompt see the most keys: they start first.
  const int f0 = (tiles - 1 - static_cast<int>(blockIdx.x / v.heads)) * kRows;
  const KvSequence s = kv_sequence(v, b);
  if (!s.ok) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0)
      atomicOr(a.status, CIM22_STATUS_CACHE_INDEX);
    return;
  }
  const int rows = s.n * a.group;
  if (f0 >= rows)
    return;
  if (warp == 20) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_at(&sm.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int offset = s.length - s.n;
  const int last = min(f0 + kRows, rows) - 1;
  int lo, hi;
  key_range(a, s.length, offset + f0 / a.group, offset + last / a.group, lo, hi);
  const int first16 = lo >> 4;
  const int all = (((hi + 15) >> 4) - first16 + kTile / 16 - 1) / (kTile / 16); // tiles
  const int each = (all + a.splits - 1) / a.splits;
  const int tile0 = min(all, split * each), count = min(all, tile0 + each) - tile0;
  const int key_base = (first16 << 4) + tile0 * kTile; // of this CTA's tile 0

  // The softmax warps look over the value scales: a page's table entry before
  // the queries, its scale after them, so that neither is waited for.
  const int first_page = key_base >> v.block_log2;
  const int pages =
      count > 0 ? ((min(key_base + count * kTile, s.length) - 1) >> v.block_log2) - first_page + 1 : 0;
  auto entry = [&](int i) { return v.table[b * v.table_stride + first_page + i]; };
  auto value_scale = [&](int page) { // 0: no such page
    return page >= 0 && page < v.pages
               ? fmaxf(v.scales[(static_cast<int64_t>(page) * v.heads + head) * 2 + 1], kKvLeastScale)
               : 0.0f;
  };
  const int thread = static_cast<int>(threadIdx.x);
  int page = -1; // not looked at until the queries are done
  if (thread < min(pages, 512))
    page = entry(thread);

  // Queries: a warp takes every 24th row, a lane 2 * kCh neighbouring elements.
  const bool negative = a.scale_log2 < 0.0f; // the products then take -q
#pragma unroll 4
  for (int r = warp; r < kRows; r += kThreads / 32) {
    constexpr int kE = 2 * kCh;
    const int f = f0 + r;
    const int d = kE * lane;
    float x[kE];
#pragma unroll
    for (int i = 0; i < kE; ++i)
      x[i] = 0.0f;
    if (f < rows) {
      const int i = f / a.group;
      load_few<T, kE>(static_cast<const T *>(a.q) + (s.row0 + i) * a.q_row_stride +
                          (head * a.group + f - i * a.group) * a.q_head_stride,
                      d, v.dim, a.q_aligned, x);
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kE; ++i)
      amax = nan_max(amax, fabsf(x[i]));
#pragma unroll
    for (int o = 16; o; o >>= 1)
      amax = nan_max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    // A row with NaN or infinity gives NaN wherever it sees a key.
    const bool wild = !(amax < INFINITY);
    float factor, inverse;
    row_factor(wild ? 0.0f : amax, factor, inverse);
    if (lane == 0)
      sm.coef[r] = wild ? NAN : inverse * fabsf(a.scale_log2);
    if (negative)
      factor = -factor;
    uint32_t h[kE / 2], l[kE / 2];
#pragma unroll
    for (int i = 0; i < kE; i += 2) {
      const float y0 = wild ? 0.0f : x[i] * factor, y1 = wild ? 0.0f : x[i + 1] * factor;
      h[i / 2] = pack_half(y0, y1);
      const float2 back = unpack_half(h[i / 2]);
      l[i / 2] = pack_half(y0 - back.x, y1 - back.y);
    }
    uint8_t *to = sm.q[kShare ? 0 : r / kM] + (d / 64) * kPanel + (r % kM) * 128 +
                  ((((d % 64) / 8) ^ (r & 7)) << 4) + (d % 8) * 2;
    if constexpr (kCh == 2) {
      *reinterpret_cast<uint2 *>(to) = make_uint2(h[0], h[1]);
      if constexpr (kParts == 2)
        *reinterpret_cast<uint2 *>(to + kCh * kPanel) = make_uint2(l[0], l[1]);
    } else {
      *reinterpret_cast<uint32_t *>(to) = h[0];
      if constexpr (kParts == 2)
        *reinterpret_cast<uint32_t *>(to + kCh * kPanel) = l[0];
    }
  }
  const float first_scale = value_scale(page);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0); // columns: scores [stream][128], outputs [stream][kD]
  int *failed = &sm.failed;
  if (warp < 16) {
    // ------------------------------------------------------------- softmax
    // The range of the value scales decides how the weights are summed.
    uint32_t least = 0x7f800000u, most = 0; // bits: they are positive
    auto widen = [&](float scale) {
      least = min(least, scale > 0.0f ? __float_as_uint(scale) : least);
      most = max(most, __float_as_uint(scale));
    };
    widen(first_scale);
    for (int i = thread + 512; i < pages; i += 512)
      widen(value_scale(entry(i)));
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0)
      sm.range[warp] = make_uint2(least, most);
    asm volatile("bar.sync 1, 512;" ::: "memory");
    const uint2 range = sm.range[lane & 15];
    least = __reduce_min_sync(0xffffffffu, range.x);
    most = __reduce_max_sync(0xffffffffu, range.y);
    const float far = log2f(__uint_as_float(most)) - kApart; // -infinity: no scales
    const bool apart = log2f(__uint_as_float(least)) < far;

    const int st = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + st * kTile + lanes, o_at = tmem + 2 * kTile + st * kD + lanes;
    const int f = f0 + (kShare ? 0 : st * kM) + row;
    const bool live = f < rows;
    const int pos = offset + (live ? f / a.group : 0);
    const int row_hi = !live ? 0 : a.causal ? min(s.length, pos + 1) : s.length;
    const int row_lo = window_start(a.window, pos);
    // A row that sees nothing takes no NaN from its query: what is hidden stays so.
    const float coef = row_lo < row_hi ? sm.coef[kShare ? row : st * kM + row] : 0.0f;
    float m = kNone, l = 0.0f;
    // What the stream carries: [split][stream][kv head][element][packed row],
    // to be multiplied by `carried`.
    const int64_t plane = v.rows * a.group;
    float *carry = kParts == 2 && a.carry
                       ? a.carry + ((static_cast<int64_t>(split) * 2 + st) * v.heads + head) * kD * plane +
                             s.row0 * a.group + (live ? f : 0)
                       : nullptr;
    float carried = 0.0f; // nothing yet
    const int mine = kShare ? (count - st + 1) / 2 : count;
    bool ok = true;
    auto take = [&](auto with_apart, int n) { // the stream's n-th tile
      const int tile = kShare ? 2 * n + st : n;
      const int key0 = key_base + tile * kTile;
      const int from = min(max(row_lo - key0, 0), kTile), to = min(max(row_hi - key0, 0), kTile);
      const bool whole =
          __all_sync(0xffffffffu, from <= kSub * half && to >= kSub * (half + 1));
      const int part0 = (2 * tile + half) % kIndex;
      // After a wait that ran out the loop goes on (later ones then return at
      // once): the other half's warp meets this one at a barrier in each round.
      ok = bar_wait(&sm.index_full[part0], ((2 * tile + half) / kIndex) & 1, failed) && ok;
      ok = bar_wait(&sm.s_full[st], n & 1, failed) && ok;
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t scale_at = smem_at(sm.scale[part0]); // of the half's four groups
      auto hide = [&](int g, uint32_t (&y)[16]) {
        const int key = kSub * half + 16 * g;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          y[i] = key + i >= from && key + i < to ? y[i] : 0xff800000u; // -infinity
      };
      // A new reference for the rows that outgrew theirs (the first is kNone).
      auto refer = [&](bool grown, float to) {
        const float shrink = grown ? exp2_approx(m - to) : 1.0f; // 0 for the first
        l = grown ? weigh(l, m, to) : l;
        m = grown ? to : m;
        carried *= shrink;
        if (n > 0 && !(carry && n % kFlush == 0)) {
          ok = bar_wait(&sm.o_full[st], (n - 1) & 1, failed) && ok;
          __syncwarp();
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int c = half * 4 * kCh; c < (half + 1) * 4 * kCh; ++c) { // its half of O
            uint32_t y[8];
            tmem_load8(o_at + 8 * c, y);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              y[i] = __float_as_uint(__uint_as_float(y[i]) * shrink);
            tmem_store8(o_at + 8 * c, y);
          }
        }
      };
      // The scores are read once for the largest exponent and once more for the
      // probabilities, 16 (a group of one scale) at a time with the next 16 on
      // their way.
      const uint32_t from_at = s_at + kSub * half;
      uint32_t x[2][16];
      float top = -INFINITY, slopes[4];
      tmem_load_start(from_at, x[0]);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t(&y)[16] = x[g & 1];
        tmem_loaded(y);
        tmem_load_start(from_at + 16 * ((g + 1) & 3), x[(g & 1) ^ 1]); // at last group 0 again
        if (!whole)
          hide(g, y);
        float best = max3(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
        float next = max3(__uint_as_float(y[3]), __uint_as_float(y[4]), __uint_as_float(y[5]));
#pragma unroll
        for (int i = 6; i < 14; i += 4) {
          best = max3(best, __uint_as_float(y[i]), __uint_as_float(y[i + 1]));
          next = max3(next, __uint_as_float(y[i + 2]), __uint_as_float(y[i + 3]));
        }
        best = max3(best, __uint_as_float(y[14]), __uint_as_float(y[15]));
        const float4 sc = load_scale(scale_at + g * 16);
        slopes[g] = score_slope(coef, sc.x);
        top = fmaxf(top, fmaf(fmaxf(best, next), slopes[g], sc.y));
      }
      // Both halves of a row have one reference.
      sm.tops[n & 1][st][half][row] = top;
      asm volatile("bar.sync %0, 64;" ::"r"(2 + st * 4 + (warp & 3)) : "memory");
      top = fmaxf(top, sm.tops[n & 1][st][half ^ 1][row]);
      if (kParts == 2 && carry && n > 0 && n % kFlush == 0) {
        // What is carried is read kAhead steps of 8 elements before it is used (a
        // prompt of 4,096, 32 heads of 128: 544 us read in place, 477 so, now 488).
        constexpr int kSteps = kD / 16, kAhead = 2;
        const int d0 = half * (kD / 2), end = min(d0 + kD / 2, v.dim);
        float old[kAhead][8];
        auto fetch = [&](int step) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float &to = old[step % kAhead][i];
            to = 0.0f;
            if (live && n > kFlush && d0 + 8 * step < end)
              to = carry[(d0 + 8 * step + i) * plane];
          }
        };
#pragma unroll
        for (int step = 0; step < kAhead; ++step)
          fetch(step);
        ok = bar_wait(&sm.o_full[st], (n - 1) & 1, failed) && ok;
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          const int d = d0 + 8 * step;
          if (d >= end)
            break;
          uint32_t y[8];
          tmem_load8(o_at + d, y);
          if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              carry[(d + i) * plane] = fmaf(old[step % kAhead][i], carried, __uint_as_float(y[i]));
          }
          if (step + kAhead < kSteps)
            fetch(step + kAhead);
        }
        carried = 1.0f;
      }
      const bool grown = top > (m == kNone ? -INFINITY : m + kGrowth<kParts>);
      if (__any_sync(0xffffffffu, grown))
        refer(grown, top - kTop<kParts>);
      if constexpr (decltype(with_apart)::value) {
        tmem_loaded(x[0]);
        l += apart_weights(from_at, scale_at, far, from - kSub * half, to - kSub * half, coef, m);
        tmem_load_start(from_at, x[0]);
      }
      const float origin = m == kNone ? 0.0f : m;
      // Probabilities over the scores: of every 32 columns 16 hold their f16,
      // the next 16 the small parts.
      uint32_t low[8];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t(&y)[16] = x[g & 1];
        tmem_loaded(y);
        // The small parts of an even group go over the next group's scores,
        // which have been read by now.
        if (kParts == 2 && (g & 1))
          tmem_store8(from_at + (g >> 1) * 32 + 16, low);
        if (g < 3)
          tmem_load_start(from_at + 16 * (g + 1), x[(g & 1) ^ 1]);
        if (!whole)
          hide(g, y);
        const float4 sc = load_scale(scale_at + g * 16);
        const float slope = slopes[g], shift = sc.y - origin;
        uint32_t high[8];
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 e = fma2(make_float2(__uint_as_float(y[i]), __uint_as_float(y[i + 1])),
                                make_float2(slope, slope), make_float2(shift, shift));
          const float2 q = kParts == 1 && i % 8 == 6
                               ? exp2_pair(e)
                               : make_float2(exp2_approx(e.x), exp2_approx(e.y));
          sum = add2(sum, q);
          high[i / 2] = pack_half(q.x, q.y);
          if constexpr (kParts == 2) {
            const float2 back = unpack_half(high[i / 2]);
            low[i / 2] = pack_half(q.x - back.x, q.y - back.y);
          }
        }
        l = fmaf(sum.x + sum.y, decltype(with_apart)::value && sc.y < far ? 0.0f : sc.z, l);
        const uint32_t at = from_at + (g >> 1) * 32 + (g & 1) * 8;
        tmem_store8(at, high);
        if (kParts == 2 && (g & 1))
          tmem_store8(at + 16, low);
      }
      tmem_stored();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      bar_arrive(&sm.p_full[st]);
      if (lane == 0) // the warp is done with its part's scales
        bar_arrive(&sm.index_empty[part0]);
    };
    // Two loops, so that the ordinary one has nothing of far scales (in one, behind
    // a test a tile, a prompt of 8,192 took 14 us more). The other takes 732 us for
    // that prompt with a block of zeros among 64, 993 with every second one.
    if (apart) {
#pragma unroll 1
      for (int n = 0; n < mine; ++n)
        take(std::true_type{}, n);
    } else {
#pragma unroll 1
      for (int n = 0; n < mine; ++n)
        take(std::false_type{}, n);
    }
    if (mine > 0)
      ok = bar_wait(&sm.o_full[st], (mine - 1) & 1, failed) && ok;
    ok = __all_sync(0xffffffffu, ok);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // Each thread finishes its half of the row's elements with the whole row's sum.
    float share = 1.0f, other = 0.0f;
    float *joined = reinterpret_cast<float *>(sm.kv); // [element][row]
    sm.sums[st][half][row] = l;
    asm volatile("bar.sync %0, 64;" ::"r"(2 + st * 4 + (warp & 3)) : "memory");
    l = sm.sums[st][0][row] + sm.sums[st][1][row];
    if constexpr (kShare) {
      // Every product has completed (both streams have waited for theirs).
      asm volatile("bar.sync 1, 512;" ::: "memory");
      if (st == 1) {
        if (half == 0) {
          sm.join[0][row] = mine > 0 ? m : kNone;
          sm.join[1][row] = l;
        }
        if (mine > 0) {
#pragma unroll 1
          for (int c = half * kCh; c < (half + 1) * kCh; ++c) {
            uint32_t x[32];
            tmem_load(o_at + 32 * c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float o = __uint_as_float(x[i]);
              if (carry && mine > kFlush && live)
                o = fmaf(carry[(32 * c + i) * plane], carried, o);
              joined[(32 * c + i) * kM + row] = o;
            }
          }
        }
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");
      if (st == 0) {
        const float m1 = sm.join[0][row];
        const float most = fmaxf(m, m1);
        share = m == kNone ? 0.0f : exp2_approx(m - most);
        other = m1 == kNone ? 0.0f : exp2_approx(m1 - most);
        l = weigh(l, m, most) + weigh(sm.join[1][row], m1, most); // NaN stays
        m = most;
      }
    }
    const bool some = m != kNone || l != l; // l of a row that sees with NaN is NaN
    if (!kShare || st == 0) {
      const bool apart = a.splits > 1;
      const float scale = !some ? 0.0f : apart ? 1.0f : 1.0f / l;
      const int i = live ? f / a.group : 0;
      const int64_t at = (s.row0 + i) * a.q_heads + head * a.group + (live ? f - i * a.group : 0);
      const int64_t slot = static_cast<int64_t>(split) * v.rows * a.q_heads + at;
#pragma unroll 1
      for (int c = half * kCh; c < (half + 1) * kCh; ++c) {
        uint32_t x[32];
        tmem_load(o_at + 32 * c, x);
        float y[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          // Where a stream had no keys its accumulators hold nothing.
          float o = __uint_as_float(x[k]);
          if (kParts == 2 && carry && mine > kFlush && live)
            o = fmaf(carry[(32 * c + k) * plane], carried, o);
          o = share == 0.0f ? 0.0f : o * share;
          if constexpr (kShare)
            if (other != 0.0f)
              o = fmaf(joined[(32 * c + k) * kM + row], other, o);
          y[k] = some ? o * scale : 0.0f;
        }
        if (live && ok) {
          if (apart) {
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              Pack<float> p;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                p.at[e] = y[k + e];
              store_pack(a.part_o + slot * v.dim, 32 * c + k, v.dim, p);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += kVec<T>) {
              Pack<T> p;
#pragma unroll
              for (int e = 0; e < kVec<T>; ++e)
                p.at[e] = from_f32<T>(y[k + e]);
              store_pack(static_cast<T *>(a.out) + at * v.dim, 32 * c + k, v.dim, p);
            }
          }
        }
      }
      if (live && ok && half == 0) {
        if (apart)
          a.part_ml[slot] = make_float2(m, l);
        else if (a.lse)
          a.lse[at] = some ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
      }
    }
  } else if (warp < 20) {
    // ---------------------------------------------------------- converters
    // A thread loads 16 codes of a token a step; eight neighbouring lanes hold two tokens of one panel, so that
    // their 16-byte stores fall in different banks.
    constexpr int kSteps = 2 * kCh;         // steps a part of 64 tokens
    constexpr int kTokens = kSub / kSteps;  // tokens a step
    const int t = threadIdx.x - 512, quarter = t >> 3, r = t & 7;
    const int token = kCh == 2 ? (quarter >> 1) * 2 + (r >> 2) : quarter * 2 + (r >> 2);
    const int part = kCh == 2 ? (quarter & 1) * 4 + (r & 3) : (r & 3);
    const bool inside = part * 16 < v.dim;
    const int lane_at = (token & 15) * v.dim + part * 16, side_at = v.dim << v.block_log2;
    // 16-byte pieces of a part's keys or values, all in flight at once.
    auto load = [&](int j, int side, uint4 (&to)[kSteps]) {
      const float4 *index = sm.scale[j % kIndex];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int place = __float_as_int(index[(i * kTokens + token) >> 4].w);
        to[i] = make_uint4(0, 0, 0, 0);
        if (place >= 0 && inside)
          to[i] = __ldg(reinterpret_cast<const uint4 *>(
              v.codes + static_cast<int64_t>(place) * (16 * v.dim) + side * side_at + lane_at));
      }
    };
    auto store = [&](int side, int j, const uint4 (&from)[kSteps]) {
      uint8_t *base = sm.kv[side][(j >> 1) & 1] + (part / 4) * kPanel + (j & 1) * (kSub * 128);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int at = i * kTokens + token;
        uint4 x, y;
        codes_to_half(from[i].x, x.x, x.y);
        codes_to_half(from[i].y, x.z, x.w);
        codes_to_half(from[i].z, y.x, y.y);
        codes_to_half(from[i].w, y.z, y.w);
        uint8_t *row = base + at * 128;
        const int chunk = (part & 3) * 2;
        *reinterpret_cast<uint4 *>(row + ((chunk ^ (at & 7)) << 4)) = x;
        *reinterpret_cast<uint4 *>(row + (((chunk + 1) ^ (at & 7)) << 4)) = y;
      }
    };
    uint4 hold[2][kSteps];
    // True for all of the warp or none.
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      return __all_sync(0xffffffffu, bar_wait(bar, parity, failed));
    };
    convert_parts(
        2 * count,
        [&](int j) { return wait(&sm.index_full[j % kIndex], (j / kIndex) & 1); },
        [&](int side, int j) { return wait(&sm.kv_empty[side][(j >> 1) & 1], ((j >> 2) - 1) & 1); },
        [&](int j, int side) { load(j, side, hold[side]); },
        [&](int side, int j) {
          store(side, j, hold[side]);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          bar_arrive(&sm.kv_full[side][j & 3]);
        },
        [&](int j) { // this warp has read part j's places
          __syncwarp();
          if (lane == 0)
            bar_arrive(&sm.index_empty[j % kIndex]);
        });
  } else {
    if (warp == 20) {
      // ----------------------------------------------------------- products
      constexpr uint32_t kS = idesc_f16(kM, kTile, false), kO = idesc_f16(kM, kD, true);
      constexpr uint32_t kSlot = kCh * kPanel / 16;
      const uint32_t q_desc = desc_k_major(smem_at(sm.q)), k_desc = desc_k_major(smem_at(sm.kv[0])),
                     v_desc = desc_mn_major(smem_at(sm.kv[1]));
      bool ok = true;
      auto wait = [&](uint64_t *bar, uint32_t parity) {
        ok = __all_sync(0xffffffffu, ok && bar_wait(bar, parity, failed));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        return ok;
      };
      // Round n of a stream takes its n-th tile. Rounds go by twos, so that
      // slots are constants; the warp stays together and elects a thread for
      // each run of products, so that their operands are uniform (one thread
      // by itself took twice as long to issue a product as the product does).
      const int rounds = kShare ? (count + 1) / 2 : count;
      auto ready = [&](int side, int tile, int slot) { // both parts of a tile
        return wait(&sm.kv_full[side][2 * slot], (tile >> 1) & 1) &&
               wait(&sm.kv_full[side][2 * slot + 1], (tile >> 1) & 1);
      };
      auto scores = [&](int st, int n, int u) { // u = n mod 2
        const int tile = kShare ? 2 * n + st : n, slot = kShare ? st : u;
        if (tile >= count || !ready(0, tile, slot))
          return;
        if (elect()) {
#pragma unroll
          for (int part = 0; part < kParts; ++part) // the small part first
#pragma unroll
            for (int i = 0; i < 4 * kCh; ++i)
              mma_ss(tmem + st * kTile,
                     q_desc + ((kShare ? 0 : st) * kSlot + (kParts - 1 - part) * kSlot +
                               ((i / 4) * kPanel + (i % 4) * 32) / 16),
                     k_desc + (slot * kSlot + ((i / 4) * kPanel + (i % 4) * 32) / 16), kS,
                     part + i > 0);
          commit(&sm.s_full[st]);
          if (kShare || st == 1)
            commit(&sm.kv_empty[0][slot]);
        }
        __syncwarp();
      };
      auto outputs = [&](int st, int n, int u) {
        const int tile = kShare ? 2 * n + st : n, slot = kShare ? st : u;
        if (tile >= count || !ready(1, tile, slot) || !wait(&sm.p_full[st], n & 1))
          return;
        const bool fresh = n == 0 || (kParts == 2 && a.carry && n % kFlush == 0);
        if (elect()) {
#pragma unroll
          for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
              mma_ts(tmem + 2 * kTile + st * kD,
                     tmem + st * kTile + ((i / 2) * 32 + (i % 2) * 8 + (kParts - 1 - part) * 16),
                     v_desc + (slot * kSlot + i * (2048 / 16)), kO, !fresh || part + i > 0);
          commit(&sm.o_full[st]);
          if (kShare || st == 1)
            commit(&sm.kv_empty[1][slot]);
        }
        __syncwarp();
      };
      scores(0, 0, 0);
      if (ok)
        scores(1, 0, 0);
#pragma unroll 1
      for (int n0 = 0; n0 < rounds && ok; n0 += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            if (ok)
              outputs(st, n0 + u, u);
            if (ok)
              scores(st, n0 + u + 1, u ^ 1);
          }
      }
      // Nothing of this CTA may be in flight when its TMEM is freed.
      if (elect())
        commit(&sm.done);
      __syncwarp();
      int unused = 0;
      bar_wait(&sm.done, 0, &unused);
    } else if (warp == 21) {
      // --------------------------------------------------------- pages, scales
      // Lane i takes a part's i-th group of 16 tokens; table entries are loaded
      // two parts ahead and scales one, so that neither is waited for here.
      const int per_page = v.block_log2 - 4;
      const int parts = 2 * count;
      auto key_of = [&](int j) { return key_base + j * kSub + (lane & 3) * 16; };
      auto entry_of = [&](int j) { // the table's entry, unchecked; -1: no token
        const int key = key_of(j);
        return j < parts && key < s.length ? v.table[b * v.table_stride + (key >> v.block_log2)] : -1;
      };
      auto scales_of = [&](int j, int entry, int &place) {
        const int key = key_of(j);
        const bool good = entry >= 0 && entry < v.pages;
        if (!good && lane < 4 && j < parts && key < s.length)
          atomicOr(a.status, CIM22_STATUS_CACHE_INDEX);
        place = good ? (((entry * v.heads + head) * 2) << per_page) +
                           ((key >> 4) & ((1 << per_page) - 1))
                     : -1;
        return good ? *reinterpret_cast<const float2 *>(
                          v.scales + (static_cast<int64_t>(entry) * v.heads + head) * 2)
                    : make_float2(0.0f, 0.0f);
      };
      int place, entry = entry_of(0), next_entry = entry_of(1);
      float2 two = scales_of(0, entry, place);
      for (int j = 0; j < parts; ++j) {
        const int after = entry_of(j + 2);
        int next_place;
        const float2 next = scales_of(j + 1, next_entry, next_place);
        const bool ok = j < kIndex ||
                        bar_wait(&sm.index_empty[j % kIndex], ((j / kIndex) - 1) & 1, failed);
        if (!__all_sync(0xffffffffu, ok))
          break;
        if (lane < 4) {
          const float sv = fmaxf(two.y, kKvLeastScale);
          sm.scale[j % kIndex][lane] = place < 0
                                      ? make_float4(0.0f, -INFINITY, 0.0f, __int_as_float(-1)) // hidden
                                      : make_float4(two.x, log2f(sv), 1.0f / sv, __int_as_float(place));
        }
        __syncwarp();
        if (lane == 0)
          bar_arrive(&sm.index_full[j % kIndex]);
        two = next;
        place = next_place;
        next_entry = after;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && *reinterpret_cast<volatile int *>(failed))
    atomicOr(a.status, CIM22_STATUS_TIMEOUT);
  if (warp == 20) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <typename T, int kCh, int kParts, bool kShare>
cudaError_t launch_prompt(const KvAttendArgs &a, int tiles, cudaStream_t stream) {
  constexpr size_t bytes = sizeof(PromptSmem<kCh>) + 1024;
  const auto kernel = kv_prompt_kernel<T, kCh, kParts, kShare>;
  static DynamicSmem allowed;
  if (const cudaError_t e = allowed.allow(kernel, bytes); e != cudaSuccess)
    return e;
  return launch_pdl(kernel, dim3(static_cast<unsigned>(tiles) * a.v.heads, a.splits, a.v.batch),
                    dim3(kThreads), bytes, stream, a, tiles);
}

} // namespace

cudaError_t kv_prompt_launch(const KvAttendArgs &a, int type, bool share, int tiles,
                             cudaStream_t stream) {
  const bool wide = a.v.dim > 64;
  if (type == CIM22_FLOAT32)
    return wide ? launch_prompt<float, 2, 2, true>(a, tiles, stream)
                : launch_prompt<float, 1, 2, true>(a, tiles, stream);
  if (type == CIM22_BFLOAT16) {
    if (share)
      return wide ? launch_prompt<__nv_bfloat16, 2, 1, true>(a, tiles, stream)
                  : launch_prompt<__nv_bfloat16, 1, 1, true>(a, tiles, stream);
    return wide ? launch_prompt<__nv_bfloat16, 2, 1, false>(a, tiles, stream)
                : launch_prompt<__nv_bfloat16, 1, 1, false>(a, tiles, stream);
  }
  if (share)
    return wide ? launch_prompt<__half, 2, 1, true>(a, tiles, stream)
                : launch_prompt<__half, 1, 1, true>(a, tiles, stream);
  return wide ? launch_prompt<__half, 2, 1, false>(a, tiles, stream)
              : launch_prompt<__half, 1, 1, false>(a, tiles, stream);
}

} // namespace cim
