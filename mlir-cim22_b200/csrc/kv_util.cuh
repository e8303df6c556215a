// kv_util.cuh - the 8-bit key/value cache as its kernels see it, and the
// checks of its descriptions.
#pragma once

#include "decoder_util.cuh"

#include <string>

namespace cim {

// The least scale a block is written with is kKvFloor * f32(1 / 127).
constexpr float kKvFloor = 0x1p-80f;
constexpr float kKvInv127 = 1.0f / 127.0f;
// Longest sequence: positions and a tile past it stay in 32 bits.
constexpr int kKvLongest = 0x7fff0000;

struct KvView {
  int8_t *codes;
  float *scales;
  int64_t pages;
  int heads, block_log2, dim;
  const int32_t *table;
  int64_t table_stride;
  int table_width;
  const int32_t *lengths, *starts;
  int64_t rows;
  int most, batch;
};

// Checks that need no device; the message goes to the caller's last error.
inline bool kv_view(const char *what, const cim22_kv_cache *c, const cim22_kv_sequences *s,
                    KvView &v) {
  const auto refuse = [&](const char *why) {
    set_last_error(std::string(what) + ": " + why);
    return false;
  };
  if (!c || !s)
    return refuse("null cache or sequences");
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return refuse("block must be 16, 32, 64 or 128 tokens");
  if (c->head_dim < 16 || c->head_dim > 128 || c->head_dim % 16)
    return refuse("head_dim must be a multiple of 16 up to 128");
  if (c->kv_heads < 1 || c->kv_heads > 32767)
    return refuse("kv_heads out of range");
  if (c->pages < 0 || c->pages > 0x7fffffff || (c->pages > 0 && (!c->codes || !c->scales)))
    return refuse("null cache, or pages out of range");
  if ((reinterpret_cast<uintptr_t>(c->codes) & 15) || (reinterpret_cast<uintptr_t>(c->scales) & 7))
    return refuse("codes must be 16-byte and scales 8-byte aligned");
  if (s->batch < 0 || s->batch > 65535)
    return refuse("batch out of range");
  if (s->batch > 0 && (!s->lengths || (s->table_width > 0 && !s->table)))
    return refuse("null lengths or table");
  if (s->table_width < 0 || (s->batch > 1 && s->table_stride < s->table_width))
    return refuse("table rows overlap");
  if (s->rows < 0 || s->most < 0 || (s->batch > 0 && !s->starts && s->rows < s->batch))
    return refuse("rows or most out of range");
  v = KvView{c->codes,  c->scales,       c->pages,      c->kv_heads, 0,
             c->head_dim, s->table,      s->table_stride, s->table_width, s->lengths,
             s->starts, s->rows,         s->starts ? s->most : 1, s->batch};
  while ((1 << v.block_log2) < c->block)
    ++v.block_log2;
  return true;
}

#if defined(__CUDACC__)
namespace {

// One sequence of a call: its rows [row0, row0 + n) sit at positions
// length - n .. length - 1. An inconsistent description leaves it empty.
struct KvSequence {
  int n, length;
  int64_t row0;
  bool ok;
};

__device__ __forceinline__ KvSequence kv_sequence(const KvView &v, int b) {
  KvSequence s;
  s.length = v.lengths[b];
  s.row0 = b;
  s.n = 1;
  if (v.starts) {
    s.row0 = v.starts[b];
    const int64_t n = static_cast<int64_t>(v.starts[b + 1]) - s.row0;
    s.n = n < 0 || n > v.most ? -1 : static_cast<int>(n);
  }
  s.ok = s.n >= 0 && s.row0 >= 0 && s.row0 + s.n <= v.rows && s.length >= 0 && s.length <= kKvLongest && (v.pages > 0 || s.length == 0) &&
         s.length <= (static_cast<int64_t>(v.table_width) << v.block_log2);
  if (!s.ok)
    s.n = s.length = 0;
  return s;
}

// The page of a sequence's block `ordinal` (within the table's width), or -1.
__device__ __forceinline__ int kv_page(const KvView &v, int b, int ordinal) {
  const int page = v.table[b * v.table_stride + ordinal];
  return page >= 0 && page < v.pages ? page : -1;
}

// Codes of (page, head, side).
__device__ __forceinline__ int8_t *kv_codes(const KvView &v, int64_t page, int head, int side) {
  return v.codes + ((((page * v.heads + head) * 2 + side) << v.block_log2) * v.dim);
}

} // namespace
#endif

} // namespace cim
