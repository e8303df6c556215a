// kv_convert.h - the order in which a converter warp of the prompt attention
// kernel (kv_attention_tc.cu) waits, loads and stores. Apart from the kernel,
// so that it can be run on the host with waits that run out.
#pragma once

#if defined(__CUDACC__)
#define CIM22_HD __host__ __device__ __forceinline__
#else
#define CIM22_HD inline
#endif

namespace cim {

// Parts of 64 tokens, keys (side 0) and values (side 1) of each, two parts to
// a tile and two tiles' slots. Part j + 1 is loaded while part j is stored.
// indexed(j): waits until the places of part j are known; emptied(side, j):
// until part j's slot has been read by the product of the tile before last.
// Both are false, for the whole warp, when the wait has run out: nothing may be
// done then that relies on it, and a load least of all, since a place that
// was never written is an address anywhere.
template <typename Indexed, typename Emptied, typename Load, typename Store, typename Used>
CIM22_HD void convert_parts(int parts, Indexed indexed, Emptied emptied, Load load, Store store,
                            Used used) {
  if (parts <= 0 || !indexed(0))
    return;
  load(0, 0);
  load(0, 1);
  used(0);
  for (int j = 0; j < parts; ++j) {
    const bool more = j + 1 < parts;
    if (j >= 4 && !emptied(0, j))
      return;
    store(0, j);
    if (more) {
      if (!indexed(j + 1))
        return;
      load(j + 1, 0);
    }
    if (j >= 4 && !emptied(1, j))
      return;
    store(1, j);
    if (more) {
      load(j + 1, 1);
      used(j + 1);
    }
  }
}

} // namespace cim
