// Sliding window with sinks, for the kernels that walk key or query tiles: query i sees key j iff
// j <= i and (j > i - window or j < sinks). Which tiles a workgroup walks, which 32 x 32 chunks a
// wave computes, and which of those it must mask.
#pragma once

#include "kernels.hpp"

namespace dadgpt {

// The key tiles (of TR rows) that queries first .. last see, in order: with a window, the sinks'
// tiles and then those from the first query's first visible key on.
template <bool WIN, int TR = 64>
struct KeyTiles {
  int last_tile, sink_tiles, first_tile;
  __device__ __forceinline__ KeyTiles(int first, int last, const WindowArg<WIN>& w)
      : last_tile(last / TR), sink_tiles(0), first_tile(0) {
    if constexpr (WIN) {
      first_tile = max(0, first - w.window + 1) / TR;
      sink_tiles = min((w.sinks + TR - 1) / TR, first_tile);
    }
  }
  __device__ __forceinline__ int count() const {
    return WIN ? sink_tiles + last_tile - first_tile + 1 : last_tile + 1;
  }
  // first row of tile t
  __device__ __forceinline__ int row(int t) const {
    return TR * (!WIN || t < sink_tiles ? t : t - sink_tiles + first_tile);
  }
};

// Keys c0 .. c0+31 against queries q0 .. q0+31, c0 <= q0 + 31: whether any pair is visible (the
// first query's window reaches furthest back), and whether all are.
__device__ __forceinline__ bool chunk_visible(int c0, int q0, const Window& w) {
  return c0 + 31 > q0 - w.window || c0 < w.sinks;
}
__device__ __forceinline__ bool chunk_whole(int c0, int q0, const Window& w) {
  return c0 + 31 <= q0 && (c0 > q0 + 31 - w.window || c0 + 31 < w.sinks);
}

// Whether key `base` + k is hidden from `query`, for small constants k.
struct HiddenKeys {
  int after, before, sinks;  // k > after, or k <= before and k >= sinks
  HiddenKeys() = default;
  __device__ __forceinline__ HiddenKeys(int base, int query, const Window& w)
      : after(query - base), before(query - base - w.window), sinks(w.sinks - base) {}
  __device__ __forceinline__ bool operator()(int k) const {
    return k > after || (k <= before && k >= sinks);
  }
};

}  // namespace dadgpt
