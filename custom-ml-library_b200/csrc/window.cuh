// The sliding window with sinks: query position i sees the keys j <= i with i - j < window or j < sinks.
#pragma once
#include "common.cuh"

namespace tsa {

struct WindowArgs {
  int window = 0;  // 0: no window
  int sinks = 0;
};

// Bits k of [0, 32) with lo <= base + k < hi.
__device__ __forceinline__ uint32_t range_bits(int64_t lo, int64_t hi, int64_t base) {
  const int a = (int)i64max(0, i64min(32, lo - base)), b = (int)i64max(0, i64min(32, hi - base));
  const uint32_t below_b = b >= 32 ? 0xffffffffu : (1u << b) - 1u;
  const uint32_t below_a = a >= 32 ? 0xffffffffu : (1u << a) - 1u;
  return below_b & ~below_a;
}

// Key tiles that a block of queries reads: those with sinks, then those from the window of its first query on.
// Tile j of the list is key tile j below `sink_tiles`, j + skip behind.
struct WindowTiles {
  int sink_tiles, skip;
  WindowTiles() = default;
  // Queries from position `first` (may be negative), keys [0, kv_end) in tiles of `tile` keys.
  __device__ __forceinline__ WindowTiles(const WindowArgs& w, int64_t first, int kv_end, int tile) {
    sink_tiles = ceil_div(min(max(w.sinks, 0), kv_end), tile);
    const int64_t low = i64max(0, i64min(kv_end, first - w.window + 1));
    skip = w.window > 0 ? max(0, (int)(low / tile) - sink_tiles) : 0;
  }
  // Length of the list when the queries see key tiles [0, tiles).
  __device__ __forceinline__ int count(int tiles) const {
    return tiles <= sink_tiles ? tiles : max(sink_tiles, tiles - skip);
  }
  __device__ __forceinline__ int tile(int j) const { return j < sink_tiles ? j : j + skip; }
};

}  // namespace tsa
