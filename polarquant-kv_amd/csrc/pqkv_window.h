// Attention behind a window: the rows of a sequence, and the tiles that they
// see (device side; the arguments are Window in pqkv_launch.h).
#pragma once

#include "pqkv_launch.h"

namespace pqkv {

// The rows of one sequence that stand in a cache of `cap` positions, of a call
// with at most `most` rows: none where the first one does not.
struct WindowRows {
  int start, count;
};
__device__ __forceinline__ WindowRows window_rows(const Window &w, int b, int most, int cap) {
  const int64_t s = w.starts ? w.starts[b] : w.start;
  int64_t n = w.counts ? w.counts[b] : w.count;
  n = n < most ? n : most;
  if (s < 0 || s >= cap || n <= 0) return {0, 0};
  return {(int)s, (int)(n < cap - s ? n : cap - s)};
}
// The 64-token tiles that rows first .. last of a sequence see: `sink` tiles from
// position 0 on, then those from `lo` (a multiple of 64) to the last row's; all
// of them hold a position that one of the rows sees.
struct WindowTiles {
  int sink, lo, tiles;
  __device__ __forceinline__ int at(int i) const { return i < sink ? 64 * i : lo + 64 * (i - sink); }
};
__device__ __forceinline__ WindowTiles window_tiles(const Window &w, int first, int last) {
  const int lo = first >= w.size ? (first - w.size + 1) & ~63 : 0;
  const int sink = min((w.sinks + 63) >> 6, lo >> 6);
  return {sink, lo, sink + ((last - lo) >> 6) + 1};
}

}  // namespace pqkv
