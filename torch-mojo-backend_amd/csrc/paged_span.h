// Positions of a paged cache, and the keys that attention over it walks: plain
// arithmetic, the same on the host.
#pragma once
#include <stdint.h>

namespace mi {

// Positions end a little below 2^31, so that 32-bit sums with a tile's length
// do not pass it.
constexpr int64_t kMaxPosition = 0x7fffff00;

// The first position that a table of `width` pages (both below 2^31) has no place for.
inline int32_t table_end(int64_t width, int64_t page_size) {
  const int64_t n = width * page_size;
  return (int32_t)(n < kMaxPosition + 1 ? n : kMaxPosition + 1);
}

// The keys below `end` that queries at positions first .. last (at most
// kMaxPosition) can see, in tiles of `tile` keys: the sinks' tiles, then the
// window's from tile `low` on.  However far the queries are, there are no more
// tiles than `end` keys have.
struct KeySpan {
  int sink_tiles, low, tiles;
  __device__ __forceinline__ KeySpan(int first, int last, int window, int sinks, int end, int tile) {
    last = min(last, end - 1);
    low = window > 0 ? max(first - window + 1, 0) / tile : 0;
    const int s = window > 0 ? min(sinks, last + 1) : 0;
    sink_tiles = min((s + tile - 1) / tile, low);
    tiles = last < 0 ? 0 : sink_tiles + max(last / tile + 1 - low, 0);
  }
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : low + i - sink_tiles; }
};
__device__ __forceinline__ bool visible(int pos, int j, int window, int sinks) {
  return j <= pos && (window <= 0 || pos - j < window || j < sinks);
}

}  // namespace mi
