// Shared by the two kernels of attention over a paged cache: the one on matrix
// cores (paged_attention_mfma.hip) and the one for everything else
// (paged_attention.hip, which also has the entry points).
#pragma once
#include "paged.h"

namespace mi {

struct DecodeArgs {
  mi355x_paged_cache c;
  PagedSeqs s;
  void* o;
  int64_t o_b, o_h, o_t;
  const void* q;
  int64_t q_b, q_h, q_t;
  int64_t batch;
  int heads, group, seq;
  int window, sinks;  // window 0: none
  int splits;         // blocks that share the keys of a row
  float scale_log2;   // scale * log2(e)
  float* part_o;      // [splits][batch * heads * seq][d]
  float2* part_ml;    // [splits][batch * heads * seq]: maximum (base 2) and sum
  int64_t row_groups, units;  // matrix cores: blocks of query rows per K/V head; (batch, K/V head, split) triples
};

// The keys that queries at positions first .. last can see, in tiles of
// `tile` keys: the sinks' tiles, then the window's from tile `low` on.
struct KeySpan {
  int sink_tiles, low, tiles;
  __device__ __forceinline__ KeySpan(int first, int last, int window, int sinks, int tile) {
    low = window > 0 ? max(first - window + 1, 0) / tile : 0;
    const int s = window > 0 ? min(sinks, last + 1) : 0;
    sink_tiles = min((s + tile - 1) / tile, low);
    tiles = last < 0 ? 0 : sink_tiles + last / tile + 1 - low;
  }
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : low + i - sink_tiles; }
};
__device__ __forceinline__ bool visible(int pos, int j, int window, int sinks) {
  return j <= pos && (window <= 0 || pos - j < window || j < sinks);
}

// Whether the matrix-core kernel takes these pages with queries of dtype.
bool paged_mfma_takes(const mi355x_paged_cache& c, int dtype);
int paged_mfma_row_tiles(int64_t rows, int64_t d);
int paged_mfma_launch(DecodeArgs a, int dtype, hipStream_t s);

}  // namespace mi
