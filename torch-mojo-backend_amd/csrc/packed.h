// Sequences of different lengths laid end to end, as the kernels see them: a
// plan in device memory that packed_plan.hip makes of a batch's offsets.
//
// The plan is a header, then two lists of tiles, of 128 rows and of 64.  A tile
// belongs to one sequence, so no kernel reads a row of another one and a NaN in
// one sequence stays there.  Lists are sorted by the tile's number within its
// sequence, last first: a causal query tile's work grows with it, as that of the
// key tile that lies as far from the end does, so either walk takes its longest
// tiles first.  Behind them the list names the rows that belong to no sequence,
// whose results are zero.
#pragma once
#include "common.h"

namespace mi {

struct PackedTile {
  int32_t start, len, tile, unused;  // a sequence's first row and length, the tile's number in it
  // (tile -1: rows start .. start + len - 1 belong to no sequence)
};
struct PackedHeader {
  int32_t count[2];    // entries of the two lists
  int32_t begin, end;  // rows of all sequences
  int32_t unused[12];
};
static_assert(sizeof(PackedTile) == 16 && sizeof(PackedHeader) == 64, "");

constexpr int kPackedRows[2] = {128, 64};

// Entries that a list can have: every sequence's tiles but its last are full,
// and rows before the first and behind the last sequence make one short tile each.
inline int64_t packed_cap(int64_t sequences, int64_t tokens, int rows) { return tokens / rows + sequences + 2; }
inline int64_t packed_bytes(int64_t sequences, int64_t tokens) {
  return (int64_t)sizeof(PackedHeader) +
         (packed_cap(sequences, tokens, 128) + packed_cap(sequences, tokens, 64)) * (int64_t)sizeof(PackedTile);
}
inline const PackedTile* packed_list(const void* plan, int64_t sequences, int64_t tokens, int rows) {
  const PackedTile* first = (const PackedTile*)((const char*)plan + sizeof(PackedHeader));
  return rows == 128 ? first : first + packed_cap(sequences, tokens, 128);
}

// The block's tile and heads of a 1-D grid of (list entries) x heads.  The tile
// varies slowest, so the longest tiles of all heads start first; blocks go to
// the 8 XCDs in turn, and neighbouring blocks take different K/V heads, so with
// 8 K/V heads or a divisor of 8 all that read one of them share an L2.
struct PackedAt {
  PackedTile t;
  int h, hk;
  bool live;
};
__device__ __forceinline__ PackedAt packed_at(const PackedTile* list, int count, uint32_t l, uint32_t heads, uint32_t kv_heads) {
  const uint32_t i = l / heads, s = l - i * heads, hk = s % kv_heads, g = s / kv_heads;
  PackedAt a{};
  a.live = i < (uint32_t)count;
  if (a.live) {  // (one entry for the block: in scalar registers, as what is made of it)
    const PackedTile t = list[i];
    a.t.start = __builtin_amdgcn_readfirstlane(t.start), a.t.len = __builtin_amdgcn_readfirstlane(t.len);
    a.t.tile = __builtin_amdgcn_readfirstlane(t.tile);
  }
  a.hk = (int)hk, a.h = (int)(hk * (heads / kv_heads) + g);
  return a;
}

}  // namespace mi
