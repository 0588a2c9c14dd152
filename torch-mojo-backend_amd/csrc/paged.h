// The paged key/value cache as its kernels see it (paged_cache.hip fills and
// reads it, paged_attention.hip attends over it).
//
// A page holds page_size tokens of every K/V head.  Token p of sequence b lies
// in page table[b][p / page_size], slot p % page_size; its row of d channels is
// d values of the cache's type, or, in a 4-bit cache, d / 2 bytes of codes and
// d / 32 (scale, minimum) pairs in f16, value = minimum + scale * code.
//
// Codes: the 32-bit word g * (d / 32) + s of a row (g < 4) holds channels
// 32 s + 8 g + e, e < 8, channel e in nibble e / 2 + 4 (e % 2).  The lanes of a
// matrix operand that share a key hold channels 8 g .. 8 g + 7 of every 32, so
// lane g finds all of its codes side by side; and a word shifted by 4 i and
// masked with 0x000f000f gives channels 2 i and 2 i + 1 as two 16-bit halves.
#pragma once
#include "common.h"
#include "paged_span.h"

namespace mi {

constexpr int kKvGroup = 32;  // channels per (scale, minimum) pair
// Values are clamped to this before they are packed: minimum + 15 * scale,
// both rounded to f16, then stays finite in f16 (61440 + 122880 * 2^-11 < 65504),
// as do twice the scale and 7.5 times it, which attention forms in f16.
constexpr double kKvLimit = 61440.0;

// Quotients of 31-bit positions by the page size: one multiply-high and a
// shift instead of the division's twenty instructions.  For a divisor that is
// no power of two, magic = floor(2^(32 + s) / divisor) + 1 with s = floor(log2
// divisor); it exceeds 2^(32 + s) / divisor by e / divisor with e <= divisor
// < 2^(s + 1), which is exact for every n < 2^31.
struct PageDiv {
  uint32_t size, magic, shift;  // magic 0: size is a power of two, n >> shift
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return magic ? __umulhi(n, magic) >> shift : n >> shift;
  }
};
inline PageDiv page_div(int64_t size) {
  PageDiv p{(uint32_t)size, 0, 0};
  while ((2ull << p.shift) <= (uint64_t)size) ++p.shift;
  if ((uint64_t)size != 1ull << p.shift) p.magic = (uint32_t)(((1ull << 32) << p.shift) / (uint64_t)size + 1);
  return p;
}

// Which token a place of the batch holds.
struct PagedSeqs {
  const int32_t* table;  // [batch][width] page numbers
  int64_t table_stride;
  uint32_t width;        // pages per sequence
  const int32_t* starts; // position of token 0 of each sequence
  const int32_t* counts; // tokens of each sequence, the rest is padding (null: all)
  PageDiv page;
  int32_t num_pages;
  int32_t end;           // positions from here on are past the table
  int32_t* error;        // set to 1 by a page or position out of range (may be null)
};

__device__ __forceinline__ int seq_count(const PagedSeqs& s, int64_t b, int seq) {
  return s.counts ? min(max(s.counts[b], 0), seq) : seq;
}

// The page of position pos, or -1 (and the error flag) where the table has
// none or names one that does not exist.
__device__ __forceinline__ int page_of(const PagedSeqs& s, int64_t b, uint32_t pos, uint32_t* slot) {
  const uint32_t i = s.page.div(pos);
  *slot = pos - i * s.page.size;
  int page = i < s.width ? s.table[b * s.table_stride + i] : -1;
  if ((uint32_t)page >= (uint32_t)s.num_pages) {
    if (s.error) *s.error = 1;
    page = -1;
  }
  return page;
}

// Rows [batch, heads, tokens, d] that can be read 16 bytes at a time.
inline bool rows_ok(const void* p, const int64_t* bht, size_t es) {
  return (uintptr_t)p % 16 == 0 && bht[0] * (int64_t)es % 16 == 0 && bht[1] * (int64_t)es % 16 == 0 &&
         bht[2] * (int64_t)es % 16 == 0;
}

// Checks of the arguments that every entry point shares; fills `s`.
int paged_args(const char* what, const mi355x_paged_cache* c, const int32_t* table, int64_t table_stride,
               int64_t table_width, const int32_t* starts, const int32_t* counts, int64_t batch, int64_t seq,
               int32_t* error, PagedSeqs* s);

}  // namespace mi
