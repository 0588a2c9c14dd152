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

// Whether the matrix-core kernel takes these pages with queries of dtype.
bool paged_mfma_takes(const mi355x_paged_cache& c, int dtype);
int paged_mfma_row_tiles(int64_t rows, int64_t d);
int paged_mfma_launch(DecodeArgs a, int dtype, hipStream_t s);

}  // namespace mi
