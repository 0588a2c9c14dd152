// The plan of a packed batch (packed.h), and its rows' positions.
#include "packed.h"

namespace mi {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kClasses = 512;  // tile numbers that are told apart; all later ones start first, in any order

// One block: a batch has one plan, which serves every layer.  A tile number's
// entries stand together behind those of all later numbers; their order among
// themselves is that of arrival, and moves no result.  With sequence i's number
// of tiles m_i, number k has as many entries as there are m_i > k: a count of
// the m_i, then two suffix sums.
// 16384 rows: one sequence 5 us, 16 of 1024 rows 11, 48 of 341 14, 16384 of one row 45.
__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(PackedHeader* head, PackedTile* list0, PackedTile* list1,
                                                                   const int32_t* offsets, int64_t n, int tokens,
                                                                   int32_t* error) {
  __shared__ int at[2][kClasses];   // entries of a class, then its next place
  __shared__ int sum[2][kClasses];
  __shared__ int bad, beyond[2];    // beyond: tiles past those of the classes
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int w = tid / kClasses, k = tid % kClasses;  // a list and a class of it
  static_assert(kPlanThreads == 2 * kClasses, "");
  at[w][k] = 0;
  if (tid == 0) bad = beyond[0] = beyond[1] = 0;
  __syncthreads();
  for (int64_t i = tid; i <= n; i += kPlanThreads) {
    const int a = offsets[i], b = i < n ? offsets[i + 1] : tokens;
    if (a < 0 || a > b || b > tokens) bad = 1;
  }
  __syncthreads();
  const int64_t seqs = bad ? 0 : n;
  // at[k] = how many sequences have k + 1 tiles (the last class: or more)
  for (int64_t i = tid; i < seqs; i += kPlanThreads) {
    const int len = offsets[i + 1] - offsets[i];
    if (len == 0) continue;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int m = (len - 1) / kPackedRows[v] + 1;
      atomicAdd(&at[v][min(m, kClasses) - 1], 1);
      if (m > kClasses) atomicAdd(&beyond[v], m - kClasses);
    }
  }
  __syncthreads();
  auto suffix = [&](int x) {  // of this thread's class and all later ones
    for (int step = 1; step < kClasses; step *= 2) {
      sum[w][k] = x;
      __syncthreads();
      if (k + step < kClasses) x += sum[w][k + step];
      __syncthreads();
    }
    return x;
  };
  int entries = suffix(at[w][k]);
  if (k == kClasses - 1) entries += beyond[w];
  const int upto = suffix(entries);
  at[w][k] = upto - entries;
  __shared__ int total[2];
  if (k == 0) total[w] = upto;
  __syncthreads();

  PackedTile* const list[2] = {list0, list1};
  for (int64_t i0 = (int64_t)wave * 64; i0 < seqs; i0 += kPlanThreads) {
    const int64_t i = i0 + lane;
    const int a = i < seqs ? offsets[i] : 0, len = i < seqs ? offsets[i + 1] - a : 0;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int m = len ? (len - 1) / kPackedRows[v] + 1 : 0;
      auto put = [&](int start, int length, int tile) {
        list[v][atomicAdd(&at[v][min(tile, kClasses - 1)], 1)] = PackedTile{start, length, tile, 0};
      };
      if (m <= 4)
        for (int t = 0; t < m; ++t) put(a, len, t);
      uint64_t more = __ballot(m > 4);  // these the wave's lanes share
      while (more) {
        const int src = __ffsll((unsigned long long)more) - 1;
        more &= more - 1;
        const int sa = __shfl(a, src, 64), sl = __shfl(len, src, 64), sm = __shfl(m, src, 64);
        for (int t = lane; t < sm; t += 64) put(sa, sl, t);
      }
    }
  }
  const int begin = bad ? 0 : n > 0 ? offsets[0] : 0, end = bad ? 0 : n > 0 ? offsets[n] : 0;
  const int rows = kPackedRows[w], before = (begin + rows - 1) / rows, behind = (tokens - end + rows - 1) / rows;
  for (int i = k; i < before + behind; i += kClasses) {
    const int start = i < before ? i * rows : end + (i - before) * rows;
    list[w][total[w] + i] = PackedTile{start, min(rows, (i < before ? begin : tokens) - start), -1, 0};
  }
  if (k == 0) head->count[w] = total[w] + before + behind;
  if (tid == 0) {
    head->begin = begin, head->end = end;
    if (bad && error) *error = 1;
  }
}

// A wave takes 64 rows: positions within their sequence, 0 of rows without one.
__global__ void __launch_bounds__(256) packed_positions_kernel(int32_t* positions, const PackedHeader* head, const PackedTile* list) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= head->count[1]) return;
  const PackedTile t = list[i];
  const int p = max(t.tile, 0) * 64 + lane;
  if (p < t.len) positions[t.start + p] = t.tile < 0 ? 0 : p;
}

}  // namespace
}  // namespace mi

using namespace mi;

static int packed_check(const char* what, int64_t sequences, int64_t tokens) {
  MI_REQUIRE(sequences >= 0 && tokens >= 0, "%s: %lld sequences of %lld rows", what, (long long)sequences, (long long)tokens);
  MI_REQUIRE(sequences < (1ll << 30) && tokens < (1ll << 30) - 1024, "%s: too many sequences or rows", what);
  return MI355X_OK;
}

extern "C" int64_t mi355x_packed_plan_bytes(int64_t sequences, int64_t tokens) {
  return packed_check("mi355x_packed_plan_bytes", sequences, tokens) ? -1 : packed_bytes(sequences, tokens);
}

extern "C" int mi355x_packed_plan(void* plan, int64_t plan_bytes, int32_t* positions, const int32_t* offsets,
                                  int64_t sequences, int64_t tokens, int32_t* error, mi355x_stream_t stream) {
  const int rc = packed_check("mi355x_packed_plan", sequences, tokens);
  if (rc) return rc;
  MI_REQUIRE(plan && offsets && (positions || tokens == 0), "mi355x_packed_plan: null pointer");
  MI_REQUIRE((uintptr_t)plan % 16 == 0, "mi355x_packed_plan: the plan must be 16-byte aligned");
  if (plan_bytes < packed_bytes(sequences, tokens))
    return fail(MI355X_EWORKSPACE, "mi355x_packed_plan: %lld bytes given, %lld needed", (long long)plan_bytes,
                (long long)packed_bytes(sequences, tokens));
  hipStream_t s = (hipStream_t)stream;
  PackedHeader* head = (PackedHeader*)plan;
  PackedTile* l0 = (PackedTile*)packed_list(plan, sequences, tokens, 128);
  PackedTile* l1 = (PackedTile*)packed_list(plan, sequences, tokens, 64);
  packed_plan_kernel<<<1, kPlanThreads, 0, s>>>(head, l0, l1, offsets, sequences, (int)tokens, error);
  const unsigned blocks = ceil_div(packed_cap(sequences, tokens, 64), 4);
  if (tokens) packed_positions_kernel<<<blocks, 256, 0, s>>>(positions, head, l1);
  return check_launch("mi355x_packed_plan");
}
