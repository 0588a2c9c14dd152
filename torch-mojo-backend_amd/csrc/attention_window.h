// What the attention kernels share: their arguments, and the partial sums of a
// windowed backward (attention.hip for 16-bit types, attention_f32.hip).
#pragma once
#include <algorithm>

#include "common.h"

namespace mi {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct alignas(16) V8 {
  T v[8];
};
template <typename T>
struct alignas(8) V4 {
  T v[4];
};

struct AttnArgs {
  void* o; int64_t o_b, o_h, o_s;
  float* lse;
  const void* q; int64_t q_b, q_h, q_s;
  const void* k; int64_t k_b, k_h, k_s;
  const void* v; int64_t v_b, v_h, v_s;
  int64_t B, H, Sq, Skv;
  float scale_log2;  // scale * log2(e)
  float scale;
  int causal;
  int64_t group;   // query heads per K/V head (grouped-query attention), >= 1
  int64_t window;  // > 0: query i sees keys i-window+1 .. i (causal only); 0: none
  int64_t sinks;   // with a window: first keys that every later query sees
  void* o_low;     // null, or (with o's strides) what rounding took from o
};

struct AttnBwdArgs {
  AttnArgs f;  // o = forward output (read), q/k/v inputs, lse
  const void* dout; int64_t do_b, do_h, do_s;
  void* dq; int64_t dq_b, dq_h, dq_s;
  void* dk; int64_t dk_b, dk_h, dk_s;
  void* dv; int64_t dv_b, dv_h, dv_s;
  float* ndelta;  // [B, H, Sq]: -D, written by attn_bwd_delta
  float* nlse2;   // [B, H, Sq]: -LSE * log2(e), written by attn_bwd_delta
  float* kv_part; // grouped backward: per-query-head dK, dV partials (f32), or null
  float* sink_part;    // sinks: f32 partials of their dK, dV (dkv_body)
  int sink_blocks;     // blocks of keys that hold sinks
  int sink_chunks;     // further blocks for each, which share the queries behind its window
  int sink_keys;       // how many sinks there are
  // (stored negated: the dK/dV and dQ steps add them, which saves a negation
  // per score)
};

// Rows of the sinks' f32 partials, of dK and then of dV: of the window of a
// block of sinks (grouped heads have that in kv_part) and of each chunk, and,
// of a last block of at most two waves, up to three more a chunk, since four or
// two waves then share a key.
struct SinkRows {
  int64_t heads;  // in all of the batch
  int keys, chunks;
  __host__ __device__ int shared() const { return keys < 64 ? keys : 64; }
  __host__ __device__ int64_t count() const {
    return heads * ((int64_t)keys * (chunks + 1) + (int64_t)shared() * 3 * chunks);
  }
  // Of head bh of the batch and a key in a block of `block`, from its window
  // (chunk -1) or a chunk, by the part-th of the waves that share the key.
  __device__ __forceinline__ int64_t at(int64_t bh, int64_t key, int chunk, int part, int block) const {
    if (part == 0) return ((int64_t)(chunk + 1) * heads + bh) * keys + key;
    return heads * keys * (chunks + 1) + ((int64_t)(3 * chunk + part - 1) * heads + bh) * shared() + key % block;
  }
};
__device__ __forceinline__ SinkRows sink_rows(const AttnBwdArgs& p) { return {p.f.B * p.f.H, p.sink_keys, p.sink_chunks}; }

// KW: keys of a wave of the kernel that left the partials, which has four.
//
// dK = scale * the sum of its f32 partials, dV likewise.  The first `plain`
// blocks take the keys that are no sinks of grouped heads, four head-dim
// elements per thread: the sum over the group's query heads, in head order.
// Each further block takes one sink, whose partials are many (a row of each
// block, or wave, that shared its queries, and each head): its threads sum every
// kSlices-th of them, and the slices are added in order.  (One thread for all
// of them waited for 112 loads in turn: 36 us for Gemma's local layer at 4096
// tokens, 15 with four slices of 64 threads each, 12.7 with sixteen.)
constexpr int kSumThreads = 1024;
template <typename T, int D, int KW>
__global__ void __launch_bounds__(kSumThreads) attn_bwd_window_sum(AttnBwdArgs p, uint32_t plain) {
  const AttnArgs& f = p.f;
  const int64_t hkn = f.H / f.group, plane = f.B * f.H * f.Skv * D;
  auto store = [&](f32x4 sk, f32x4 sv, int64_t b, int64_t hk, int64_t key, int64_t d) {
    V4<T> k4, v4;
#pragma unroll
    for (int e = 0; e < 4; ++e) k4.v[e] = (T)(sk[e] * f.scale), v4.v[e] = (T)sv[e];
    *(V4<T>*)((T*)p.dk + b * p.dk_b + hk * p.dk_h + key * p.dk_s + d) = k4;
    *(V4<T>*)((T*)p.dv + b * p.dv_b + hk * p.dv_h + key * p.dv_s + d) = v4;
  };
  f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sv = sk;
  if (blockIdx.x < plain) {
    const int64_t keys = f.Skv - p.sink_keys, i4 = (int64_t)blockIdx.x * kSumThreads + threadIdx.x;
    if (i4 >= f.B * hkn * keys * (D / 4)) return;
    const int64_t row = i4 / (D / 4), d = (i4 - row * (D / 4)) * 4, bhk = row / keys, hk = bhk % hkn, b = bhk / hkn;
    const int64_t key = row - bhk * keys + p.sink_keys;
#pragma unroll 4
    for (int64_t g = 0; g < f.group; ++g) {
      const float* pk = p.kv_part + (((g * f.B + b) * hkn + hk) * f.Skv + key) * D + d;
      sk += *(const f32x4*)pk, sv += *(const f32x4*)(pk + plane);
    }
    return store(sk, sv, b, hk, key, d);
  }
  constexpr int kSlices = kSumThreads / (D / 4);
  __shared__ f32x4 part[2][kSumThreads];
  const int64_t row = blockIdx.x - plain, key = row % p.sink_keys, bhk = row / p.sink_keys, hk = bhk % hkn, b = bhk / hkn;
  const int slice = threadIdx.x / (D / 4), d = (int)(threadIdx.x % (D / 4)) * 4;
  const SinkRows rows = sink_rows(p);
  const int64_t splane = rows.count() * D;
  // the waves that shared the sink's block
  const int waves = (int)min((int64_t)4, (p.sink_keys - key / (4 * KW) * (4 * KW) + KW - 1) / KW);
  const int parts = waves == 1 ? 4 : waves == 2 ? 2 : 1;
  const int each = 1 + p.sink_chunks * parts, total = (int)f.group * each;  // partials of a head, of all
#pragma unroll 4
  for (int i = slice; i < total; i += kSlices) {
    const int g = i / each, n = i - g * each, c = (n - 1) / parts;
    const int64_t h = hk * f.group + g;
    const float* pk = n == 0 && p.kv_part ? p.kv_part + (((g * f.B + b) * hkn + hk) * f.Skv + key) * D
                                          : p.sink_part + rows.at(b * f.H + h, key, n == 0 ? -1 : c, n == 0 ? 0 : n - 1 - c * parts, 4 * KW) * D;
    sk += *(const f32x4*)(pk + d), sv += *(const f32x4*)(pk + d + (n == 0 && p.kv_part ? plane : splane));
  }
  part[0][threadIdx.x] = sk, part[1][threadIdx.x] = sv;
  __syncthreads();
  if (slice) return;
  for (int i = 1; i < kSlices; ++i) sk += part[0][threadIdx.x + i * (D / 4)], sv += part[1][threadIdx.x + i * (D / 4)];
  store(sk, sv, b, hk, key, d);
}

// Blocks that share the steps behind the window of a block of sinks: eight
// steps each, which their four waves share where there are few sinks, so that
// one is shorter than a block of a window of 512 and more.  Fewer and longer
// ones where there would be more than 4096, sixteen a CU, in all: each leaves
// partials of its sinks.
inline int sink_chunks(int64_t heads, int64_t sq, int64_t window, int64_t sinks) {
  const int64_t rest = (sq + 63) / 64 - window / 64;
  if (sinks <= 0 || rest <= 0) return 0;
  const int64_t blocks = std::max<int64_t>(1, heads * ((sinks + 63) / 64));
  return (int)std::min<int64_t>((rest + 7) / 8, std::max<int64_t>(1, std::min<int64_t>(1024, 4096 / blocks)));
}
inline int64_t sink_keys(int64_t skv, int64_t sinks) { return std::min(skv, sinks); }

// The sinks' part of the arguments; their partials lie behind the workspace's
// other parts.
inline void window_parts(AttnBwdArgs& a, int64_t d) {
  const int64_t rows = a.f.B * a.f.H * a.f.Sq;
  a.sink_chunks = sink_chunks(a.f.B * a.f.H, a.f.Sq, a.f.window, a.f.sinks), a.sink_keys = (int)sink_keys(a.f.Skv, a.f.sinks);
  float* end = a.kv_part ? a.kv_part + 2 * a.f.B * a.f.H * a.f.Skv * d : a.ndelta + 2 * rows;
  a.sink_part = (float*)(((uintptr_t)end + 255) & ~(uintptr_t)255);
}

// Blocks of the two kinds of attn_bwd_window_sum.
inline int64_t window_sum_plain(const AttnBwdArgs& a, int D) {
  return a.kv_part ? (a.f.B * (a.f.H / a.f.group) * (a.f.Skv - a.sink_keys) * (D / 4) + kSumThreads - 1) / kSumThreads : 0;
}
inline int64_t window_sum_blocks(const AttnBwdArgs& a, int D) {
  return window_sum_plain(a, D) + a.f.B * (a.f.H / a.f.group) * a.sink_keys;
}

// What a launch can have, 2^32 threads, for all of a backward's before its first.
inline int window_launches(const AttnBwdArgs& a, int D, int64_t delta_threads, int64_t blocks) {
  const int64_t sums = window_sum_blocks(a, D);
  MI_REQUIRE(delta_threads < (1ll << 32) - kThreads, "mi355x_attn_bwd_sink: %lld threads", (long long)delta_threads);
  MI_REQUIRE(blocks < (1ll << 32) / kThreads, "mi355x_attn_bwd_sink: %lld blocks", (long long)blocks);
  MI_REQUIRE(sums < (1ll << 32) / kSumThreads, "mi355x_attn_bwd_sink: %lld sums of sinks and heads", (long long)sums);
  return MI355X_OK;
}

template <typename T, int D, int KW>
inline void window_sum_launch(const AttnBwdArgs& a, hipStream_t s) {
  const int64_t sums = window_sum_blocks(a, D);
  if (sums) attn_bwd_window_sum<T, D, KW><<<(unsigned)sums, kSumThreads, 0, s>>>(a, (uint32_t)window_sum_plain(a, D));
}

}  // namespace
}  // namespace mi
