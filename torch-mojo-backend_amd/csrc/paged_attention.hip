// Attention of new tokens over a paged key/value cache.
//
//   o = softmax(scale q K^T over the visible keys) V,
// key j visible to the query at position p iff j <= p and, with a window,
// p - j < window or j < sinks.
#include <math.h>

#include "paged_attention.h"

namespace mi {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// any type and head_dim: a block owns one query row and a split of its keys;
// each 16 lanes of it take every 16th key, a lane eight (or twice eight)
// channels, and the sixteen partial softmaxes are joined through LDS.  Query
// heads that share keys read them once each: for head_dims that the matrix-core
// kernel has no tile for, and f32 queries over 4 bits.  Loads and FMAs of shared
// rows bound it: one token of 8 sequences of 4096 keys, 32 heads over 8, bf16 at 96
// 103 us (37 at 128 on matrix cores), f32 over 4 bits at 128 103 (bf16 26); a prompt
// [1, 32 over 8, 2048, 96] 2.6 ms.
// ---------------------------------------------------------------------------
template <typename CT>
struct Oct8 {
  CT v[8];
};

template <typename CT>
__device__ __forceinline__ void load_oct(float (&x)[8], const void* base, int64_t at, const f16* sc, int oct, int d) {
  if constexpr (sizeof(CT) == 1) {
    const int s = oct % (d / kKvGroup);
    const uint32_t w = ((const uint32_t*)((const uint8_t*)base + at))[oct];
    const float step = (float)sc[2 * s], low = (float)sc[2 * s + 1];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(step, (float)(w >> (4 * (e / 2 + 4 * (e % 2))) & 15), low);
  } else {
    const Oct8<CT> o = *(const Oct8<CT>*)((const CT*)base + at + oct * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32(o.v[e]);
  }
}
// First channel of the eight that a row's piece `oct` holds.
template <typename CT>
__device__ __forceinline__ int oct_channel(int oct, int d) {
  if constexpr (sizeof(CT) == 1) {
    const int n = d / kKvGroup;
    return oct % n * kKvGroup + oct / n * 8;
  }
  return oct * 8;
}

template <typename T, typename CT>
__global__ void __launch_bounds__(kThreads) paged_attn_rows(DecodeArgs a) {
  __shared__ float so[16][256];
  __shared__ float sm[16], sl[16];
  const int d = (int)a.c.d, octs = d / 8;
  const int lane = threadIdx.x & 15, stream = threadIdx.x >> 4;
  const uint32_t row = blockIdx.x;  // over batch * heads * seq, token fastest
  const uint32_t t = row % a.seq, bh = row / a.seq;
  const int h = bh % a.heads;
  const int64_t b = bh / a.heads;
  const int hk = h / a.group;
  const bool real = (int)t < seq_count(a.s, b, a.seq);
  const int64_t at = (int64_t)a.s.starts[b] + t;
  int pos = real && at >= 0 && at <= kMaxPosition ? (int)at : -1;
  if (real && (pos < 0 || pos >= a.s.end) && a.s.error) *a.s.error = 1;
  const KeySpan span(pos, pos, a.window, a.sinks, a.s.end, 16);
  const int per = (span.tiles + a.splits - 1) / a.splits, first = blockIdx.y * per;
  const int last = min(first + per, span.tiles);
  float q[2][8], o[2][8], m = -INFINITY, l = 0.f;
  const T* Q = (const T*)a.q + b * a.q_b + h * a.q_h + t * a.q_t;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int oct = lane + 16 * u;
      q[u][e] = oct < octs ? to_f32(Q[oct_channel<CT>(oct, d) + e]) : 0.f;
      o[u][e] = 0.f;
    }
  for (int i = first; i < last; ++i) {
    const int j = span.tile(i) * 16 + stream;
    if (!visible(pos, j, a.window, a.sinks)) continue;
    uint32_t slot;
    const int page = page_of(a.s, b, j, &slot);
    if (page < 0) continue;
    const int64_t ka = page * a.c.k_phs[0] + hk * a.c.k_phs[1] + slot * a.c.k_phs[2];
    const int64_t va = page * a.c.v_phs[0] + hk * a.c.v_phs[1] + slot * a.c.v_phs[2];
    const f16 *ks = nullptr, *vs = nullptr;
    if constexpr (sizeof(CT) == 1) {
      ks = (const f16*)a.c.k_scales + page * a.c.ks_phs[0] + hk * a.c.ks_phs[1] + slot * a.c.ks_phs[2];
      vs = (const f16*)a.c.v_scales + page * a.c.vs_phs[0] + hk * a.c.vs_phs[1] + slot * a.c.vs_phs[2];
    }
    float s = 0.f, x[8];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (lane + 16 * u < octs) {
        load_oct<CT>(x, a.c.k, ka, ks, lane + 16 * u, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(q[u][e], x[e], s);
      }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) s += __shfl_xor(s, off, 64);
    s *= a.scale_log2;
    const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;  // of a NaN score: m, and p is NaN
    const float alpha = exp2f(m - ref), p = exp2f(s - ref);
    l = l * alpha + p;
    m = mn;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (lane + 16 * u < octs) {
        load_oct<CT>(x, a.c.v, va, vs, lane + 16 * u, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[u][e] = fmaf(p, x[e], o[u][e] * alpha);
      }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 16 * u < octs) so[stream][oct_channel<CT>(lane + 16 * u, d) + e] = o[u][e];
  if (lane == 0) sm[stream] = m, sl[stream] = l;
  __syncthreads();
  float mx = -INFINITY;
  for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sm[i]);
  const float base = mx == -INFINITY ? 0.f : mx;
  float total = 0.f, acc = 0.f;
  for (int i = 0; i < 16; ++i) {
    const float w = exp2f(sm[i] - base);
    total += w * sl[i];
    if ((int)threadIdx.x < d) acc += w * so[i][threadIdx.x];
  }
  const int64_t rows = a.batch * a.heads * a.seq;
  if (a.splits > 1) {
    if ((int)threadIdx.x < d) a.part_o[(blockIdx.y * rows + row) * d + threadIdx.x] = acc;
    if (threadIdx.x == 0) a.part_ml[blockIdx.y * rows + row] = make_float2(mx, total);
  } else if ((int)threadIdx.x < d) {
    ((T*)a.o)[b * a.o_b + h * a.o_h + t * a.o_t + threadIdx.x] = from_f32<T>(total != 0.f ? acc / total : 0.f);
  }
}

// Joins the (at most 64) splits of a row: o = sum_s 2^(m_s - m) o_s / sum_s
// 2^(m_s - m) l_s.  A lane of each wave weighs one split; the waves then take
// turns at the splits' rows, four channels a lane, so that a row costs two
// trips to memory however many splits it has (3.2 us for 4 rows of 5 splits,
// 4.0 for 64 splits: a launch and those trips).
template <typename T>
__global__ void __launch_bounds__(kThreads) paged_attn_join(DecodeArgs a) {
  __shared__ float4 sum[kThreads / 64][64];
  const int d = (int)a.c.d, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t rows = a.batch * a.heads * a.seq;
  const uint32_t row = blockIdx.x;
  const float2 ml = lane < a.splits ? a.part_ml[lane * rows + row] : make_float2(-INFINITY, 0.f);
  const float mx = wave_max(ml.x);
  const float w = mx == -INFINITY ? 1.f : exp2f(ml.x - mx);  // sums of 0, or of NaN
  const float total = wave_sum(w * ml.y);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kEach = 16;  // of 64 splits to a wave; all of their loads in flight
  const int ch = min(lane * 4, d - 4);
  float4 x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = wave + i * (kThreads / 64);
    if (s < a.splits) x[i] = *(const float4*)(a.part_o + (s * rows + row) * d + ch);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = wave + i * (kThreads / 64);
    if (s < a.splits) {
      const float ws = __shfl(w, s, 64);
      acc.x += ws * x[i].x, acc.y += ws * x[i].y, acc.z += ws * x[i].z, acc.w += ws * x[i].w;
    }
  }
  sum[wave][lane] = acc;
  __syncthreads();
  if ((int)threadIdx.x * 4 >= d) return;
  for (int i = 1; i < kThreads / 64; ++i) {
    const float4 x = sum[i][lane];
    acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
  }
  const uint32_t t = row % a.seq, bh = row / a.seq;
  const float inv = total != 0.f ? 1.f / total : 0.f;
  T* o = (T*)a.o + bh / a.heads * a.o_b + bh % a.heads * a.o_h + t * a.o_t + lane * 4;
  o[0] = from_f32<T>(acc.x * inv), o[1] = from_f32<T>(acc.y * inv);
  o[2] = from_f32<T>(acc.z * inv), o[3] = from_f32<T>(acc.w * inv);
}

// Keys that one query can see at most.
int64_t most_keys(const mi355x_paged_cache& c, int64_t width, int64_t window, int64_t sinks) {
  int64_t n = width * c.page_size;
  if (n > kMaxPosition) n = kMaxPosition;
  return window > 0 && window < n && sinks < n - window ? window + sinks : n;
}

// Keys up to which one block does a row: a second launch costs 3.5 us and as
// long again to reach the GPU, a block's tiles of 32 keys (16 in f32) about 2 us
// for each that a wave has.  Calls replayed one after another, us with one block
// and with splits: rows of 256 bytes and less 384 keys bf16 [8, 32 over 8, 128]
// 9.6 and 9.9, [1, 12, 64] 7.9 and 8.7 (f32 [3 x 4, 12, 64] 333 keys 11.4 and
// 10.2, but 11.9 and 14.1 as calls of their own); of 512 bytes bf16 [1, 4 over 1,
// 256] 256 keys 11.6 and 11.9, 384 keys 13.8 and 12.2; of 1024 bytes 256 keys f32
// [1, 4 over 1, 256] 20.3 and 17.3; an element a lane f32 [1, 4, 96] 128 keys 10.0
// and 10.0, 256 keys 15.9 and 13.0.  All of it for few rows: with more blocks than
// `few` below the parts cost more than they save up to 384 keys (bf16 [64, 4 over
// 1, 256] 14.8 and 13.2, [256] 21.7 and 36.1; f32 [16, 32, 96] 38 and 31, [32] 48 and
// 61).  The host knows the table's capacity, not the lengths: a short context in a
// wide table is split all the same.
int64_t keys_of_a_block(const mi355x_paged_cache& c, int dtype) {
  if (!paged_mfma_takes(c, dtype)) return 128;
  const int64_t bytes = c.d * (dtype == MI355X_F32 ? 4 : 2);
  return bytes <= 256 ? 384 : bytes <= 512 ? 256 : 128;
}

// Blocks that share the keys of a row, where rows alone are too few to fill
// the 256 CUs: eight blocks a CU in all (lengths differ, and the last round is
// shorter than with four: 282 against 276 us for the batch above
// paged_attn_mfma), of at least 128 keys each.
int plan_splits(const mi355x_paged_cache& c, int64_t width, int64_t batch, int64_t heads, int64_t seq, int64_t window,
                int64_t sinks, int dtype) {
  const int64_t keys = most_keys(c, width, window, sinks);
  int64_t blocks = batch * heads * seq, few = 512;
  if (paged_mfma_takes(c, dtype)) {
    few = 128;
    const int64_t rows = heads / c.kv_heads * seq, per = 16 * paged_mfma_row_tiles(rows, c.d);
    blocks = batch * c.kv_heads * ((rows + per - 1) / per);
  }
  if (keys <= 384 && (keys <= keys_of_a_block(c, dtype) || blocks > few)) return 1;
  int64_t n = blocks > 0 ? (2048 + blocks - 1) / blocks : 1;
  if (n > (keys + 127) / 128) n = (keys + 127) / 128;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

template <typename T>
int attn_launch(const DecodeArgs& a, int dtype, hipStream_t s) {
  const int64_t rows = a.batch * a.heads * a.seq;
  if (paged_mfma_takes(a.c, dtype)) {
    const int rc = paged_mfma_launch(a, dtype, s);
    if (rc) return rc;
  } else {
    const dim3 grid((unsigned)rows, (unsigned)a.splits);
    if (a.c.bits == 4) paged_attn_rows<T, uint8_t><<<grid, kThreads, 0, s>>>(a);
    else paged_attn_rows<T, T><<<grid, kThreads, 0, s>>>(a);
  }
  if (a.splits > 1) paged_attn_join<T><<<(unsigned)rows, kThreads, 0, s>>>(a);
  return check_launch("mi355x_paged_attn");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi355x_paged_attn_workspace_bytes(const mi355x_paged_cache* cache, int64_t table_width,
                                                     int64_t batch, int64_t heads, int64_t seq, int64_t window,
                                                     int64_t sinks, int dtype) {
  if (!cache || cache->kv_heads <= 0 || table_width < 0 || batch <= 0 || heads <= 0 || seq <= 0) return 0;
  const int splits = plan_splits(*cache, table_width, batch, heads, seq, window, sinks, dtype);
  return splits > 1 ? splits * batch * heads * seq * (cache->d + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int mi355x_paged_attn(void* o, const int64_t* o_bht, const void* q, const int64_t* q_bht,
                                 const mi355x_paged_cache* cache, const int32_t* table, int64_t table_stride,
                                 int64_t table_width, const int32_t* starts, const int32_t* counts, int64_t batch,
                                 int64_t heads, int64_t seq, double scale, int64_t window, int64_t sinks, int dtype,
                                 void* workspace, int64_t ws_bytes, int32_t* error, mi355x_stream_t stream) {
  PagedSeqs s;
  int rc = paged_args("mi355x_paged_attn", cache, table, table_stride, table_width, starts, counts, batch, seq, error,
                      &s);
  if (rc) return rc;
  if (dtype != MI355X_F32 && dtype != MI355X_BF16 && dtype != MI355X_F16)
    return fail(MI355X_EUNSUPPORTED, "mi355x_paged_attn: dtype %d is not supported (f32/bf16/f16)", dtype);
  MI_REQUIRE(cache->bits == 4 || cache->dtype == dtype, "mi355x_paged_attn: queries of dtype %d over pages of dtype %d",
             dtype, cache->dtype);
  MI_REQUIRE(heads > 0 && heads < 65536 && heads % cache->kv_heads == 0,
             "mi355x_paged_attn: heads (%lld) must be a multiple of kv_heads (%lld)", (long long)heads,
             (long long)cache->kv_heads);
  MI_REQUIRE(window >= 0 && sinks >= 0, "mi355x_paged_attn: bad window or sinks");
  MI_REQUIRE(isfinite(scale), "mi355x_paged_attn: scale must be finite");
  if (batch == 0 || seq == 0) return MI355X_OK;
  MI_REQUIRE(o && q, "mi355x_paged_attn: null pointer");
  MI_REQUIRE(rows_ok(q, q_bht, dtype_size(dtype)), "mi355x_paged_attn: rows of queries must be 16-byte aligned");
  // (a launch has below 2^32 threads: a block a row below, 16 rows and more a block on matrix cores)
  const int64_t most = paged_mfma_takes(*cache, dtype) ? 1ll << 31 : 1ll << 24;
  MI_REQUIRE(batch * heads * seq < most, "mi355x_paged_attn: batch x heads x tokens must be below %lld", (long long)most);
  const int64_t need = mi355x_paged_attn_workspace_bytes(cache, table_width, batch, heads, seq, window, sinks, dtype);
  if (need && (!workspace || ws_bytes < need))
    return fail(MI355X_EWORKSPACE, "mi355x_paged_attn: workspace %lld < %lld", (long long)ws_bytes, (long long)need);
  DecodeArgs a{};
  a.c = *cache, a.s = s;
  a.o = o, a.o_b = o_bht[0], a.o_h = o_bht[1], a.o_t = o_bht[2];
  a.q = q, a.q_b = q_bht[0], a.q_h = q_bht[1], a.q_t = q_bht[2];
  a.batch = batch, a.heads = (int)heads, a.group = (int)(heads / cache->kv_heads), a.seq = (int)seq;
  // a window or sinks past every position are the same as one that ends there
  a.window = (int)(window < kMaxPosition ? window : 0), a.sinks = (int)(sinks < kMaxPosition ? sinks : kMaxPosition);
  a.splits = plan_splits(*cache, table_width, batch, heads, seq, window, sinks, dtype);
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.part_o = (float*)workspace;
  a.part_ml = (float2*)(a.part_o + a.splits * batch * heads * seq * cache->d);
  if (dtype == MI355X_F32) return attn_launch<float>(a, dtype, (hipStream_t)stream);
  if (dtype == MI355X_BF16) return attn_launch<bf16>(a, dtype, (hipStream_t)stream);
  return attn_launch<f16>(a, dtype, (hipStream_t)stream);
}
