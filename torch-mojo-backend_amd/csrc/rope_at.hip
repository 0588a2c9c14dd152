// Rotary positions from the positions themselves: pair j of a row's first
// `turned` channels is turned by the angle p f_j of its position p,
//   (a, b) -> scale (a cos - b sin, b cos + a sin),
// the pair being channels (j, j + turned / 2), or (2j, 2j + 1) interleaved; the
// channels behind are copied.  `inverse` turns the other way, which with the
// same scale is the transposed map, the backward.
//
// Bound: HBM, every row read and written once.  There are no tables to make, keep
// or read: a block owns a few tokens and takes their angles for all heads of q
// and k, one sine and cosine a (token, pair), so that the arithmetic is a small
// part of what a row's bytes cost (bf16, 16384 tokens of 40 rows of 128: 65.6 us a
// direction, 336 MB, 5.1 TB/s).  An angle in f32 is off by its size times
// 2^-24, 0.06 at position 10^6; here p f_j / 2 pi is formed in f64, its whole
// turns are dropped there, and only the rest of a turn is rounded to f32.
#include <algorithm>

#include "common.h"

namespace mi {
namespace {

constexpr int kThreads = 256;
constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)

struct Side {
  const void* x;
  void* y;
  int64_t xb, xh, xt, yb, yh, yt;
};
struct RopeAt {
  Side q, k;
  const void* positions;
  int64_t positions_b;  // elements from one batch's positions to the next
  const double* freq;
  int64_t tokens;       // of the whole batch
  int seq, heads, rows;  // rows: heads of q, then of k
  int turned, d, per_row;
  int tpb;              // tokens of a block
  int share;            // items of a token that a block takes
  float scale, sign;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// VEC: channels of a load.  A row's items: half layout VEC pairs (two loads),
// interleaved VEC / 2 pairs (one load; a lane of VEC 1 takes a pair in two
// loads as in the half layout), then copies of VEC channels.
template <typename T, int VEC, bool LACED, typename P>
__global__ void __launch_bounds__(kThreads) rope_at_kernel(RopeAt p) {
  extern __shared__ float2 turn[];  // [tpb][turned / 2] scaled (cos, sin)
  constexpr bool TWO = !LACED || VEC == 1;
  constexpr int PAIRS = TWO ? VEC : VEC / 2;
  const int half = p.turned / 2, tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * p.tpb;
  const int nt = (int)min((int64_t)p.tpb, p.tokens - t0);
  for (int i = tid; i < nt * half; i += kThreads) {
    const int lt = i / half, j = i - lt * half;
    const int64_t t = t0 + lt, b = t / p.seq;
    const double turns = (double)((const P*)p.positions)[b * p.positions_b + (t - b * p.seq)] * p.freq[j] * kTurn;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c * p.scale, s * p.sign);
  }
  __syncthreads();
  const int items = p.rows * p.per_row, first = blockIdx.y * p.share, mine = min(items - first, p.share);
  const int turning = half / PAIRS;
  // the thread's items, kThreads apart, without a division each
  int lt = tid / mine, at = first + tid - lt * mine;
  const int dt = kThreads / mine, da = kThreads - dt * mine;
  constexpr int U = 4;
  while (lt < nt) {
    T* dst[U];
    int lo[U], hi[U], pair[U], n = 0;
    Vec<T, VEC> a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (lt >= nt) break;
      const int r = at / p.per_row, c = at - r * p.per_row;
      const bool isq = r < p.heads;
      const Side& s = isq ? p.q : p.k;
      const int64_t t = t0 + lt, bb = t / p.seq, tt = t - bb * p.seq, h = isq ? r : r - p.heads;
      const T* src = (const T*)s.x + bb * s.xb + h * s.xh + tt * s.xt;
      dst[u] = (T*)s.y + bb * s.yb + h * s.yh + tt * s.yt;
      if (c < turning) {
        pair[u] = lt * half + c * PAIRS;
        lo[u] = c * PAIRS * (LACED ? 2 : 1);
        hi[u] = LACED ? lo[u] + 1 : lo[u] + half;
        if constexpr (TWO) b[u] = *(const Vec<T, VEC>*)(src + hi[u]);
      } else {
        pair[u] = -1;
        lo[u] = p.turned + (c - turning) * VEC;
      }
      a[u] = *(const Vec<T, VEC>*)(src + lo[u]);
      n = u + 1;
      at += da, lt += dt;
      if (at >= first + mine) at -= mine, ++lt;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= n) break;
      if (pair[u] >= 0) {
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          const float2 w = turn[pair[u] + e];
          T& ra = TWO ? a[u].v[e] : a[u].v[2 * e];
          T& rb = TWO ? b[u].v[e] : a[u].v[(2 * e + 1) % VEC];
          const float x = to_f32(ra), y = to_f32(rb);
          ra = (T)fmaf(x, w.x, -(y * w.y));
          rb = (T)fmaf(y, w.x, x * w.y);
        }
        if constexpr (TWO) *(Vec<T, VEC>*)(dst[u] + hi[u]) = b[u];
      }
      *(Vec<T, VEC>*)(dst[u] + lo[u]) = a[u];
    }
  }
}

template <typename T, int VEC, bool LACED>
int launch(const RopeAt& a, bool wide, dim3 grid, size_t lds, hipStream_t s) {
  if (wide) rope_at_kernel<T, VEC, LACED, int64_t><<<grid, kThreads, lds, s>>>(a);
  else rope_at_kernel<T, VEC, LACED, int32_t><<<grid, kThreads, lds, s>>>(a);
  return check_launch("mi355x_rope_at");
}

template <typename T>
int run(RopeAt a, bool laced, bool wide_positions, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  auto aligned = [](const void* p, int64_t b, int64_t h, int64_t t) {
    return (uintptr_t)p % 16 == 0 && b % V == 0 && h % V == 0 && t % V == 0;
  };
  bool vec = a.d % V == 0 && a.turned % (laced ? V : 2 * V) == 0;
  for (const Side* x : {&a.q, &a.k})
    if (x->x) vec = vec && aligned(x->x, x->xb, x->xh, x->xt) && aligned(x->y, x->yb, x->yh, x->yt);
  const int v = vec ? V : 1;
  a.per_row = a.turned / (laced && vec ? V : 2 * v) + (a.d - a.turned) / v;
  const int items = a.rows * a.per_row, half = std::max(1, a.turned / 2);
  // tokens whose angles keep a block's threads busy once, but 1024 blocks where
  // the batch has them (f32, 2042 tokens of 24 rows of 64 with 32 channels turned:
  // 128 blocks of 16 tokens 14.8 us, 681 of 3 8.5, one each 7.8); where it has
  // few, a token's rows are shared by blocks, four items a thread, since each
  // then takes its angles again (one token of 5 rows of 256: one block, 3.0 us)
  a.tpb = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(16, kThreads / half), a.tokens / 1024));
  int64_t blocks = (a.tokens + a.tpb - 1) / a.tpb;
  int parts = 1;
  if (blocks < 512) parts = (int)std::min<int64_t>((items + kThreads * 4 - 1) / (kThreads * 4), std::max<int64_t>(1, 512 / blocks));
  a.share = (items + parts - 1) / parts;
  MI_REQUIRE(blocks * kThreads < (1ll << 32), "mi355x_rope_at: too many tokens");
  const dim3 grid((unsigned)blocks, (unsigned)((items + a.share - 1) / a.share));
  const size_t lds = (size_t)a.tpb * (a.turned / 2) * sizeof(float2);
  if (!vec) return laced ? launch<T, 1, true>(a, wide_positions, grid, lds, s) : launch<T, 1, false>(a, wide_positions, grid, lds, s);
  return laced ? launch<T, V, true>(a, wide_positions, grid, lds, s) : launch<T, V, false>(a, wide_positions, grid, lds, s);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi355x_rope_at(void* q_out, const int64_t* qo_bht, const void* q, const int64_t* q_bht, int64_t heads,
                              void* k_out, const int64_t* ko_bht, const void* k, const int64_t* k_bht, int64_t kv_heads,
                              const void* positions, int positions_dtype, int64_t positions_stride, const double* frequencies,
                              int64_t batch, int64_t seq, int64_t d, int64_t turned, int interleaved, double scale,
                              int inverse, int dtype, mi355x_stream_t stream) {
  MI_REQUIRE(batch >= 0 && seq >= 0 && heads >= 0 && kv_heads >= 0 && d > 0, "mi355x_rope_at: bad shape");
  MI_REQUIRE(turned >= 0 && turned % 2 == 0 && turned <= d, "mi355x_rope_at: %lld channels of %lld to turn", (long long)turned, (long long)d);
  MI_REQUIRE(positions_dtype == MI355X_I32 || positions_dtype == MI355X_I64, "mi355x_rope_at: positions must be int32 or int64");
  if (d > 4096) return fail(MI355X_EUNSUPPORTED, "mi355x_rope_at: head_dim %lld (up to 4096)", (long long)d);
  MI_REQUIRE(heads + kv_heads <= 65536 && seq < (1ll << 31), "mi355x_rope_at: too many heads or tokens");
  MI_REQUIRE(fabs(scale) < 1e38, "mi355x_rope_at: scale %g", scale);
  if (batch * seq == 0 || heads + kv_heads == 0) return MI355X_OK;
  MI_REQUIRE((!heads || (q && q_out)) && (!kv_heads || (k && k_out)) && positions && (frequencies || turned == 0),
             "mi355x_rope_at: null pointer");
  RopeAt a{};
  if (heads) a.q = Side{q, q_out, q_bht[0], q_bht[1], q_bht[2], qo_bht[0], qo_bht[1], qo_bht[2]};
  if (kv_heads) a.k = Side{k, k_out, k_bht[0], k_bht[1], k_bht[2], ko_bht[0], ko_bht[1], ko_bht[2]};
  a.positions = positions, a.positions_b = positions_stride, a.freq = frequencies;
  a.tokens = batch * seq, a.seq = (int)seq, a.heads = (int)heads, a.rows = (int)(heads + kv_heads);
  a.turned = (int)turned, a.d = (int)d;
  a.scale = (float)scale, a.sign = inverse ? -a.scale : a.scale;
  const bool wide = positions_dtype == MI355X_I64;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case MI355X_F32: return run<float>(a, interleaved != 0, wide, s);
    case MI355X_BF16: return run<bf16>(a, interleaved != 0, wide, s);
    case MI355X_F16: return run<f16>(a, interleaved != 0, wide, s);
  }
  return fail(MI355X_EUNSUPPORTED, "mi355x_rope_at: unsupported dtype %d", dtype);
}
