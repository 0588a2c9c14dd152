// Log-probabilities of given tokens, the distribution's entropy and its largest
// entries, from rows of logits, and their gradient:
//   m = max_j x_j, s = sum_j exp(x_j - m), logp_j = (x_j - m) - ln s
//   H = ln s - sum_j exp(x_j - m) (x_j - m) / s
//   dx_j = sum_i g_i [j = token i] - p_j (sum_i g_i + g_H (logp_j + H)),
// i over the given token and the top ones.  x - m is kept apart from ln s (both
// are saved for the backward): x - lse would lose the bits that m and ln s share,
// and H is a difference of the two terms above, not of lse and sum p x.
//
// Bound: HBM.  The forward reads the logits once: a block holds a row, or a
// segment of one, in registers, so that the maximum, the sums and the search for
// the largest entries are passes over registers.  Long rows and few rows are cut
// into segments, whose results a second kernel joins.  The backward reads the
// logits once and writes the gradient once.  1000 x 50257 f32 with entropy and 5
// top entries: 51.5 us and 5 to join, 201 MB; the gradient of 8192 x 50257 bf16 320
// us, 1.65 GB, 5.1 TB/s.
//
// Largest entries: a lane's maximum is known from the first pass.  The k-th
// largest of a wave's 64 is a bound that k entries of the row reach, and so is
// the largest of the waves' bounds; the entries that reach it, a few more than k
// as a rule, go to a list, and an entry's place is the number of entries that
// come before it.  Rows with so many ties that the list is too short, and those
// with a NaN (which comes first, as in a sort), take their entries one after
// another, the largest key below the last one each.  Keys are the value's order
// and the index, so that equal values stand by index.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace mi {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloor = -200.f;  // exponents (base 2) below are as good as this: exp2 of it is 0 in f32
constexpr int kMostTop = 64;
typedef unsigned long long u64;

__device__ __forceinline__ float hw_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// (a NaN stays one)
__device__ __forceinline__ float not_below(float x) { return x < kFloor ? kFloor : x; }

// 16 bytes of a row, V elements.  Rows begin anywhere: a load need not be
// aligned.
template <typename T>
struct Chunk {
  static constexpr int V = 16 / sizeof(T);
  u32x4 w;
  // whole elements i .. i + V - 1
  __device__ __forceinline__ void load(const T* row, int64_t i) { __builtin_memcpy(&w, row + i, 16); }
  // those of them that lie before n and from `first` on, for the others `rest`
  __device__ __forceinline__ void load_end(const T* row, int64_t i, int64_t n, int64_t first = 0, float rest = -INFINITY) {
    union { T v[V]; u32x4 w; } u;
#pragma unroll
    for (int e = 0; e < V; ++e) u.v[e] = i + e >= first && i + e < n ? row[i + e] : (T)rest;
    w = u.w;
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[e]);
    } else {
      const uint32_t u = w[e >> 1];
      return to_f32(__builtin_bit_cast(T, (unsigned short)(e & 1 ? u >> 16 : u & 0xffffu)));
    }
  }
  // what was made of it is made again, not held (16 chunks' 128 values would
  // take half of a lane's registers)
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t u = w[e];
      asm volatile("" : "+v"(u));
      w[e] = u;
    }
  }
};

// Elements between a 16-byte boundary and p (a row of an odd number of 16-bit
// elements begins anywhere; loads that do not lie on 4 bytes run at 90% of the others' rate).
template <typename T>
__device__ __forceinline__ int lead_of(const T* p) { return (int)((uintptr_t)p & 15) / (int)sizeof(T); }

// Where a value stands among f32 values, and the key that a larger value, or of
// equal ones the lower index, has the larger of.  0 is no entry's key.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 is 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o == 0xffffffffu ? 0x7fc00000u : o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ u64 key_of(float x, uint32_t index) { return (u64)order_of(x) << 32 | (uint32_t)~index; }

struct LpArgs {
  const void* x;
  int64_t ld, n, c;
  const int64_t* tokens;
  int64_t ignore;
  int32_t* error;
  float *logprobs, *entropy, *stats, *top_logprobs;  // stats: [n][2], m and ln s, or null
  int64_t* top_tokens;
  int top;
  int segments;       // of a row; more than one: partials
  int64_t seg;        // elements of a segment
  float* part;        // [n][segments][3]: m, s, sum of exp(x - m) (x - m)
  u64* part_keys;     // [n][segments][top]
};

// What a row's statistics give, by one thread.
template <typename T>
__device__ __forceinline__ void finish_row(const LpArgs& p, int64_t row, float m, float s, float t) {
  const float ls = log2f(s) * kLn2;
  if (p.stats) p.stats[2 * row] = m, p.stats[2 * row + 1] = ls;
  if (p.entropy) p.entropy[row] = ls - t / s;
  if (p.logprobs) {
    const int64_t k = p.tokens[row];
    float lp = 0.f;
    if (k != p.ignore) {
      if (k < 0 || k >= p.c) {
        if (p.error) *p.error = 1;
      } else {
        lp = to_f32(((const T*)p.x)[row * p.ld + k]) - m - ls;
      }
    }
    p.logprobs[row] = lp;
  }
}
__device__ __forceinline__ void put_top(const LpArgs& p, int64_t row, int place, u64 key, float m, float ls) {
  p.top_logprobs[row * p.top + place] = value_of((uint32_t)(key >> 32)) - m - ls;
  p.top_tokens[row * p.top + place] = (int64_t)(uint32_t)~(uint32_t)key;
}

__device__ __forceinline__ u64 wave_max_key(u64 k) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const u64 o = __shfl_xor(k, off, 64);
    k = o > k ? o : k;
  }
  return k;
}

// NW waves take a row's segment, CPT chunks a lane; NW = 1: a block of four waves
// takes four.
template <typename T, int NW, int CPT>
struct LpShape {
  static constexpr int kThreads = NW == 1 ? 256 : 64 * NW;
  static constexpr int kUnits = kThreads / (64 * NW);  // segments of a block
  static constexpr int64_t kMost = (int64_t)64 * NW * CPT * Chunk<T>::V;  // elements of a segment
  static constexpr int kList = NW == 1 ? 256 : 1024;
};

template <typename T, int NW, int CPT, bool ENT>
__global__ void __launch_bounds__((LpShape<T, NW, CPT>::kThreads)) lp_rows(LpArgs p) {
  typedef LpShape<T, NW, CPT> S;
  constexpr int V = Chunk<T>::V, LIST = S::kList;
  __shared__ u64 list_s[S::kUnits][LIST];
  __shared__ float red[S::kUnits][NW][2];
  __shared__ float bounds[S::kUnits][NW];
  __shared__ u64 best[S::kUnits][NW];
  __shared__ int count_s[S::kUnits];
  const int unit = S::kUnits == 1 ? 0 : threadIdx.x >> 6;
  const int tid = S::kUnits == 1 ? threadIdx.x : threadIdx.x & 63, lane = threadIdx.x & 63, wave = tid >> 6;
  const int64_t item = (int64_t)blockIdx.x * S::kUnits + unit;
  if (item >= p.n * p.segments) return;  // (a wave as a whole; nothing below waits for other units')
  const int64_t row = item / p.segments, e0 = (item - row * p.segments) * p.seg, len = min(p.seg, p.c - e0);
  const T* const x = (const T*)p.x + row * p.ld + e0;
  // of the unit's waves; one wave needs no barrier but what LDS itself orders
  auto sync = [&] {
    if constexpr (NW == 1) __builtin_amdgcn_wave_barrier(), __threadfence_block();
    else __syncthreads();
  };
  Chunk<T> ch[CPT];
  const int nfull = (int)(len / V), nit = ((int)((len + V - 1) / V) + 64 * NW - 1) / (64 * NW);
  Chunk<T> end;  // the last chunk, where it is short, in the lane that has it; -inf elsewhere
  end.load_end(x, (int64_t)nfull * V, nfull % (64 * NW) == tid ? len : 0);
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    if (i >= nit) continue;
    if (tid + i * 64 * NW < nfull) ch[i].load(x, (int64_t)(tid + i * 64 * NW) * V);
    else ch[i] = end;
  }
  if (tid == 0) count_s[unit] = 0;
  float mine = -INFINITY;  // NaN where the lane has one
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    if (i >= nit) continue;
    float v[V + 1];
    v[0] = mine;
#pragma unroll
    for (int e = 0; e < V; ++e) v[1 + e] = ch[i].get(e);
    mine = max_nan(v);
    ch[i].forget();
  }
  float m = wave_max_nan(mine);
  if constexpr (NW > 1) {
    if (lane == 0) red[unit][wave][0] = m;
    sync();
    m = red[unit][0][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = nan_max(m, red[unit][w][0]);
    sync();
  }
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    if (i >= nit) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // (NaNs that the floor hides are in m)
      const float d = (ch[i].get(e) - m) * kLog2e;
      if constexpr (ENT) {
        const float f = fmaxf(d, kFloor), q = hw_exp2(f);
        s += q, t = fmaf(q, f, t);
      } else {
        s += hw_exp2(d);
      }
    }
    ch[i].forget();
  }
  s = wave_sum(s), t = wave_sum(t);
  if constexpr (NW > 1) {
    if (lane == 0) red[unit][wave][0] = s, red[unit][wave][1] = t;
    sync();
    s = t = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += red[unit][w][0], t += red[unit][w][1];
  }
  t *= kLn2;
  if (tid == 0) {
    if (p.segments == 1) finish_row<T>(p, row, m, s, t);
    else p.part[3 * item] = m, p.part[3 * item + 1] = s, p.part[3 * item + 2] = t;
  }
  if (p.top == 0) return;

  u64* const list = list_s[unit];
  const int k = p.top;
  const float ls = log2f(s) * kLn2;
  auto put = [&](int place, u64 key) {
    if (p.segments == 1) put_top(p, row, place, key, m, ls);
    else p.part_keys[item * k + place] = key;
  };
  if (m == m) {
    int before = 0;  // lanes of the wave whose maximum is larger
    for (int i = 0; i < 64; ++i) before += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), i)) > mine;
    float bound = before < k ? mine : INFINITY;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) bound = fminf(bound, __shfl_xor(bound, off, 64));
    if constexpr (NW > 1) {
      if (lane == 0) bounds[unit][wave] = bound;
      sync();
#pragma unroll
      for (int w = 0; w < NW; ++w) bound = fmaxf(bound, bounds[unit][w]);
    }
    if (mine >= bound) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        if (i >= nit) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = ch[i].get(e);
          const int at = (tid + i * 64 * NW) * V + e;
          if (v >= bound && at < len) {
            const int place = atomicAdd(&count_s[unit], 1);
            if (place < LIST) list[place] = key_of(v, (uint32_t)(e0 + at));
          }
        }
      }
    }
    sync();
    const int count = count_s[unit];
    if (count <= LIST) {
      for (int i = tid; i < count; i += 64 * NW) {
        const u64 key = list[i];
        int place = 0;
        for (int j = 0; j < count; ++j) place += list[j] > key;
        if (place < k) put(place, key);
      }
      for (int i = count + tid; i < k; i += 64 * NW) put(i, 0);  // a segment of fewer entries
      return;
    }
  }
  // one after another, from memory: these rows are rare, and kept in registers
  // for them 128 values' keys would take all of a lane's
  u64 last = ~0ull;
  for (int i = 0; i < k; ++i) {
    u64 key = 0;
    if (last) {
#pragma unroll 1
      for (int c = 0; c < nit; ++c) {
        const int at = (tid + c * 64 * NW) * V;
        Chunk<T> w = end;
        if (at + V <= len) w.load(x, at);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const u64 o = key_of(w.get(e), (uint32_t)(e0 + at + e));
          if (at + e < len && o < last && o > key) key = o;
        }
      }
      key = wave_max_key(key);
      if constexpr (NW > 1) {
        sync();
        if (lane == 0) best[unit][wave] = key;
        sync();
#pragma unroll
        for (int w = 0; w < NW; ++w) key = best[unit][w] > key ? best[unit][w] : key;
      }
    }
    if (tid == 0) put(i, key);
    last = key;
  }
}

// Without top entries nothing is looked at twice: a block walks its segment with
// a running maximum m, s = sum 2^f and t = sum 2^f f, f = (x - m) log2(e), which
// move to a new maximum as t = (t + s d) 2^d, s = s 2^d.  An exponential an element
// and what stands around it bound the walk, so f is one instruction, x log2(e) -
// r with r = m log2(e) as rounded, and what r is off by is taken out of the sums at
// the end; that holds for the finite x below kNear, and -inf makes 2^f f a NaN.  A
// wave that meets anything else takes its batch again, and those that follow,
// with f as it is defined, an exponent of -200 for all below it (8192 x 50257
// bf16, 0.82 GB, 192 us with that for all, 176 so, 4.7 TB/s).
constexpr int kStreamThreads = 256;
constexpr float kNear = 32768.f;
// What fills a row's last chunk: 2^f of it is 0 for every m below kNear.
template <typename T>
constexpr float kFill = -1e30f;
template <>
constexpr float kFill<f16> = -65504.f;
template <typename T, bool ENT>
__global__ void __launch_bounds__(kStreamThreads) lp_stream(LpArgs p) {
  constexpr int V = Chunk<T>::V, U = 4, W = kStreamThreads / 64;
  __shared__ float red[W][3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t item = blockIdx.x, row = item / p.segments, e0 = (item - row * p.segments) * p.seg;
  // chunks are cut where memory is, from up to V - 1 elements before the segment
  const T* const begin = (const T*)p.x + row * p.ld + e0;
  const int first = lead_of(begin), len = first + (int)min(p.seg, p.c - e0), nc = (len + V - 1) / V;
  const T* const x = begin - first;
  float m = -INFINITY, r = 0.f, s = 0.f, t = 0.f;
  bool nan = false, near = true;
  auto settle = [&]() {  // the sums with f = (x - m) log2(e): by 2^-e, e = m log2(e) - r
    if (m == -INFINITY) return;
    const float e = fmaf(m, kLog2e, -r), k = e * kLn2, g = fmaf(0.5f * k, k, -k);
    t = fmaf(-e, s, t);
    t = fmaf(g, t, t), s = fmaf(g, s, s);
  };
  for (int c0 = tid; c0 < nc; c0 += kStreamThreads * U) {
    Chunk<T> ch[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (c0 + u * kStreamThreads) * V;
      if (i >= first && i + V <= len) ch[u].load(x, i);
      else ch[u].load_end(x, i, len, first, kFill<T>);
    }
    if (near) {
      const float m0 = m, r0 = r, s0 = s, t0 = t;
      bool far = false;
      float v[U * V];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) v[u * V + e] = ch[u].get(e);
      const float top = max_nan(v);
      if (top > m) {
        const float r1 = top * kLog2e, d = m == -INFINITY ? kFloor : fmaxf(r - r1, kFloor), f = hw_exp2(d);
        if constexpr (ENT) t = fmaf(s, d, t) * f;
        s *= f, m = top, r = r1;
        far = !(fabsf(top) < kNear);
      }
#pragma unroll
      for (int e = 0; e < U * V; ++e) {
        const float f = fmaf(v[e], kLog2e, -r), q = hw_exp2(f);
        s += q;
        if constexpr (ENT) t = fmaf(q, f, t);
      }
      const float sum = ENT ? t : s;
      if (!__builtin_amdgcn_ballot_w64(far || sum != sum)) continue;
      m = m0, r = r0, s = s0, t = t0;
      settle();
      near = false;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (c0 + u * kStreamThreads) * V;
      if (i < first || i + V > len) ch[u].load_end(x, i, len, first);
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = ch[u].get(e);
      const float top = max_nan(v);
      nan |= top != top;
      if (top > m) {
        const float d = fmaxf((m - top) * kLog2e, kFloor), f = hw_exp2(d);
        if constexpr (ENT) t = fmaf(s, d, t) * f;
        s *= f, m = top;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float f = fmaxf((v[e] - m) * kLog2e, kFloor), q = hw_exp2(f);
        s += q;
        if constexpr (ENT) t = fmaf(q, f, t);
      }
    }
  }
  if (near) settle();
  if (nan) m = __uint_as_float(0x7fc00000u);
  // to the block's maximum; what a NaN or an infinity makes of the sums is in m
  float all = wave_max_nan(m);
  if (lane == 0) red[wave][0] = all;
  __syncthreads();
  all = red[0][0];
#pragma unroll
  for (int w = 1; w < W; ++w) all = nan_max(all, red[w][0]);
  const float d = fmaxf((m - all) * kLog2e, kFloor), f = hw_exp2(d);
  t = wave_sum(fmaf(s, d, t) * f), s = wave_sum(s * f);
  if (lane == 0) red[wave][1] = s, red[wave][2] = t;
  __syncthreads();
  if (tid) return;
  s = t = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) s += red[w][1], t += red[w][2];
  t *= kLn2;
  if (p.segments == 1) finish_row<T>(p, row, all, s, t);
  else p.part[3 * item] = all, p.part[3 * item + 1] = s, p.part[3 * item + 2] = t;
}

// A row's segments: one block, kJoinList keys at most.  The bound here: with r =
// ceil(k / segments), the ceil(k / r)-th largest of the segments' r-th keys (of
// their maxima, where there are k segments), which r entries of each of as many
// segments reach.
constexpr int kJoinThreads = 256, kJoinList = 4096, kMostSegments = 512;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) lp_join(LpArgs p) {
  __shared__ u64 list[kJoinList];
  __shared__ u64 heads[kMostSegments];
  __shared__ float red[kJoinThreads / 64][3];
  __shared__ u64 bound_s;
  __shared__ int count_s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = p.segments, k = p.top;
  const int64_t row = blockIdx.x;
  const float* const part = p.part + row * g * 3;
  const u64* const keys = p.part_keys + row * g * k;
  const int r = k ? (k + g - 1) / g : 1, need = k ? (k + r - 1) / r : 0;
  if (tid == 0) count_s = 0, bound_s = 0;
  float m = -INFINITY;
  for (int i = tid; i < g; i += kJoinThreads) {
    m = nan_max(m, part[3 * i]);
    if (k) heads[i] = keys[(int64_t)i * k + r - 1];
  }
  m = wave_max_nan(m);
  if (lane == 0) red[wave][0] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 64; ++w) m = nan_max(m, red[w][0]);
  float s = 0.f, t = 0.f;
  for (int i = tid; i < g; i += kJoinThreads) {
    const float ps = part[3 * i + 1], pt = part[3 * i + 2], d = not_below((part[3 * i] - m) * kLog2e), f = hw_exp2(d);
    // of a segment whose entries are all -inf nothing counts, and its own sums are NaN
    const bool none = part[3 * i] == -INFINITY && m > -INFINITY;
    s += none ? 0.f : ps * f, t += none ? 0.f : (pt + ps * d * kLn2) * f;
    if (k) {
      const u64 mine = heads[i];
      int before = 0;
      for (int j = 0; j < g; ++j) before += heads[j] > mine;
      if (mine && before == need - 1) bound_s = mine;
    }
  }
  s = wave_sum(s), t = wave_sum(t);
  if (lane == 0) red[wave][1] = s, red[wave][2] = t;
  __syncthreads();
  s = t = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 64; ++w) s += red[w][1], t += red[w][2];
  if (tid == 0) finish_row<T>(p, row, m, s, t);
  if (!k) return;
  const u64 bound = bound_s;
  for (int i = tid; i < g * k; i += kJoinThreads) {
    const u64 key = keys[i];
    if (key && key >= bound) list[atomicAdd(&count_s, 1)] = key;
  }
  __syncthreads();
  const float ls = log2f(s) * kLn2;
  const int count = count_s;
  for (int i = tid; i < count; i += kJoinThreads) {
    const u64 key = list[i];
    int place = 0;
    for (int j = 0; j < count; ++j) place += list[j] > key;
    if (place < k) put_top(p, row, place, key, m, ls);
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
struct LpBwd {
  void* dx;
  const void* x;
  int64_t ld_dx, ld, n, c;
  const float *stats, *entropy;
  const int64_t *tokens, *top_tokens;
  const float *d_logprobs, *d_entropy, *d_top;  // null: none
  int64_t ignore;
  int top;
  int64_t share;  // columns of a block, a multiple of a chunk
  int past;       // whether the gradient is stored past the caches
};

// 16 bytes at an element's alignment.
template <typename T>
using Chunk8 = uint32_t __attribute__((ext_vector_type(4), aligned(sizeof(T))));

// Rows go last first: the forward has read those last, and what of them the 256
// MB cache still holds is not read from memory again.  A gradient that does not
// fit that cache is stored past it, or it would push the logits out and be written
// back during the next kernel (8192 x 50257 bf16, forward and backward, 2.47 GB:
// 582 us first to last, 560 last to first, 525 with both, 496 with chunks that lie
// on 16 bytes and the forward's shorter exponent; a small gradient stays for the
// product that reads it next).
constexpr int64_t kMemoryCache = 256ll << 20;
constexpr int kBwdThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kBwdThreads) lp_bwd(LpBwd p) {
  constexpr int V = Chunk<T>::V, U = 4;
  const int tid = threadIdx.x;
  const int64_t row = p.n - 1 - blockIdx.x, c0 = blockIdx.y * p.share, c1 = min(p.ld_dx, c0 + p.share);
  const T* const x = (const T*)p.x + row * p.ld;
  T* const dx = (T*)p.dx + row * p.ld_dx;
  const float m = p.stats[2 * row], ls = p.stats[2 * row + 1];
  const int64_t token = p.d_logprobs ? p.tokens[row] : -1;
  const bool given = p.d_logprobs && token != p.ignore && token >= 0 && token < p.c;
  const float g = given ? p.d_logprobs[row] : 0.f, gh = p.d_entropy ? p.d_entropy[row] : 0.f;
  float total = g;
  if (p.d_top)
    for (int i = 0; i < p.top; ++i) total += p.d_top[row * p.top + i];
  // -p_j (total + gh (logp_j + H)), logp_j = z_j ln 2
  const float l2 = ls * kLog2e, base = gh != 0.f ? fmaf(gh, p.entropy[row], total) : total, slope = gh * kLn2;
  auto at = [&](float v) {
    const float z = not_below(fmaf(v - m, kLog2e, -l2));
    return -hw_exp2(z) * fmaf(slope, z, base);
  };
  // chunks lie on 16 bytes where those of the row and of its gradient can
  const int64_t begin = c0 - (((uintptr_t)(x + c0) ^ (uintptr_t)(dx + c0)) & 15 ? 0 : lead_of(x + c0));
  for (int64_t j0 = begin + tid * V; j0 < c1; j0 += kBwdThreads * V * U) {
    Chunk<T> ch[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + u * kBwdThreads * V;
      if (j < c1) {
        if (j >= c0 && j + V <= p.c) ch[u].load(x, j);
        else ch[u].load_end(x, j, p.c, c0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + u * kBwdThreads * V;
      if (j >= c1) break;
      float r[V];
      struct { T v[V]; } o;
#pragma unroll
      for (int e = 0; e < V; ++e) r[e] = at(ch[u].get(e));
      if (j + V > p.c || (uint64_t)(token - j) < V) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (given && j + e == token) r[e] += g;
          if (j + e >= p.c) r[e] = 0.f;  // the columns that pad a row
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) o.v[e] = (T)r[e];
      if (j >= c0 && j + V <= c1) {
        Chunk8<T> w;
        __builtin_memcpy(&w, o.v, 16);
        if (p.past) __builtin_nontemporal_store(w, (Chunk8<T>*)(dx + j));
        else *(Chunk8<T>*)(dx + j) = w;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (j + e >= c0 && j + e < c1) dx[j + e] = o.v[e];
      }
    }
  }
  if (!p.d_top) return;
  // the top tokens' columns again, over what the block has written
  __syncthreads();
  for (int i = tid; i < p.top; i += kBwdThreads) {
    const int64_t j = p.top_tokens[row * p.top + i];
    if (j < c0 || j >= min(c1, p.c)) continue;
    float r = at(to_f32(x[j])) + p.d_top[row * p.top + i];
    if (given && j == token) r += g;
    dx[j] = (T)r;
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// How rows are cut.  A row that one wave's, or one block's, registers hold is
// not, where there are enough rows to fill the 256 CUs; else into segments of 8 KB
// and more for 512 blocks in all, of which the join takes kJoinList keys (one
// bf16 row of 262144, 20 top entries: 9.8 us and 5.8 to join 64 segments, 11.4 and
// 4.8 of 32, 8.5 and 8.3 of 128).  Rows of 8192 x 50257 bf16 stream in 176 us; held
// in registers they took 239, in blocks of 16 waves 346.
struct LpPlan {
  int waves;      // of a segment: 1, 4 or 8; 0: lp_stream's block
  int64_t segments, seg;
};
template <typename T>
LpPlan plan_of(int64_t n, int64_t c, int top) {
  constexpr int V = Chunk<T>::V;
  constexpr int64_t one = LpShape<T, 1, 16>::kMost, four = LpShape<T, 4, 8>::kMost, eight = LpShape<T, 8, 16>::kMost;
  if (c <= one && (n >= 512 || c <= one / 4)) return {1, 1, c};
  if (!top && n >= 512) return {0, 1, c};
  if (c <= eight && n >= 256) return {8, 1, c};
  int64_t g = (c + eight - 1) / eight;
  if (n < 512) g = std::max<int64_t>(g, std::min<int64_t>((512 + n - 1) / n, c / (four / 4)));
  g = std::max<int64_t>(1, std::min<int64_t>(g, std::min(kMostSegments, top ? kJoinList / top : kMostSegments)));
  const int64_t seg = ((c + g - 1) / g + V - 1) / V * V;
  g = (c + seg - 1) / seg;
  return {!top ? 0 : seg <= one / 8 ? 1 : seg <= four ? 4 : 8, g, g == 1 ? c : seg};
}

template <typename T, int NW, int CPT>
void lp_launch(const LpArgs& a, hipStream_t s) {
  typedef LpShape<T, NW, CPT> S;
  const unsigned blocks = ceil_div(a.n * a.segments, S::kUnits);
  if (a.entropy) lp_rows<T, NW, CPT, true><<<blocks, S::kThreads, 0, s>>>(a);
  else lp_rows<T, NW, CPT, false><<<blocks, S::kThreads, 0, s>>>(a);
}

template <typename T>
int lp_fwd(LpArgs a, void* workspace, int64_t ws_bytes, hipStream_t s) {
  const LpPlan g = plan_of<T>(a.n, a.c, a.top);
  a.segments = (int)g.segments, a.seg = g.seg;
  MI_REQUIRE((g.waves == 0 || g.seg <= LpShape<T, 8, 16>::kMost), "mi355x_token_logprobs_fwd: %lld columns", (long long)a.c);
  MI_REQUIRE(a.n * g.segments < (1ll << 32) / 1024, "mi355x_token_logprobs_fwd: %lld rows", (long long)a.n);
  if (g.segments > 1) {
    const int64_t items = a.n * g.segments, need = items * (8 * (int64_t)a.top + 12) + 16;
    if (!workspace || ws_bytes < need)
      return fail(MI355X_EWORKSPACE, "mi355x_token_logprobs_fwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
    a.part_keys = (u64*)(((uintptr_t)workspace + 15) & ~(uintptr_t)15);
    a.part = (float*)(a.part_keys + items * a.top);
  }
  if (g.waves == 0) {
    const unsigned blocks = (unsigned)(a.n * g.segments);
    if (a.entropy) lp_stream<T, true><<<blocks, kStreamThreads, 0, s>>>(a);
    else lp_stream<T, false><<<blocks, kStreamThreads, 0, s>>>(a);
  } else if (g.waves == 1) lp_launch<T, 1, 16>(a, s);
  else if (g.waves == 4) lp_launch<T, 4, 8>(a, s);
  else lp_launch<T, 8, 16>(a, s);
  if (g.segments > 1) lp_join<T><<<(unsigned)a.n, kJoinThreads, 0, s>>>(a);
  return check_launch("mi355x_token_logprobs_fwd");
}

template <typename T>
int lp_bwd_launch(LpBwd a, hipStream_t s) {
  constexpr int64_t V = Chunk<T>::V;
  // a block a row, or where rows are few, 512 blocks in all of 2048 chunks at least
  int64_t parts = a.n < 512 ? std::min<int64_t>((512 + a.n - 1) / a.n, a.ld_dx / V / 2048 + 1) : 1;
  a.past = a.n * a.ld_dx * (int64_t)sizeof(T) > kMemoryCache;
  a.share = ((a.ld_dx + parts - 1) / parts + V - 1) / V * V;
  parts = (a.ld_dx + a.share - 1) / a.share;
  lp_bwd<T><<<dim3((unsigned)a.n, (unsigned)parts), kBwdThreads, 0, s>>>(a);
  return check_launch("mi355x_token_logprobs_bwd");
}

int lp_check(const char* what, int64_t n, int64_t c, int64_t ld, int top, int dtype) {
  // (a walk's 32-bit places go a batch past a row's end: lp_stream's 1024 chunks of 8)
  MI_REQUIRE(n >= 0 && c > 0 && c < (1ll << 31) - (1 << 14), "%s: %lld rows of %lld columns", what, (long long)n, (long long)c);
  MI_REQUIRE(n < (1ll << 23), "%s: %lld rows", what, (long long)n);
  MI_REQUIRE(ld >= 0 && top >= 0 && top <= c, "%s: stride %lld, %d top entries", what, (long long)ld, top);
  if (top > kMostTop) return fail(MI355X_EUNSUPPORTED, "%s: %d top entries (up to %d)", what, top, kMostTop);
  if (dtype != MI355X_F32 && dtype != MI355X_BF16 && dtype != MI355X_F16)
    return fail(MI355X_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  return MI355X_OK;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi355x_token_logprobs_workspace_bytes(int64_t n, int64_t c, int top, int dtype) {
  if (lp_check("mi355x_token_logprobs_workspace_bytes", n, c, 0, top, dtype)) return -1;
  const LpPlan g = n == 0 ? LpPlan{1, 1, c} : dtype == MI355X_F32 ? plan_of<float>(n, c, top) : plan_of<bf16>(n, c, top);
  return g.segments == 1 ? 0 : n * g.segments * (8 * (int64_t)top + 12) + 16;
}

extern "C" int mi355x_token_logprobs_fwd(float* logprobs, float* entropy, float* stats, float* top_logprobs,
                                         int64_t* top_tokens, const void* logits, int dtype, int64_t ld,
                                         const int64_t* tokens, int64_t n, int64_t c, int top, int64_t ignore_index,
                                         int32_t* error, void* workspace, int64_t ws_bytes, mi355x_stream_t stream) {
  const int rc = lp_check("mi355x_token_logprobs_fwd", n, c, ld, top, dtype);
  if (rc || n == 0) return rc;
  MI_REQUIRE(logits && (!logprobs || tokens) && (!top || (top_logprobs && top_tokens)),
             "mi355x_token_logprobs_fwd: null pointer");
  LpArgs a{};
  a.x = logits, a.ld = ld, a.n = n, a.c = c, a.tokens = tokens, a.ignore = ignore_index, a.error = error;
  a.logprobs = logprobs, a.entropy = entropy, a.stats = stats, a.top_logprobs = top_logprobs, a.top_tokens = top_tokens;
  a.top = top;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MI355X_F32) return lp_fwd<float>(a, workspace, ws_bytes, s);
  if (dtype == MI355X_BF16) return lp_fwd<bf16>(a, workspace, ws_bytes, s);
  return lp_fwd<f16>(a, workspace, ws_bytes, s);
}

extern "C" int mi355x_token_logprobs_bwd(void* dx, int64_t ld_dx, const void* logits, int dtype, int64_t ld,
                                         const float* stats, const float* entropy, const int64_t* tokens,
                                         const int64_t* top_tokens, int top, const float* d_logprobs,
                                         const float* d_entropy, const float* d_top, int64_t n, int64_t c,
                                         int64_t ignore_index, mi355x_stream_t stream) {
  const int rc = lp_check("mi355x_token_logprobs_bwd", n, c, ld, top, dtype);
  if (rc || n == 0) return rc;
  MI_REQUIRE(dx && logits && stats && (!d_logprobs || tokens) && (!d_entropy || entropy) && (!d_top || !top || top_tokens),
             "mi355x_token_logprobs_bwd: null pointer");
  MI_REQUIRE(ld_dx >= c, "mi355x_token_logprobs_bwd: rows of dx %lld apart", (long long)ld_dx);
  LpBwd a{};
  a.dx = dx, a.x = logits, a.ld_dx = ld_dx, a.ld = ld, a.n = n, a.c = c, a.stats = stats, a.entropy = entropy;
  a.tokens = tokens, a.top_tokens = top_tokens, a.d_logprobs = d_logprobs, a.d_entropy = d_entropy;
  a.d_top = top ? d_top : nullptr, a.top = top, a.ignore = ignore_index;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MI355X_F32) return lp_bwd_launch<float>(a, s);
  if (dtype == MI355X_BF16) return lp_bwd_launch<bf16>(a, s);
  return lp_bwd_launch<f16>(a, s);
}
