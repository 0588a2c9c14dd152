// Filling and reading a paged key/value cache: new keys (rotated on the way)
// and values go to their pages, and rows come back as values.
//
// Every row of new queries, keys and values is read once and written once, so
// both kernels are bound by memory traffic for a prompt and by latency for a
// single token: one launch does q, k and v, 16 bytes of 16-bit values at a
// time.
//
// Rotation, half-split: y[i] = x[i] cos[p][i] - x[i + d/2] sin[p][i] and
// y[i + d/2] = x[i + d/2] cos[p][i + d/2] + x[i] sin[p][i + d/2].
//
// 4 bits: m = f16(min), s = f16((max - min) / 15) over 32 channels, each rounded to
// f32 first, code =
// clamp(rint((x - m) / s), 0, 15).  The rotation and the quotient are those of
// f64: products of two values of at most 24 bits are exact there, so which
// side of a border a value falls on depends neither on the order nor on the
// contraction of the operations.  A group with a NaN or an infinity reads back
// as NaN.
#include <math.h>

#include <type_traits>

#include "paged.h"

namespace mi {

int paged_args(const char* what, const mi355x_paged_cache* c, const int32_t* table, int64_t table_stride,
               int64_t table_width, const int32_t* starts, const int32_t* counts, int64_t batch, int64_t seq,
               int32_t* error, PagedSeqs* s) {
  MI_REQUIRE(c, "%s: null cache", what);
  const bool four = c->bits == 4;
  if (!four && c->dtype != MI355X_F32 && c->dtype != MI355X_BF16 && c->dtype != MI355X_F16)
    return fail(MI355X_EUNSUPPORTED, "%s: pages of dtype %d are not supported (f32/bf16/f16, or 4 bits)", what, c->dtype);
  MI_REQUIRE(four || c->bits == 0, "%s: bits must be 4, or 0 for pages of dtype", what);
  if (c->d <= 0 || c->d > 256 || c->d % (four ? kKvGroup : 8))
    return fail(MI355X_EUNSUPPORTED, "%s: head_dim %lld must be a multiple of %d up to 256", what, (long long)c->d,
                four ? kKvGroup : 8);
  MI_REQUIRE(c->kv_heads > 0 && c->kv_heads < 65536, "%s: bad kv_heads %lld", what, (long long)c->kv_heads);
  MI_REQUIRE(c->num_pages > 0 && c->num_pages < (1ll << 31) && c->page_size > 0 && c->page_size < (1ll << 31),
             "%s: bad page count or size", what);
  MI_REQUIRE(batch >= 0 && batch < 65536 && seq >= 0 && seq < (1ll << 31), "%s: bad batch or sequence length", what);
  MI_REQUIRE(table_width >= 0 && table_width < (1ll << 31), "%s: bad page table", what);
  MI_REQUIRE(c->k && c->v && (!four || (c->k_scales && c->v_scales)), "%s: null pages", what);
  MI_REQUIRE(!batch || !seq || (starts && (table || !table_width)), "%s: null page table or starts", what);
  const int64_t es = four ? 1 : (int64_t)dtype_size(c->dtype);
  for (const int64_t* st : {c->k_phs, c->v_phs})
    for (int i = 0; i < 3; ++i)
      MI_REQUIRE(st[i] >= 0 && st[i] * es % 16 == 0, "%s: rows of pages must be 16 bytes apart or a multiple", what);
  MI_REQUIRE(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0, "%s: pages must be 16-byte aligned", what);
  if (four) {
    for (const int64_t* st : {c->ks_phs, c->vs_phs})
      for (int i = 0; i < 3; ++i) MI_REQUIRE(st[i] >= 0 && st[i] % 2 == 0, "%s: bad strides of the scales", what);
    MI_REQUIRE(((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) % 4 == 0, "%s: scales must be 4-byte aligned", what);
  }
  *s = PagedSeqs{table, table_stride, (uint32_t)table_width, starts, counts, page_div(c->page_size),
                 (int32_t)c->num_pages, table_end(table_width, c->page_size), error};
  return MI355X_OK;
}

namespace {

constexpr int kThreads = 256;

// Eight consecutive values.
template <typename T>
struct alignas(16) Oct {
  T v[8];
};

struct Rows {  // [batch, heads, seq, d] view with unit d stride
  void* p;
  int64_t b, h, t;
};

struct AppendArgs {
  mi355x_paged_cache c;
  PagedSeqs s;
  Rows q, qo, k, v;
  const void *cos, *sin;  // null: no rotation
  int64_t rope_len;
  int heads, kv_heads, seq, d;
  int64_t tokens;      // batch * seq
  uint32_t per_token;  // threads of a token: (heads + 2 kv_heads) * d / 8
};

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& r, int64_t b, int64_t h, int64_t t) {
  return (const T*)r.p + b * r.b + h * r.h + t * r.t;
}

// Channels ch .. ch + 7 of the row at x turned by the angles of position pos,
// in the type W that the products are taken in.
template <typename W, typename T, typename RT>
__device__ __forceinline__ void rotate(W (&y)[8], const T* x, const RT* cos_t, const RT* sin_t, int64_t pos, int ch,
                                       int d) {
  const int half = d / 2;
  const bool low = ch < half;
  const Oct<T> a = *(const Oct<T>*)(x + ch), b = *(const Oct<T>*)(x + (low ? ch + half : ch - half));
  const Oct<RT> c = *(const Oct<RT>*)(cos_t + pos * d + ch), s = *(const Oct<RT>*)(sin_t + pos * d + ch);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const W t = (W)to_f32(b.v[e]) * (W)to_f32(s.v[e]);
    y[e] = (W)to_f32(a.v[e]) * (W)to_f32(c.v[e]) + (low ? -t : t);
  }
}

// f16 of an f64 value by way of f32, as the cache's format has it (and a host
// without a conversion in one step).  The compiler would make it one rounding,
// which differs where the f32 value is halfway between two f16 ones: in one of
// 15000 scales.
__device__ __forceinline__ f16 to_f16_by_f32(double x) {
  float f = (float)x;
  asm("" : "+v"(f));
  return (f16)f;
}

// Packs the eight channels of this lane; four neighbouring lanes hold the 32
// channels that share a scale.  W is a type that holds the values exactly.
// A code is clamp(rint((x - base) / step), 0, 15) as the quotient in f64 has
// it: an f32 quotient is within 2^-22 of it and settles all lanes but the one
// in 6000 with a value next to a border, (c + 1/2) * step of 16 bits, which
// settles those.  (The 64-bit quotients took 8 us of 42 for the prompts above
// paged_append_heads.)
template <typename W>
__device__ __forceinline__ void pack_row(W (&x)[8], uint32_t* codes, f16* scales, int ch, int d) {
  const W limit = (W)kKvLimit;
  W lo = x[0], hi = x[0], nan = (W)0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    nan = fma(x[e], (W)0, nan);  // of an infinity too
    lo = fmin(lo, x[e]), hi = fmax(hi, x[e]);
  }
  int bad = !(nan == (W)0);
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    lo = fmin(lo, __shfl_xor(lo, off, 64));
    hi = fmax(hi, __shfl_xor(hi, off, 64));
    bad |= __shfl_xor(bad, off, 64);
  }
  if (lo < -limit || hi > limit) {  // the codes, too, are those of clamped values
    lo = fmin(fmax(lo, -limit), limit), hi = fmin(fmax(hi, -limit), limit);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmin(fmax(x[e], -limit), limit);
  }
  // times 1 / 15 is within 2^-53 of the quotient, which f32 does not resolve
  const f16 step16 = bad ? (f16)NAN : to_f16_by_f32(((double)hi - (double)lo) * (1.0 / 15.0));
  const f16 base16 = bad ? (f16)NAN : to_f16_by_f32(lo);
  uint32_t w = 0;
  if ((float)step16 > 0.f) {
    const float inv = 1.f / (float)step16;
    const W base = (W)(float)base16;
    float far = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = fminf(fmaxf((float)(x[e] - base) * inv, 0.f), 15.f), c = rintf(q);
      far = fmaxf(far, fabsf(q - c));
      w |= (uint32_t)c << (4 * (e / 2 + 4 * (e % 2)));
    }
    if (far > 0.5f - 1e-5f) {
      const double step = (double)(float)step16;
      w = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double v = (double)x[e] - (double)base;
        const float k = floorf(fminf(fmaxf((float)v * inv, 0.f), 15.f));
        const double border = ((double)k + 0.5) * step;
        const uint32_t c = (uint32_t)k, up = v > border || (v == border && (c & 1));
        w |= min(c + up, 15u) << (4 * (e / 2 + 4 * (e % 2)));
      }
    }
  }
  const int s = ch / kKvGroup, g = ch % kKvGroup / 8;
  codes[g * (d / kKvGroup) + s] = w;
  if (g == 0) {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    *(f16x2*)(scales + 2 * s) = f16x2{step16, base16};
  }
}

// The place of token t of sequence b, or false: padding, or out of range.
__device__ __forceinline__ bool place_of(const AppendArgs& a, int64_t b, int64_t pos, int* page, uint32_t* slot) {
  *page = -1;
  if (pos < 0 || pos > kMaxPosition || (a.cos && pos >= a.rope_len)) {
    if (a.s.error) *a.s.error = 1;
  } else {
    *page = page_of(a.s, b, (uint32_t)pos, slot);
  }
  return *page >= 0;
}

// A thread owns channels ch .. ch + 7 and their partners half a row on, of
// kHeads rows of one token and of one kind (query, key or value, the same for
// a block): the angles are read once for all of them, and their loads are all
// in flight before the first is used.  Four prompts of 2048 tokens, 16 query
// and 8 K/V heads of 128 at most, into 4 bits (89 MB): 35 us (eight rows a
// thread 12 more, one or two up to 5 more), where a copy takes 17.  Waiting bounds
// it: four waves a SIMD (116 registers), twice over, load, pack and store one
// after another, and a wave waits for memory in 61% of its cycles; VALU work
// issues in about a third of them (the f64 rotation is little of it), LDS in 2%, and
// the 76 MB that pass HBM are 2.2 TB/s.  Five of 333 at most into f32 pages (13 MB)
// 6.2 us, one token 3.0, a launch.
constexpr int kHeads = 4;

template <typename T, typename RT, bool FOUR>
__global__ void __launch_bounds__(kThreads) paged_append_heads(AppendArgs a) {
  const int half = a.d / 2;
  const uint32_t lanes = a.d / 16, id = blockIdx.x * kThreads + threadIdx.x, token = id / lanes;
  const int ch = (int)(id - token * lanes) * 8;
  if (token >= (uint32_t)a.tokens) return;
  const uint32_t bi = token / a.seq, t = token - bi * a.seq;
  const int64_t b = bi;
  // blockIdx.y: groups of K heads, then of V heads, then of query heads, so that
  // in 4 bits the blocks that pack do not come last (39 us so, for the prompts
  // above; 38 with the kinds side by side)
  const int nk = (a.kv_heads + kHeads - 1) / kHeads;
  int group = blockIdx.y;
  const bool is_k = group < nk, is_q = group >= 2 * nk;
  if (!is_k) group -= is_q ? 2 * nk : nk;
  const int h0 = group * kHeads, n = min(kHeads, (is_q ? a.heads : a.kv_heads) - h0);
  const Rows& src = is_q ? a.q : is_k ? a.k : a.v;
  const T* x = row_of<T>(src, b, h0, t) + ch;
  Oct<T> lo[kHeads], hi[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (i < n) lo[i] = *(const Oct<T>*)(x + i * src.h), hi[i] = *(const Oct<T>*)(x + i * src.h + half);
  const bool real = (int)t < seq_count(a.s, b, a.seq);
  const int64_t pos = (int64_t)a.s.starts[b] + t;
  const bool turns = (is_q || is_k) && a.cos;
  Oct<RT> cl, cv, sl, sv;
  if (turns && real && pos >= 0 && pos < a.rope_len) {
    const RT *c = (const RT*)a.cos + pos * a.d + ch, *s = (const RT*)a.sin + pos * a.d + ch;
    cl = *(const Oct<RT>*)c, cv = *(const Oct<RT>*)(c + half);
    sl = *(const Oct<RT>*)s, sv = *(const Oct<RT>*)(s + half);
  }
  auto turn = [&](auto& y, auto& z, int i) {  // the rotated halves, in y's type
    typedef std::remove_reference_t<decltype(y[0])> W;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const W p = (W)to_f32(lo[i].v[e]), q = (W)to_f32(hi[i].v[e]);
      y[e] = p * (W)to_f32(cl.v[e]) - q * (W)to_f32(sl.v[e]);
      z[e] = q * (W)to_f32(cv.v[e]) + p * (W)to_f32(sv.v[e]);
    }
  };
  auto turn_rows = [&](int i) {  // lo and hi rotated and rounded to the rows' type
    float y[8], z[8];
    turn(y, z, i);
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[i].v[e] = from_f32<T>(y[e]), hi[i].v[e] = from_f32<T>(z[e]);
  };
  if (is_q) {
    const bool ok = real && pos >= 0 && pos < a.rope_len;
    T* o = (T*)a.qo.p + b * a.qo.b + h0 * a.qo.h + t * a.qo.t + ch;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= n) break;
      if (ok) turn_rows(i);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[i].v[e] = hi[i].v[e] = from_f32<T>(0.f);
      *(Oct<T>*)(o + i * a.qo.h) = lo[i], *(Oct<T>*)(o + i * a.qo.h + half) = hi[i];
    }
    return;
  }
  int page;
  uint32_t slot;
  if (!real || !place_of(a, b, pos, &page, &slot)) return;
  const int64_t* st = is_k ? a.c.k_phs : a.c.v_phs;
  const int64_t at = page * st[0] + h0 * st[1] + slot * st[2];
  if constexpr (FOUR) {
    const int64_t* ss = is_k ? a.c.ks_phs : a.c.vs_phs;
    uint8_t* codes = (uint8_t*)(is_k ? a.c.k : a.c.v) + at;
    f16* scales = (f16*)(is_k ? a.c.k_scales : a.c.v_scales) + page * ss[0] + h0 * ss[1] + slot * ss[2];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= n) break;
      uint32_t* c = (uint32_t*)(codes + i * st[1]);
      if (turns) {
        double y[8], z[8];
        turn(y, z, i);
        pack_row(y, c, scales + i * ss[1], ch, a.d);
        pack_row(z, c, scales + i * ss[1], ch + half, a.d);
      } else {
        float y[8], z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = to_f32(lo[i].v[e]), z[e] = to_f32(hi[i].v[e]);
        pack_row(y, c, scales + i * ss[1], ch, a.d);
        pack_row(z, c, scales + i * ss[1], ch + half, a.d);
      }
    }
  } else {
    T* o = (T*)(is_k ? a.c.k : a.c.v) + at + ch;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= n) break;
      if (turns) turn_rows(i);
      *(Oct<T>*)(o + i * st[1]) = lo[i], *(Oct<T>*)(o + i * st[1] + half) = hi[i];
    }
  }
}

// Rows whose halves are no whole pieces of eight channels, or in 4 bits of 32
// (head_dim 24, or 96 in 4 bits): a thread owns eight channels of one row, and
// reads their partners for the rotation again.  A block's threads are 256
// consecutive (token, row, eight channels) of one sequence; the rows of a
// token are its query heads, then K, then V.
template <typename T, typename RT, bool FOUR>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendArgs a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t t = id / a.per_token;
  if (t >= (uint32_t)a.seq) return;
  const int64_t b = blockIdx.y;
  const uint32_t octs = a.d / 8, r = (id - t * a.per_token) / octs;
  const int ch = (int)(id - t * a.per_token - r * octs) * 8;
  const bool real = (int)t < seq_count(a.s, b, a.seq);
  const int64_t pos = (int64_t)a.s.starts[b] + t;
  const int h = (int)r - a.heads;  // >= 0: a K head, and from kv_heads on a V head
  if (h < 0) {
    Oct<T> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.v[e] = from_f32<T>(0.f);
    if (real && pos >= 0 && pos < a.rope_len) {
      float y[8];
      rotate(y, row_of<T>(a.q, b, r, t), (const RT*)a.cos, (const RT*)a.sin, pos, ch, a.d);
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = from_f32<T>(y[e]);
    }
    *(Oct<T>*)((T*)a.qo.p + b * a.qo.b + r * a.qo.h + t * a.qo.t + ch) = o;
    return;
  }
  const bool is_k = h < a.kv_heads;
  const int64_t hk = is_k ? h : h - a.kv_heads;
  int page;
  uint32_t slot;
  if (!real || !place_of(a, b, pos, &page, &slot)) return;  // the same for all lanes of a group
  const int64_t* st = is_k ? a.c.k_phs : a.c.v_phs;
  const int64_t at = page * st[0] + hk * st[1] + slot * st[2];
  const T* x = row_of<T>(is_k ? a.k : a.v, b, hk, t);
  if constexpr (FOUR) {
    const int64_t* ss = is_k ? a.c.ks_phs : a.c.vs_phs;
    uint32_t* codes = (uint32_t*)((uint8_t*)(is_k ? a.c.k : a.c.v) + at);
    f16* scales = (f16*)(is_k ? a.c.k_scales : a.c.v_scales) + page * ss[0] + hk * ss[1] + slot * ss[2];
    if (is_k && a.cos) {
      double y[8];
      rotate(y, x, (const RT*)a.cos, (const RT*)a.sin, pos, ch, a.d);
      pack_row(y, codes, scales, ch, a.d);
    } else {
      const Oct<T> o = *(const Oct<T>*)(x + ch);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = to_f32(o.v[e]);
      pack_row(y, codes, scales, ch, a.d);
    }
  } else {
    Oct<T> o;
    if (is_k && a.cos) {
      float y[8];
      rotate(y, x, (const RT*)a.cos, (const RT*)a.sin, pos, ch, a.d);
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = from_f32<T>(y[e]);
    } else {
      o = *(const Oct<T>*)(x + ch);
    }
    *(Oct<T>*)((T*)(is_k ? a.c.k : a.c.v) + at + ch) = o;
  }
}

struct GatherArgs {
  mi355x_paged_cache c;
  PagedSeqs s;
  Rows k, v;
  int kv_heads, seq, d;
  uint32_t per_token;  // 2 kv_heads * d / 8
};

// Eight channels a thread.  Padding is written as well, zeros: the rows of the
// prompts above from 4 bits to f32, 67 MB written and 13 read, in 17.5 us, 4.6
// TB/s, as a copy.  Full rows of 4 sequences of 2048, 8 heads of 128: f32 24 us, 5.6
// TB/s; bf16 15 us, 4.6; 4 bits to f32 20 us, 3.8, to 16 bits 17 us, 2.5, where
// unpacking is as long.
// T: the type of the values written; CT: of the pages (uint8_t: 4 bits).
template <typename T, typename CT>
__global__ void __launch_bounds__(kThreads) paged_gather_kernel(GatherArgs a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t t = id / a.per_token;
  if (t >= (uint32_t)a.seq) return;
  const int64_t b = blockIdx.y;
  const uint32_t octs = a.d / 8, r = (id - t * a.per_token) / octs;
  const uint32_t oct = id - t * a.per_token - r * octs;
  const bool is_k = r < (uint32_t)a.kv_heads;
  const int64_t hk = is_k ? r : r - a.kv_heads;
  const int64_t pos = (int64_t)a.s.starts[b] + t;
  uint32_t slot = 0;
  int page = -1;
  if ((int)t < seq_count(a.s, b, a.seq)) {
    if (pos < 0 || pos > kMaxPosition) {
      if (a.s.error) *a.s.error = 1;
    } else {
      page = page_of(a.s, b, (uint32_t)pos, &slot);
    }
  }
  Oct<T> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o.v[e] = from_f32<T>(0.f);
  int ch = (int)oct * 8;
  if (page >= 0) {
    const int64_t* st = is_k ? a.c.k_phs : a.c.v_phs;
    const int64_t at = page * st[0] + hk * st[1] + slot * st[2];
    if constexpr (sizeof(CT) == 1) {
      const int n = a.d / kKvGroup, g = (int)oct / n, s = (int)oct % n;
      ch = s * kKvGroup + g * 8;
      const uint32_t w = ((const uint32_t*)((const uint8_t*)(is_k ? a.c.k : a.c.v) + at))[oct];
      const int64_t* ss = is_k ? a.c.ks_phs : a.c.vs_phs;
      const f16* sc = (const f16*)(is_k ? a.c.k_scales : a.c.v_scales) + page * ss[0] + hk * ss[1] + slot * ss[2];
      const float step = (float)sc[2 * s], base = (float)sc[2 * s + 1];
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = from_f32<T>(fmaf(step, (float)(w >> (4 * (e / 2 + 4 * (e % 2))) & 15), base));
    } else {
      const Oct<CT> x = *(const Oct<CT>*)((const CT*)(is_k ? a.c.k : a.c.v) + at + ch);
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = from_f32<T>(to_f32(x.v[e]));
    }
  }
  const Rows& w = is_k ? a.k : a.v;
  *(Oct<T>*)((T*)w.p + b * w.b + hk * w.h + t * w.t + ch) = o;
}

template <typename T, typename RT, bool FOUR>
int append_launch(const AppendArgs& a, hipStream_t s) {
  if (a.d % (FOUR ? 2 * kKvGroup : 16) == 0) {
    const int64_t threads = a.tokens * (a.d / 16);
    MI_REQUIRE(threads < (1ll << 32) - kThreads, "mi355x_paged_append: more than 2^36 values of one head");
    const unsigned groups = ceil_div(a.heads, kHeads) + 2 * ceil_div(a.kv_heads, kHeads);
    paged_append_heads<T, RT, FOUR><<<dim3(ceil_div(threads, kThreads), groups), kThreads, 0, s>>>(a);
  } else {
    const int64_t per_token = a.per_token;
    MI_REQUIRE(per_token * a.seq < (1ll << 32) - kThreads, "mi355x_paged_append: more than 2^35 values of one sequence");
    paged_append_kernel<T, RT, FOUR>
        <<<dim3(ceil_div(per_token * a.seq, kThreads), (unsigned)(a.tokens / a.seq)), kThreads, 0, s>>>(a);
  }
  return check_launch("mi355x_paged_append");
}

template <typename T>
int append_rows(const AppendArgs& a, int rope_dtype, hipStream_t s) {
  const bool f32 = rope_dtype == MI355X_F32;
  if (a.c.bits == 4) return f32 ? append_launch<T, float, true>(a, s) : append_launch<T, T, true>(a, s);
  return f32 ? append_launch<T, float, false>(a, s) : append_launch<T, T, false>(a, s);
}

template <typename T>
int gather_launch(const GatherArgs& a, dim3 grid, hipStream_t s) {
  if (a.c.bits == 4) paged_gather_kernel<T, uint8_t><<<grid, kThreads, 0, s>>>(a);
  else if (a.c.dtype == MI355X_F32) paged_gather_kernel<T, float><<<grid, kThreads, 0, s>>>(a);
  else if (a.c.dtype == MI355X_BF16) paged_gather_kernel<T, bf16><<<grid, kThreads, 0, s>>>(a);
  else paged_gather_kernel<T, f16><<<grid, kThreads, 0, s>>>(a);
  return check_launch("mi355x_paged_gather");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi355x_paged_append(const mi355x_paged_cache* cache, const int32_t* table, int64_t table_stride,
                                   int64_t table_width, const int32_t* starts, const int32_t* counts, const void* k,
                                   const int64_t* k_bht, const void* v, const int64_t* v_bht, void* q_out,
                                   const int64_t* qo_bht, const void* q, const int64_t* q_bht, const void* cos_table,
                                   const void* sin_table, int rope_dtype, int64_t rope_len, int64_t batch,
                                   int64_t heads, int64_t seq, int dtype, int32_t* error, mi355x_stream_t stream) {
  PagedSeqs s;
  int rc = paged_args("mi355x_paged_append", cache, table, table_stride, table_width, starts, counts, batch, seq,
                      error, &s);
  if (rc) return rc;
  if (dtype != MI355X_F32 && dtype != MI355X_BF16 && dtype != MI355X_F16)
    return fail(MI355X_EUNSUPPORTED, "mi355x_paged_append: dtype %d is not supported (f32/bf16/f16)", dtype);
  MI_REQUIRE(cache->bits == 4 || cache->dtype == dtype, "mi355x_paged_append: rows of dtype %d into pages of dtype %d",
             dtype, cache->dtype);
  MI_REQUIRE(!cos_table == !sin_table, "mi355x_paged_append: cos and sin come together");
  MI_REQUIRE(!cos_table || (cache->d % 16 == 0 && rope_len >= 0),
             "mi355x_paged_append: the rotation needs a head_dim that is a multiple of 16");
  MI_REQUIRE(!cos_table || rope_dtype == MI355X_F32 || rope_dtype == dtype,
             "mi355x_paged_append: cos and sin must be f32 or of the rows' dtype");
  MI_REQUIRE(!q == !q_out && (!q || cos_table), "mi355x_paged_append: queries are taken with an output and a rotation");
  MI_REQUIRE(heads >= 0 && heads < 65536 && (q || heads == 0), "mi355x_paged_append: bad heads %lld", (long long)heads);
  if (batch == 0 || seq == 0) return MI355X_OK;
  const size_t es = dtype_size(dtype);
  MI_REQUIRE(k && v, "mi355x_paged_append: null pointer");
  MI_REQUIRE(rows_ok(k, k_bht, es) && rows_ok(v, v_bht, es) && (!q || (rows_ok(q, q_bht, es) && rows_ok(q_out, qo_bht, es))),
             "mi355x_paged_append: rows must be 16-byte aligned");
  MI_REQUIRE(((uintptr_t)cos_table | (uintptr_t)sin_table) % 16 == 0, "mi355x_paged_append: cos and sin must be 16-byte aligned");
  AppendArgs a{};
  a.c = *cache, a.s = s;
  a.k = Rows{(void*)k, k_bht[0], k_bht[1], k_bht[2]}, a.v = Rows{(void*)v, v_bht[0], v_bht[1], v_bht[2]};
  if (q) a.q = Rows{(void*)q, q_bht[0], q_bht[1], q_bht[2]}, a.qo = Rows{q_out, qo_bht[0], qo_bht[1], qo_bht[2]};
  a.cos = cos_table, a.sin = sin_table, a.rope_len = rope_len;
  a.heads = (int)heads, a.kv_heads = (int)cache->kv_heads, a.seq = (int)seq, a.d = (int)cache->d;
  MI_REQUIRE(batch * seq < (1ll << 31), "mi355x_paged_append: batch x tokens must be below 2^31");
  a.tokens = batch * seq;
  a.per_token = (uint32_t)((heads + 2 * cache->kv_heads) * (cache->d / 8));
  const int rdt = cos_table ? rope_dtype : MI355X_F32;
  if (dtype == MI355X_F32) return append_rows<float>(a, rdt, (hipStream_t)stream);
  if (dtype == MI355X_BF16) return append_rows<bf16>(a, rdt, (hipStream_t)stream);
  return append_rows<f16>(a, rdt, (hipStream_t)stream);
}

extern "C" int mi355x_paged_gather(void* k, const int64_t* k_bht, void* v, const int64_t* v_bht,
                                   const mi355x_paged_cache* cache, const int32_t* table, int64_t table_stride,
                                   int64_t table_width, const int32_t* starts, const int32_t* counts, int64_t batch,
                                   int64_t seq, int dtype, int32_t* error, mi355x_stream_t stream) {
  PagedSeqs s;
  int rc = paged_args("mi355x_paged_gather", cache, table, table_stride, table_width, starts, counts, batch, seq,
                      error, &s);
  if (rc) return rc;
  if (dtype != MI355X_F32 && dtype != MI355X_BF16 && dtype != MI355X_F16)
    return fail(MI355X_EUNSUPPORTED, "mi355x_paged_gather: dtype %d is not supported (f32/bf16/f16)", dtype);
  if (batch == 0 || seq == 0) return MI355X_OK;
  MI_REQUIRE(k && v, "mi355x_paged_gather: null pointer");
  const size_t es = dtype_size(dtype);
  MI_REQUIRE(rows_ok(k, k_bht, es) && rows_ok(v, v_bht, es), "mi355x_paged_gather: rows must be 16-byte aligned");
  GatherArgs a{};
  a.c = *cache, a.s = s;
  a.k = Rows{k, k_bht[0], k_bht[1], k_bht[2]}, a.v = Rows{v, v_bht[0], v_bht[1], v_bht[2]};
  a.kv_heads = (int)cache->kv_heads, a.seq = (int)seq, a.d = (int)cache->d;
  const int64_t per_token = 2 * cache->kv_heads * (cache->d / 8);
  MI_REQUIRE(per_token * seq < (1ll << 32) - kThreads, "mi355x_paged_gather: more than 2^35 values of one sequence");
  a.per_token = (uint32_t)per_token;
  const dim3 grid(ceil_div(per_token * seq, kThreads), (unsigned)batch);
  if (dtype == MI355X_F32) return gather_launch<float>(a, grid, (hipStream_t)stream);
  if (dtype == MI355X_BF16) return gather_launch<bf16>(a, grid, (hipStream_t)stream);
  return gather_launch<f16>(a, grid, (hipStream_t)stream);
}
