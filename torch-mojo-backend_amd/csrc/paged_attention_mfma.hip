// Attention over a paged cache on matrix cores: f32, bf16 and f16 pages, and
// 4-bit pages, at head_dim 64, 128 and 256.
//
// A new token reads every visible row of K and V once and does 4 operations a
// value and query head with it: memory bounds it, and all that matters is that
// enough loads are in flight and that nothing else takes longer than they do.
//
// A wave owns 16 query rows at a time (QT times) of one K/V head: the heads of
// its group, token by token, so the keys that they share are read once.  It
// walks tiles of 32 keys (16 in f32), four waves of a block taking turns, and
// keeps its own running maximum, sum and output; nothing waits for another
// wave before the end.  The rows go straight to registers:
//   S^T = K Q^T: K's operand (a key's channels 8 g .. 8 g + 7 of every 32 in
//     lane group g) is how a row lies in memory;
//   O^T += V^T P^T: V's operand has eight keys of one channel in a lane.  Each
//     lane loads eight channels of its eight keys and exchanges halves of
//     words in registers (v_perm_b32, half an instruction a value); its O^T
//     tiles then hold every eighth channel.  No LDS, no transposing loads.
// The accumulator layout of S^T (keys 4 g .. 4 g + 3 of a query in lane group
// g) is the operand layout of P^T, for tiles in the order of the keys.
//
// P is split in two halves of the pages' type, so its rounding (2^-8 in bf16)
// does not show beside the result's; for a few new tokens the second product
// costs nothing (for a prompt it is a third of the MFMAs).  Exponentials are the
// hardware's, within a step of f32: f32 results are 3.1e-7 off in the 2-norm where
// the plain form's are 2.1e-7.
//
// 4-bit rows are turned into f16 in registers: masked nibbles under f16's
// exponent of 512, less 512, are half the codes, two a register.  For bf16
// queries a value is minimum + 2 * scale * (code / 2) in one rounding and P one
// f16 value: 2^-11 each, an eighth of the result's own step.  For f16 queries
// these would be as large as that, so nothing is rounded: the scale is taken as
// a sum of two numbers of 7 and 4 bits, whose products with a code fit f16, the
// minimums have a product of their own (they are the same for the 8 channels
// of a word), and P is split.  Queries go to f16 with their row's exponent
// taken out, which keeps bf16's values as they are.
//
// Blocks split the keys of long sequences; paged_attn_join adds the parts.
//
// 32 sequences of up to 16384 keys, 32 query heads over 8 of 128: 275 us in
// bf16, 5.7 TB/s (a pass that only reads reaches 6.3 here).  In 4 bits 139 us, 3.5
// TB/s: turning the codes takes 57% of the issue slots and the waits on the
// lookups and loads of a tile most of the rest (164 us with f16 queries).  One
// token over 516 keys of 4 heads over 1 of 256, bf16: 9.9 us, of which a tile of
// 32 keys is 2; over 8191 in 4 bits 9.7.  A prompt runs here too, 16 or 32 rows a
// block, which read each K and V row again: [1, 32 over 8, 2048, 128] bf16 137 us
// where attention over rows laid out densely takes 88, [1, 4 over 1, 2048, 256] 212
// and 70; over 4 bits 143 and 137 (f16 queries 188 and 253).
#include <math.h>

#include <type_traits>

#include "mfma.h"
#include "paged_attention.h"

namespace mi {
namespace {

constexpr int NW = 4;  // waves of a block

typedef f16 f16x2 __attribute__((ext_vector_type(2)));

// Over the four lane groups: v_permlane{16,32}_swap of a value with itself
// leaves the lane 16 (32) further on in the second result.
__device__ __forceinline__ float group_max(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float group_sum(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Where the rows of a tile are: lane l looked up key l % TK of it.
struct Places {
  int page, slot;
  uint32_t live;  // keys that some row may see and whose page exists
};

// Rows of a cache, for one K/V head.  row(tensor, ...) is byte `at` of the row
// of key 16 kt + k of the tile in k, v, ks or vs; what is not live lies in
// page 0.  Rows close together (P16): 16 keys share a page, K and V are laid
// out alike and scales like their rows a quarter as far apart, so that the 16
// keys have one offset, the same for all lanes and, shifted, for all tensors,
// and the lane's own part of an address is 32 bits that no tile changes.
enum Tensor { kKeys, kValues, kKeyScales, kValueScales };
template <bool P16>
struct CacheRows {
  const char* base[4];
  int64_t page_bytes[4], slot_bytes[4];
  __device__ __forceinline__ CacheRows(const mi355x_paged_cache& c, int es, int64_t hk) {
    const void* p[4] = {c.k, c.v, c.k_scales, c.v_scales};
    const int64_t* st[4] = {c.k_phs, c.v_phs, c.ks_phs, c.vs_phs};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int n = t < 2 ? es : 2;
      base[t] = (const char*)p[t] + hk * st[t][1] * n, page_bytes[t] = st[t][0] * n, slot_bytes[t] = st[t][2] * n;
    }
  }
  __device__ __forceinline__ const char* row(int t, const Places& p, int kt, int k, int at) const {
    if constexpr (P16) {
      const uint32_t page = __builtin_amdgcn_readlane(p.page, 16 * kt), slot = __builtin_amdgcn_readlane(p.slot, 16 * kt);
      const uint64_t off = (uint64_t)page * (uint32_t)page_bytes[0] + slot * (uint32_t)slot_bytes[0];
      return base[t] + (t < 2 ? off : off >> 2) + (uint32_t)((t < 2 ? k * (int)slot_bytes[0] : k * (int)slot_bytes[0] / 4) + at);
    } else {
      const int64_t page = __shfl(p.page, 16 * kt + k, 64), slot = __shfl(p.slot, 16 * kt + k, 64);
      return base[t] + page * page_bytes[t] + slot * slot_bytes[t] + at;
    }
  }
};
bool rows_close(const mi355x_paged_cache& c, int64_t es) {
  const int64_t page = c.k_phs[0] * es, slot = c.k_phs[2] * es;
  bool ok = c.page_size % 16 == 0 && page < (1ll << 32) && slot * (c.page_size + 16) < (1ll << 31) &&
            c.v_phs[0] == c.k_phs[0] && c.v_phs[2] == c.k_phs[2];
  if (c.bits == 4)
    for (const int64_t* st : {c.ks_phs, c.vs_phs}) ok &= st[0] * 8 == page && st[2] * 8 == slot;
  return ok;
}

// ---------------------------------------------------------------------------
// page formats
// ---------------------------------------------------------------------------
// What a format adds up beside o: nothing.
struct NoRest {
  template <int N>
  __device__ __forceinline__ void scale(float (&)[N]) {}
  template <typename O>
  __device__ __forceinline__ void finish(O&) {}
};

// 16-bit pages of T.
template <typename T, int D_>
struct Pages16 {
  static constexpr int D = D_, KT = 2, VW = D >= 128 ? 8 : 4, NU = D / (16 * VW), kBytes = 2, kMore = 64;
  typedef typename Mfma<T>::frag frag;
  typedef uint32_t vword __attribute__((ext_vector_type(VW / 2)));
  template <int QT>
  using Rest = NoRest;
  struct Keys {
    frag k[KT][D / 32];
  };
  struct Values {
    vword v[8][NU];
  };
  struct Query {
    frag q[D / 32];
    float scale;
  };
  static __device__ __forceinline__ int channel(int u, int e, int c) { return (u * 16 + c) * VW + e; }
  template <typename QT_>
  static __device__ __forceinline__ void load_query(Query& q, const QT_* row, bool real, int g, float scale_log2) {
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) q.q[s][e] = (T)0.f;
    if (real)
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        q.q[s] = *(const frag*)(row + s * 32 + g * 8);
        if (scale_log2 < 0.f)
#pragma unroll
          for (int e = 0; e < 8; ++e) q.q[s][e] = -q.q[s][e];
      }
    q.scale = fabsf(scale_log2);
  }
  template <bool P16>
  static __device__ __forceinline__ void load_keys(Keys& r, const CacheRows<P16>& c, const Places& p, int lr, int g) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const T* row = (const T*)c.row(kKeys, p, kt, lr, g * 16);
#pragma unroll
      for (int s = 0; s < D / 32; ++s) r.k[kt][s] = *(const frag*)(row + s * 32);
    }
  }
  template <bool P16>
  static __device__ __forceinline__ void load_values(Values& r, const CacheRows<P16>& c, const Places& p, int lr, int g) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T* row = (const T*)c.row(kValues, p, i >> 2, 4 * g + (i & 3), lr * VW * 2);
#pragma unroll
      for (int u = 0; u < NU; ++u) r.v[i][u] = *(const vword*)(row + u * 16 * VW);
    }
  }
  static __device__ __forceinline__ void hide_values(Values& r, uint32_t live, int g) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(live >> (16 * (i >> 2) + 4 * g + (i & 3)) & 1))
#pragma unroll
        for (int u = 0; u < NU; ++u) r.v[i][u] = vword(0);
  }
  template <int QT>
  static __device__ __forceinline__ void scores(f32x4 (&s)[KT][QT], const Keys& r, const Query (&q)[QT]) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) x = Mfma<T>::mma(r.k[kt][ks], q[qt].q[ks], x);
        s[kt][qt] = x;
      }
  }
  template <int QT>
  static __device__ __forceinline__ void add_values(f32x4 (&o)[NU][VW][QT], NoRest&, const Values& r, const f32x4 (&p)[KT][QT]) {
    frag hi[QT], lo[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const T h = (T)p[kt][qt][e];
          hi[qt][4 * kt + e] = h;
          lo[qt][4 * kt + e] = (T)(p[kt][qt][e] - (float)h);
        }
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        union {
          uint32_t w[4];
          frag f;
        } v;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v.w[i] = __builtin_amdgcn_perm(r.v[2 * i + 1][u][e / 2], r.v[2 * i][u][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          o[u][e][qt] = Mfma<T>::mma(v.f, hi[qt], o[u][e][qt]);
          o[u][e][qt] = Mfma<T>::mma(v.f, lo[qt], o[u][e][qt]);
        }
      }
  }
};

// f32 pages: v_mfma_f32_16x16x4_f32, one key (or channel) a lane group; with
// the keys of a product step taken as 4 g + step, V's rows need no exchange.
template <int D_>
struct Pages32 {
  static constexpr int D = D_, KT = 1, VW = 4, NU = D / 64, kBytes = 4, kMore = 64;
  template <int QT>
  using Rest = NoRest;
  struct Keys {
    f32x4 k[D / 16];
  };
  struct Values {
    f32x4 v[4][NU];
  };
  struct Query {
    f32x4 q[D / 16];
    float scale;
  };
  static __device__ __forceinline__ int channel(int u, int e, int c) { return u * 64 + c * 4 + e; }
  static __device__ __forceinline__ void load_query(Query& q, const float* row, bool real, int g, float scale_log2) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s) q.q[s] = real ? *(const f32x4*)(row + s * 16 + g * 4) : f32x4{0.f, 0.f, 0.f, 0.f};
    if (scale_log2 < 0.f)
#pragma unroll
      for (int s = 0; s < D / 16; ++s) q.q[s] = -q.q[s];
    q.scale = fabsf(scale_log2);
  }
  template <bool P16>
  static __device__ __forceinline__ void load_keys(Keys& r, const CacheRows<P16>& c, const Places& p, int lr, int g) {
    const float* k = (const float*)c.row(kKeys, p, 0, lr, g * 16);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) r.k[s] = *(const f32x4*)(k + s * 16);
  }
  template <bool P16>
  static __device__ __forceinline__ void load_values(Values& r, const CacheRows<P16>& c, const Places& p, int lr, int g) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* v = (const float*)c.row(kValues, p, 0, 4 * g + i, lr * 16);
#pragma unroll
      for (int u = 0; u < NU; ++u) r.v[i][u] = *(const f32x4*)(v + u * 64);
    }
  }
  static __device__ __forceinline__ void hide_values(Values& r, uint32_t live, int g) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(live >> (4 * g + i) & 1))
#pragma unroll
        for (int u = 0; u < NU; ++u) r.v[i][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  template <int QT>
  static __device__ __forceinline__ void scores(f32x4 (&s)[KT][QT], const Keys& r, const Query (&q)[QT]) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) x = __builtin_amdgcn_mfma_f32_16x16x4f32(r.k[ks][e], q[qt].q[ks][e], x, 0, 0, 0);
      s[0][qt] = x;
    }
  }
  template <int QT>
  static __device__ __forceinline__ void add_values(f32x4 (&o)[NU][VW][QT], NoRest&, const Values& r, const f32x4 (&p)[KT][QT]) {
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < VW; ++e)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[u][e][qt] = __builtin_amdgcn_mfma_f32_16x16x4f32(r.v[i][u][e], p[0][qt][i], o[u][e][qt], 0, 0, 0);
  }
};

// 4-bit pages, queries of T.
template <typename T, int D_>
struct Pages4 {
  static constexpr int D = D_, KT = 2, VW = D >= 128 ? 8 : 4, NU = D / (16 * VW), NG = D / kKvGroup, kBytes = 1;
  static constexpr bool EXACT = std::is_same_v<T, f16>;
  static constexpr int kMore = EXACT ? 96 : 64;
  typedef f16x8 frag;
  typedef uint32_t row_words __attribute__((ext_vector_type(NG)));  // a lane's codes of a K row, or the row's scales
  struct Keys {
    row_words k[KT], ks[KT];
  };
  struct Values {
    uint32_t v[8][NU], vs[8][NU];
  };
  // The minimums' share of O, by word; o has that of half the codes.
  template <int QT>
  struct Minimums {
    f32x4 m[NU][QT] = {};
    __device__ __forceinline__ void scale(float (&alpha)[QT]) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) m[u][qt] *= alpha[qt];
    }
    __device__ __forceinline__ void finish(f32x4 (&o)[NU][VW][QT]) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < VW; ++e)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) o[u][e][qt] = 2.f * o[u][e][qt] + m[u][qt];
    }
  };
  template <int QT>
  using Rest = std::conditional_t<EXACT, Minimums<QT>, NoRest>;
  struct Query {
    frag q[D / 32];
    float scale;
  };
  // V's lane c holds word c + 16 u of a row; at head_dim 64 two lanes share a
  // word, c < 8 its even channels and c >= 8 its odd ones.
  static __device__ __forceinline__ int word(int u, int c) { return D >= 128 ? c + 16 * u : c & 7; }
  static __device__ __forceinline__ int channel(int u, int e, int c) {
    const int w = word(u, c);
    return w % NG * kKvGroup + w / NG * 8 + (D >= 128 ? e : 2 * e + (c >> 3));
  }
  static __device__ __forceinline__ void load_query(Query& q, const T* row, bool real, int g, float scale_log2) {
    float x[D / 32][8], top = 0.f;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      typename Mfma<T>::frag v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)0.f;
      if (real) v = *(const typename Mfma<T>::frag*)(row + s * 32 + g * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[s][e] = (float)v[e], top = fmaxf(top, fabsf(x[s][e]));
    }
    top = group_max(top);
    const int ex = top > 0.f && top < INFINITY ? ilogbf(top) : 0;
    const float sign = scale_log2 < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) q.q[s][e] = (f16)ldexpf(sign * x[s][e], -ex);
    q.scale = ldexpf(fabsf(scale_log2), ex);
  }
  template <bool P16>
  static __device__ __forceinline__ void load_keys(Keys& r, const CacheRows<P16>& c, const Places& p, int lr, int g) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      r.k[kt] = *(const row_words*)c.row(kKeys, p, kt, lr, g * (D / 8));
      r.ks[kt] = *(const row_words*)c.row(kKeyScales, p, kt, lr, 0);
    }
  }
  template <bool P16>
  static __device__ __forceinline__ void load_values(Values& r, const CacheRows<P16>& c, const Places& p, int lr, int g) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        r.v[i][u] = *(const uint32_t*)c.row(kValues, p, i >> 2, 4 * g + (i & 3), word(u, lr) * 4);
        r.vs[i][u] = *(const uint32_t*)c.row(kValueScales, p, i >> 2, 4 * g + (i & 3), word(u, lr) % NG * 4);
      }
    }
  }
  static __device__ __forceinline__ void hide_values(Values& r, uint32_t live, int g) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(live >> (16 * (i >> 2) + 4 * g + (i & 3)) & 1))
#pragma unroll
        for (int u = 0; u < NU; ++u) r.vs[i][u] = 0;
  }
  // Half the codes of nibble i of both halves of w.  `mask` is 0x000f000f in a
  // vector register: an instruction takes one constant from elsewhere, and two
  // make it an AND and an OR.
  static __device__ __forceinline__ f16x2 half_codes(uint32_t w, int i, uint32_t mask) {
    return __builtin_bit_cast(f16x2, (w >> (4 * i) & mask) | 0x60006000u) - (f16)512.f;
  }
  // s as a number of 7 bits, whose product with half a code is exact, and the rest
  static __device__ __forceinline__ f16x2 upper(f16x2 s) {
    return __builtin_bit_cast(f16x2, __builtin_bit_cast(uint32_t, s) & 0xfff0fff0u);
  }
  static __device__ __forceinline__ uint32_t nibbles() {
    uint32_t mask;
    asm("v_mov_b32 %0, 0x000f000f" : "=v"(mask));
    return mask;
  }
  template <int QT>
  static __device__ __forceinline__ void scores(f32x4 (&s)[KT][QT], const Keys& r, const Query (&q)[QT]) {
    const uint32_t mask = nibbles();
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      f32x4 low[QT];  // EXACT: the minimums' share
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) s[kt][qt] = low[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NG; ++ks) {
        const f16x2 sm = __builtin_bit_cast(f16x2, (uint32_t)r.ks[kt][ks]);
        const f16x2 sc = f16x2{sm[0], sm[0]}, mn = f16x2{sm[1], sm[1]};
        union {
          f16x2 h[4];
          frag f;
        } k, rest, m;
        if constexpr (EXACT) {
          const f16x2 up = upper(sc), down = sc - up;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f16x2 c = half_codes(r.k[kt][ks], i, mask);
            k.h[i] = c * up, rest.h[i] = c * down, m.h[i] = mn;
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            s[kt][qt] = Mfma<f16>::mma(k.f, q[qt].q[ks], s[kt][qt]);
            s[kt][qt] = Mfma<f16>::mma(rest.f, q[qt].q[ks], s[kt][qt]);
            low[qt] = Mfma<f16>::mma(m.f, q[qt].q[ks], low[qt]);
          }
        } else {
          const f16x2 sc2 = sc + sc;
#pragma unroll
          for (int i = 0; i < 4; ++i) k.h[i] = __builtin_elementwise_fma(half_codes(r.k[kt][ks], i, mask), sc2, mn);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) s[kt][qt] = Mfma<f16>::mma(k.f, q[qt].q[ks], s[kt][qt]);
        }
      }
      if constexpr (EXACT)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[kt][qt] = 2.f * s[kt][qt] + low[qt];
    }
  }
  template <int QT>
  static __device__ __forceinline__ void add_values(f32x4 (&o)[NU][VW][QT], Rest<QT>& rest, const Values& r, const f32x4 (&p)[KT][QT]) {
    frag hi[QT], lo[QT];  // lo: EXACT alone
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f16 h = (f16)p[kt][qt][e];
          hi[qt][4 * kt + e] = h;
          if (EXACT) lo[qt][4 * kt + e] = (f16)(p[kt][qt][e] - (float)h);
        }
    const uint32_t mask = nibbles();
    const bool odd = D < 128 && (threadIdx.x & 8);
    auto add = [&](f32x4& x, frag v, int qt) {
      x = Mfma<f16>::mma(v, hi[qt], x);
      if (EXACT) x = Mfma<f16>::mma(v, lo[qt], x);
    };
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      uint32_t even_w[4], odd_w[4];  // words of two keys: their even, their odd channels
      f16x2 s[4], down[4];
      union {
        f16x2 h[4];
        frag f;
      } m;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = r.v[2 * i][u], b = r.v[2 * i + 1][u], x = r.vs[2 * i][u], y = r.vs[2 * i + 1][u];
        even_w[i] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        odd_w[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        if (odd) even_w[i] = odd_w[i];
        s[i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(y, x, 0x05040100u));
        m.h[i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(y, x, 0x07060302u));
        if constexpr (EXACT) down[i] = s[i] - upper(s[i]), s[i] = upper(s[i]);
        else s[i] = s[i] + s[i];
      }
      if constexpr (EXACT)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) add(rest.m[u][qt], m.f, qt);
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        union {
          f16x2 h[4];
          frag f;
        } v, w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f16x2 c = D >= 128 ? half_codes(e % 2 ? odd_w[i] : even_w[i], e / 2, mask) : half_codes(even_w[i], e, mask);
          if constexpr (EXACT) v.h[i] = c * s[i], w.h[i] = c * down[i];
          else v.h[i] = __builtin_elementwise_fma(c, s[i], m.h[i]);
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          add(o[u][e][qt], v.f, qt);
          if constexpr (EXACT) add(o[u][e][qt], w.f, qt);
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------
// Waves of a SIMD that the registers are shared out to: what keys, values,
// queries and output take, and some more.
template <typename F, int QT>
constexpr int waves_of() {
  const int regs = (int)(sizeof(typename F::Keys) + sizeof(typename F::Values)) / 4 +
                   QT * ((int)sizeof(typename F::Query) / 4 + F::D / 4) + F::kMore;
  return regs <= 128 ? 4 : regs <= 168 ? 3 : regs <= 256 ? 2 : 1;
}

template <typename F, typename T, int QT, bool P16>
__global__ void __launch_bounds__(64 * NW, (waves_of<F, QT>())) paged_attn_mfma(DecodeArgs a) {
  constexpr int D = F::D, KT = F::KT, TK = 16 * KT, VW = F::VW, NU = F::NU, W = 16 * VW;
  __shared__ float so[NW][16][W + 4];
  __shared__ float sm[NW][16 * QT], sl[NW][16 * QT];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int lr = lane & 15, g = lane >> 4;
  // The row groups of a part of a head's keys run on one XCD, whose L2 they share.
  const uint32_t i0 = blockIdx.x >> 3;
  const uint32_t unit = i0 / a.row_groups * 8 + (blockIdx.x & 7), rg = i0 % a.row_groups;
  if (unit >= (uint32_t)a.units) return;
  const uint32_t hkn = (uint32_t)a.c.kv_heads;
  const int split = unit % a.splits;
  const int64_t hk = unit / a.splits % hkn, b = unit / a.splits / hkn;
  const int rows = a.group * a.seq, r0 = (int)rg * 16 * QT;
  const int count = seq_count(a.s, b, a.seq);
  const int64_t start = a.s.starts[b];

  typename F::Query q[QT];
  int pos[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = r0 + qt * 16 + lr, t = r / a.group, h = (int)hk * a.group + r - t * a.group;
    const int64_t at = start + t;
    const bool real = r < rows && t < count;
    const bool ok = real && at >= 0 && at <= kMaxPosition;
    if (real && (!ok || at >= a.s.end) && a.s.error) *a.s.error = 1;
    pos[qt] = ok ? (int)at : -1;
    F::load_query(q[qt], (const T*)a.q + b * a.q_b + h * a.q_h + t * a.q_t, ok, g, a.scale_log2);
  }
  // positions of the block's first and last row (rows are token by token)
  const int t0 = r0 / a.group, t1 = min(min((r0 + 16 * QT - 1) / a.group, count - 1), a.seq - 1);
  const int64_t last64 = t1 >= t0 ? start + t1 : -1, first64 = start + t0;
  const int last = (int)min(max(last64, (int64_t)-1), kMaxPosition);
  const int first = (int)min(max(first64, (int64_t)-1), kMaxPosition);
  const KeySpan span(first, last, a.window, a.sinks, a.s.end, TK);
  const int top_key = min(last, a.s.end - 1);  // a position past the table is an error, and sees what the table has
  const int low = a.window > 0 ? max(first - a.window + 1, 0) : 0;
  const int per = (span.tiles + a.splits - 1) / a.splits;
  const int end = min((split + 1) * per, span.tiles);

  auto look_up = [&](int i) {
    Places p{0, 0, 0};
    const int j = span.tile(i) * TK + (lane & (TK - 1));
    bool live = j <= top_key && (j >= low || j < a.sinks);
    // 16 keys of one page: its number is wanted if any of them is live
    const int j16 = j & ~15;
    const bool wanted = P16 ? j16 <= top_key && (j16 + 15 >= low || j16 < a.sinks) : live;
    if (wanted) {
      uint32_t slot;
      const int page = page_of(a.s, b, (uint32_t)j, &slot);
      live = live && page >= 0;
      p.page = max(page, 0), p.slot = page >= 0 ? (int)slot : P16 ? lane & 15 : 0;
    }
    p.live = (uint32_t)__builtin_amdgcn_ballot_w64(live) & (uint32_t)((1ull << TK) - 1);
    return p;
  };
  float m[QT], l[QT];
  f32x4 o[NU][VW][QT];
  typename F::template Rest<QT> rest;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m[qt] = -INFINITY, l[qt] = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < VW; ++e) o[u][e][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Registers hold one tile: its keys make room for the next ones as soon as
  // the scores are taken, its values after their product.  The rest of the
  // time the loads have comes from the other waves of the SIMD, of which
  // there are more than with two tiles in registers.
  typename F::Keys keys;
  typename F::Values values;
  const CacheRows<P16> rows_of(a.c, F::kBytes, hk);
  int i = split * per + wave;
  Places here{0, 0, 0}, next{0, 0, 0};
  if (i < end) {
    here = look_up(i);
    F::template load_keys<P16>(keys, rows_of, here, lr, g);
    F::template load_values<P16>(values, rows_of, here, lr, g);
    if (i + NW < end) next = look_up(i + NW);
  }
  for (; i < end; i += NW) {
    const int j0 = span.tile(i) * TK;
    const uint32_t live = here.live;
    const bool more = i + NW < end;
    // every key of the tile is seen by every row
    const bool whole = live == (uint32_t)((1ull << TK) - 1) && j0 + TK - 1 <= first &&
                       (a.window <= 0 || last - j0 < a.window || j0 + TK <= a.sinks);
    f32x4 s[KT][QT];
    F::scores(s, keys, q);
    if (more) F::template load_keys<P16>(keys, rows_of, next, lr, g);
    // the scale is not negative (its sign went into q), so the maximum can be
    // taken before it
    bool moved = false;
    float top[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!whole) {
            const int k = 16 * kt + 4 * g + e;
            if (!(live >> k & 1) || !visible(pos[qt], j0 + k, a.window, a.sinks)) s[kt][qt][e] = -INFINITY;
          }
          mx = fmaxf(mx, s[kt][qt][e]);
        }
      mx = group_max(mx);
      top[qt] = fmaxf(m[qt], mx == -INFINITY ? mx : mx * q[qt].scale);
      moved |= top[qt] > m[qt];
    }
    if (__builtin_amdgcn_ballot_w64(moved)) {
      float alpha[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        alpha[qt] = top[qt] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[qt] - top[qt]);
        l[qt] *= alpha[qt];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < VW; ++e) o[u][e][qt] *= alpha[qt];
        m[qt] = top[qt];
      }
      rest.scale(alpha);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float base = m[qt] == -INFINITY ? 0.f : m[qt];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = fmaf(s[kt][qt][e], q[qt].scale, -base);
          if (!whole && s[kt][qt][e] == -INFINITY) x = -INFINITY;  // a scale of zero would make it NaN
          const float p = __builtin_amdgcn_exp2f(x);
          s[kt][qt][e] = p;
          l[qt] += p;
        }
    }
    if (!whole) F::hide_values(values, live, g);
    F::add_values(o, rest, values, s);
    if (more) {
      F::template load_values<P16>(values, rows_of, next, lr, g);
      here = next;
      if (i + 2 * NW < end) next = look_up(i + 2 * NW);
    }
  }

  rest.finish(o);

  // join the waves
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] = group_sum(l[qt]);
    if (g == 0) sm[wave][qt * 16 + lr] = m[qt], sl[wave][qt * 16 + lr] = l[qt];
  }
  __syncthreads();
  const int64_t total_rows = a.batch * a.heads * a.seq;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sm[w][qt * 16 + lr]);
    // (rows without a maximum have sums of 0, or of NaN)
    const float mine = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[qt] - mx);
    // the row that this thread stores, and its sum
    const int sr = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int r = r0 + qt * 16 + sr, t = r / a.group, h = (int)hk * a.group + r - t * a.group;
    float smx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) smx = fmaxf(smx, sm[w][qt * 16 + sr]);
#pragma unroll
    for (int w = 0; w < NW; ++w)
      sum += smx == -INFINITY ? sl[w][qt * 16 + sr] : __builtin_amdgcn_exp2f(sm[w][qt * 16 + sr] - smx) * sl[w][qt * 16 + sr];
    // padding took part where tiles were whole: it leaves nothing
    const bool none = t >= count || start + t < 0 || start + t > kMaxPosition;
    if (none) smx = -INFINITY, sum = 0.f;
    const int64_t row = (b * a.heads + h) * a.seq + t;
    if (a.splits > 1 && r < rows && c == 0) a.part_ml[split * total_rows + row] = make_float2(smx, sum);
    const float inv = a.splits > 1 ? 1.f : (sum != 0.f ? 1.f / sum : 0.f);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      __syncthreads();
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4)
#pragma unroll
        for (int e = 0; e < VW; e += 4)
          *(float4*)&so[wave][lr][(4 * g + e4) * VW + e] =
              make_float4(o[u][e][qt][e4] * mine, o[u][e + 1][qt][e4] * mine, o[u][e + 2][qt][e4] * mine, o[u][e + 3][qt][e4] * mine);
      __syncthreads();
      if (r >= rows) continue;
      float x[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) x[e] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int e = 0; e < VW; ++e) x[e] += none ? 0.f : so[w][sr][c * VW + e];
      if (a.splits > 1) {
        float* dst = a.part_o + (split * total_rows + row) * D;
#pragma unroll
        for (int e = 0; e < VW; ++e) dst[F::channel(u, e, c)] = x[e];
      } else {
        T* dst = (T*)a.o + b * a.o_b + h * a.o_h + t * a.o_t;
#pragma unroll
        for (int e = 0; e < VW; ++e) dst[F::channel(u, e, c)] = from_f32<T>(x[e] * inv);
      }
    }
  }
}

template <typename F, typename T, int QT>
void launch(const DecodeArgs& a, unsigned blocks, hipStream_t s) {
  if (rows_close(a.c, F::kBytes)) paged_attn_mfma<F, T, QT, true><<<blocks, 64 * NW, 0, s>>>(a);
  else paged_attn_mfma<F, T, QT, false><<<blocks, 64 * NW, 0, s>>>(a);
}

template <typename F, typename T>
void launch_rows(const DecodeArgs& a, int qt, unsigned blocks, hipStream_t s) {
  if constexpr (F::D < 256)
    if (qt == 2) return launch<F, T, 2>(a, blocks, s);
  launch<F, T, 1>(a, blocks, s);
}

template <int D>
void launch_format(const DecodeArgs& a, int qt, int dtype, unsigned blocks, hipStream_t s) {
  if (a.c.bits == 4) {
    if (dtype == MI355X_BF16) launch_rows<Pages4<bf16, D>, bf16>(a, qt, blocks, s);
    else launch_rows<Pages4<f16, D>, f16>(a, qt, blocks, s);
  } else if (dtype == MI355X_F32) {
    launch_rows<Pages32<D>, float>(a, qt, blocks, s);
  } else if (dtype == MI355X_BF16) {
    launch_rows<Pages16<bf16, D>, bf16>(a, qt, blocks, s);
  } else {
    launch_rows<Pages16<f16, D>, f16>(a, qt, blocks, s);
  }
}

}  // namespace

bool paged_mfma_takes(const mi355x_paged_cache& c, int dtype) {
  if (c.d != 64 && c.d != 128 && c.d != 256) return false;
  if (c.bits != 4) return true;
  if (dtype == MI355X_F32) return false;  // queries would lose what f16 does not hold
  const int64_t align = c.d / 8 < 16 ? c.d / 8 : 16;  // of a row of scales
  for (const int64_t* st : {c.ks_phs, c.vs_phs})
    for (int i = 0; i < 3; ++i)
      if (st[i] * 2 % align) return false;
  return ((uintptr_t)c.k_scales | (uintptr_t)c.v_scales) % align == 0;
}

// Query rows of 16 that share a block: two where there are that many and
// registers hold their output (head_dim 256 would spill).
int paged_mfma_row_tiles(int64_t rows, int64_t d) { return rows > 16 && d < 256 ? 2 : 1; }

int paged_mfma_launch(DecodeArgs a, int dtype, hipStream_t s) {
  const int qt = paged_mfma_row_tiles((int64_t)a.group * a.seq, a.c.d);
  a.row_groups = ((int64_t)a.group * a.seq + 16 * qt - 1) / (16 * qt);
  a.units = a.batch * a.c.kv_heads * a.splits;
  const int64_t blocks = (a.units + 7) / 8 * 8 * a.row_groups;
  MI_REQUIRE(blocks < (1ll << 24), "mi355x_paged_attn: %lld blocks", (long long)blocks);
  if (a.c.d == 64) launch_format<64>(a, qt, dtype, (unsigned)blocks, s);
  else if (a.c.d == 128) launch_format<128>(a, qt, dtype, (unsigned)blocks, s);
  else launch_format<256>(a, qt, dtype, (unsigned)blocks, s);
  return MI355X_OK;
}

}  // namespace mi
