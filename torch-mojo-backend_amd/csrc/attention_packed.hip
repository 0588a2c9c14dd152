// Causal attention over sequences of different lengths laid end to end, with a
// window where asked for and grouped K/V heads, forward and backward, on matrix
// cores (bf16 and f16; f32 in attention_f32.hip).
//
// For the rows i, j of one sequence, j <= i and (window w) i - j < w:
//   S = scale q_i k_j, P = softmax_j(S), O = P V, LSE_i = log sum_j exp(S)
//   D_i = dO_i O_i, dP = dO V^T, dS = P (dP - D), dV = P^T dO,
//   dQ = scale dS K, dK = scale dS^T Q, those of a K/V head summed over its query heads.
//
// A block takes a tile of one sequence from the plan (packed.h) and one head,
// and walks 64-row tiles of that sequence alone; rows past its end are loaded as
// the last row and masked.  Products are laid out so that a query's softmax
// state (backward: a key's, or a query's, sums) stays in its lanes:
//   forward  S^T = K Q^T, O^T += V^T P^T, P^T fed from S^T's accumulators;
//   dK, dV   S = Q K^T (keys are columns), dV^T += dO^T P, dK^T += Q^T dS;
//   dQ       S^T = K Q^T, dQ^T += K^T dS^T.
// The transposed operands are read from row-major tiles (ds_read_b64_tr_b16).
// head_dim is any multiple of 8.  Kernels are made for the widths W of 64, 96, 128,
// 192 and 256 channels, with rows of D = 64, 128 or 256 in LDS; a head_dim between
// two runs those of the next (RAG), with zeros in the channels past it.
// P and dS are rounded to the type for their products, half a step each; what
// rounding takes from a 16-bit O is kept (o_low) and D taken from both.  LSE is that
// of the rounded P, by whose sum O is divided, so that the backward's P carries its
// rounding and its own.
//
// What bounds them: at 128 channels the matrix units, at the rate of a large matrix
// product (16384 rows in 4 sequences, 32 over 8 heads, bf16: forward 622 us, 1015
// TFLOP/s of the pairs seen; dK and dV 1240, dQ 758, 1020 and 1250 with the products
// that both take; matrix units busy 51, 47 and 62% of the cycles at 2.2 GHz).  At 64
// the softmax's arithmetic beside them (16384 rows, 96 heads: 830 TFLOP/s of the
// tiles' pairs), and in short sequences a block's first loads and last stores and
// the tiles' masked corners: 48 sequences of 16384 rows, 12 heads, 44 us forward,
// 126 MB and 20.8 GFLOP in tiles, 98 us backward.  At 256 the reads of LDS.
#include <algorithm>
#include <atomic>

#include "attention_f32.h"
#include "attention_tile.h"
#include "packed.h"

extern __shared__ __attribute__((aligned(1024))) char packed_lds[];

namespace mi {
namespace {

// Strides in elements, of rows and of heads.
struct Rows {
  const void* p;
  int64_t row, head;
  template <typename T>
  __device__ __forceinline__ T* at(int64_t r, int64_t h) const { return (T*)p + r * row + h * head; }
};

struct PackedArgs {
  Rows q, k, v, o, dout, dq, dk, dv;
  const void* o_low;  // null, or laid out as o
  float* lse;         // [heads][tokens]
  const PackedHeader* head;
  const PackedTile* tiles[2];  // of 128 and of 64 rows
  int tokens, heads, kv_heads, d;
  int window;          // 0: none
  bool all_fine;       // whether the call can have no other tiles than fine ones (the backward, below)
  float c, sign, scale;  // |scale| log2(e), scale's sign
  float *ndelta, *nlse2;  // [heads][tokens]: -D, -LSE log2(e)
  float* kv_part;      // dK and then dV of each query head [group][kv_heads][tokens][D] (f32), or null
};

// Loads of 64-row tiles into the layout of KvLayout by NW waves.  A lane's rows
// of a tile lie NW * RPI apart, and the chunk it takes of them is the same (of
// rows 8 apart, at head_dim 256 in four waves, one of two), so that one or two
// 32-bit offsets a lane serve all: addresses made lane by lane took 16 registers
// of the backward's and an add a load.  Chunks past d are left as they are: RAG,
// zeros that the block wrote before its first load, or past W, never read.
constexpr int64_t kMostRowBytes = (1ll << 32) / 64 - 64;  // of 64 rows' offsets in 32 bits
template <int W>
constexpr int kLayout = W <= 64 ? 64 : W <= 128 ? 128 : 256;
template <int W, int NW, bool RAG>
struct TileLoad {
  static constexpr int D = kLayout<W>;
  static constexpr bool PART = RAG || W < D;
  typedef KvLayout<D> L;
  static constexpr int IT = L::TILE / 1024 / NW, STEP = NW * L::RPI;
  static constexpr int KINDS = (STEP & (D == 64 ? 7 : 15)) ? 2 : 1;
  static_assert(STEP % 8 == 0, "");
  const char* g;
  uint32_t rs;
  uint32_t off[KINDS];
  bool keep[KINDS];
  __device__ __forceinline__ void init(const void* base, int64_t rs_bytes, int d) {
    g = (const char*)base;
    rs = (uint32_t)rs_bytes;
    const int lane = threadIdx.x & 63, r = wave_id() * L::RPI + lane / L::CH;
#pragma unroll
    for (int k = 0; k < KINDS; ++k) {
      const int c = (lane % L::CH) ^ L::swz(r + k * STEP);
      off[k] = r * rs + c * 16;
      keep[k] = !PART || c * 8 < d;
    }
  }
  __device__ __forceinline__ void issue(int row0, int nrows, char* dst) const {
    const int wave = wave_id();
    const char* tb = g + (int64_t)row0 * rs;
    const unsigned lds = lds_base_of(dst) + wave * 1024;
    if (row0 + 64 <= nrows) {
#pragma unroll
      for (int it = 0; it < IT; ++it)
        if (!PART || keep[it % KINDS]) dma_b128_at(tb + (uint64_t)(it * STEP) * rs, off[it % KINDS], lds + it * (NW * 1024));
    } else {
      const int r = wave * L::RPI + (int)(threadIdx.x & 63) / L::CH;
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const uint32_t o = off[it % KINDS] - r * rs + min(r + it * STEP, nrows - 1 - row0) * rs;
        if (!PART || keep[it % KINDS]) dma_b128_at(tb, o, lds + it * (NW * 1024));
      }
    }
  }
};

// RAG: zeros in a block's tiles, before the first load.
__device__ __forceinline__ void clear_lds(char* lds, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *(u32x4*)(lds + i) = u32x4{0, 0, 0, 0};
  __syncthreads();
}

// 16 rows' fragments of a wave: row lr, channels 32 ks + 8 lg .. + 7 (zeros past
// d), times +-1 or 0.
template <typename T, int W, bool RAG>
__device__ __forceinline__ void load_frags(const T* row, bool there, int lg, int d, float sign, typename Mfma<T>::frag (&f)[W / 32]) {
#pragma unroll
  for (int ks = 0; ks < W / 32; ++ks) {
    f[ks] = there && (!RAG || ks * 32 + lg * 8 < d) ? *(const typename Mfma<T>::frag*)(row + ks * 32 + lg * 8) : zero_frag<T>();
    if (sign != 1.f)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[ks][e] = (T)(to_f32(f[ks][e]) * sign);
  }
}

// Zeros in rows that belong to no sequence.
template <typename T>
__device__ __forceinline__ void zero_rows(const Rows& x, const PackedTile& t, int h, int d) {
  const int per = d / 8;
  for (int i = threadIdx.x; i < t.len * per; i += blockDim.x) {
    const int r = i / per;
    V8<T> z;
#pragma unroll
    for (int e = 0; e < 8; ++e) z.v[e] = (T)0.f;
    T* p = x.at<T>(t.start + r, h) + (i - r * per) * 8;
    *(V4<T>*)p = *(const V4<T>*)z.v, *(V4<T>*)(p + 4) = *(const V4<T>*)z.v;
  }
}

// ---------------------------------------------------------------------------
// forward.  NW waves take QPW queries each, QPB in all; with KH = 2 the waves'
// halves take half of a tile's keys each and join at the end.
// ---------------------------------------------------------------------------
template <typename T, int W, bool RAG, int NW, int QPW, int KH>
__global__ void __launch_bounds__(64 * NW, W > 128 ? 1 : 2) packed_fwd(PackedArgs p) {
  constexpr int D = kLayout<W>;
  constexpr int QT = QPW / 16, QPB = NW / KH * QPW;
  constexpr int LIST = QPB == 128 ? 0 : 1;
  static_assert(QPB == kPackedRows[LIST], "");
  typedef typename Mfma<T>::frag frag;
  typedef KvLayout<D> L;
  constexpr int KS = W / 32, DT = W / 16;
  constexpr int STAGE = 2 * L::TILE;
  constexpr int KN = 64 / KH;
  char* const lds = packed_lds;

  const PackedAt at = packed_at(p.tiles[LIST], p.head->count[LIST], blockIdx.x, p.heads, p.kv_heads);
  if (!at.live) return;
  const int start = at.t.start, len = at.t.len, h = at.h;
  float* const lse = p.lse + (int64_t)h * p.tokens + start;
  if (at.t.tile < 0) {
    zero_rows<T>(p.o, at.t, h, p.d);
    for (int i = threadIdx.x; i < len; i += blockDim.x) lse[i] = -INFINITY;
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = KH == 1 ? wave_id() : wave_id() % (NW / KH);
  const int wk = KH == 1 ? 0 : wave_id() / (NW / KH);
  const int lr = lane & 15, lg = lane >> 4;
  const int q0 = at.t.tile * QPB, qw = q0 + wave * QPW;
  const int window = p.window > 0 ? min(p.window, len) : len;

  if constexpr (RAG) clear_lds(lds, 2 * STAGE);
  TileLoad<W, NW, RAG> kl, vl;
  kl.init(p.k.at<T>(start, at.hk), p.k.row * (int64_t)sizeof(T), p.d);
  vl.init(p.v.at<T>(start, at.hk), p.v.row * (int64_t)sizeof(T), p.d);
  const int kv_end = min(len, q0 + QPB);
  const int j0 = max(0, q0 - window + 1) / 64;  // the first tile that any query sees
  kl.issue(j0 * 64, len, lds);
  vl.issue(j0 * 64, len, lds + L::TILE);

  frag qf[QT][KS];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int qi = qw + qt * 16 + lr;
    load_frags<T, W, RAG>(p.q.at<T>(start + min(qi, len - 1), h), qi < len, lg, p.d, p.sign, qf[qt]);
  }
  frag ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (T)1.0f;
  float m[QT];
  f32x4 oacc[DT][QT], lacc[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m[qt] = -INFINITY;
    lacc[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int sw = L::swz(lr);
  const TrOffsets<D> tro;
  const float c = p.c;
  int buf = 0;
  auto step = [&](int j, auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const int kb0 = j * 64;
    __builtin_amdgcn_s_waitcnt(0xc07f & 0x3f70);  // vmcnt(0)
    __syncthreads();
    if (kb0 + 64 < kv_end) {
      char* nx = lds + (buf ^ 1) * STAGE;
      kl.issue(kb0 + 64, len, nx);
      vl.issue(kb0 + 64, len, nx + L::TILE);
    }
    const char* Kt = lds + buf * STAGE + wk * (L::TILE / KH);
    const char* Vt = Kt + L::TILE;
    const int kb = kb0 + wk * KN;  // the wave's first key
    buf ^= 1;
    // a tile that none of the wave's queries see: its loads and barriers only
    if (MASK && (kb > qw + QPW - 1 || kb + KN - 1 < qw - window + 1 || qw >= len)) return;
    // the keys kb + lo .. lim are visible to the lane's query (keys past the
    // sequence lie behind every query of it)
    int lo[QT], lim[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int qi = qw + qt * 16 + lr;
      lim[qt] = qi - kb;
      lo[qt] = qi - window + 1 - kb;
    }
    f32x4 s[4 / KH][QT];
    float mx[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) mx[qt] = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4 / KH; ++kt) {
      frag kf[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[ks] = *(const frag*)(Kt + (kt * 16 + lr) * L::ROWB + (((ks * 4 + lg) ^ sw) << 4));
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) a = Mfma<T>::mma(kf[ks], qf[qt][ks], a);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = kt * 16 + lg * 4 + e;
          if (MASK && (key > lim[qt] || key < lo[qt])) a[e] = -INFINITY;
          mx[qt] = fmaxf(mx[qt], a[e]);
        }
        s[kt][qt] = a;
      }
    }
    // the running maximum is a reference that moves when a row's maximum
    // passes it by more than kSlack: most steps rescale nothing
    float mxc[QT];
    bool need = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      mxc[qt] = group_max(mx[qt]) * c;
      need |= mxc[qt] > m[qt] + kSlack;
    }
    if (__builtin_amdgcn_ballot_w64(need)) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const float m_new = fmaxf(m[qt], mxc[qt]);
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m[qt] - m_new);
        lacc[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) oacc[dt][qt] *= alpha;
        m[qt] = m_new;
      }
    }
    float m_use[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) m_use[qt] = m[qt] == -INFINITY ? 0.f : m[qt];
#pragma unroll
    for (int ks2 = 0; ks2 < 2 / KH; ++ks2) {
      frag pf[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) pf[qt][4 * u + e] = (T)fast_exp2(fmaf(s[2 * ks2 + u][qt][e], c, -m_use[qt]));
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) lacc[qt] = Mfma<T>::mma(ones, pf[qt], lacc[qt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const frag vf = tr_frag_at<T, D>(Vt, tro, dt, 2 * ks2, 2 * ks2 + 1);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) oacc[dt][qt] = Mfma<T>::mma(vf, pf[qt], oacc[dt][qt]);
      }
    }
  };
  const int nkb = (kv_end + 63) / 64;
  // masked [j0, jl) (the window's edge), unmasked [jl, ju), masked [ju, nkb)
  const int jl = min(nkb, max(j0, (max(0, qw + QPW - window) + 63) / 64));
  const int ju = max(jl, min(nkb, qw / 64));
  int j = j0;
  for (; j < jl; ++j) step(j, BoolTag<true>{});
  for (; j < ju; ++j) step(j, BoolTag<false>{});
  for (; j < nkb; ++j) step(j, BoolTag<true>{});

  float l[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) l[qt] = lacc[qt][0];
  if constexpr (KH == 2) {
    static_assert(NW / 2 * QT * (DT * 1024 + 512) <= 2 * STAGE, "");
    __builtin_amdgcn_s_waitcnt(0xc07f & 0x3f70);
    __syncthreads();
    f32x4* const ox = (f32x4*)lds + wave * QT * DT * 64 + lane;
    float2* const mx = (float2*)(lds + NW / 2 * QT * DT * 1024) + wave * QT * 64 + lane;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
      if (wk) {
        mx[qt * 64] = make_float2(m[qt], l[qt]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) ox[(qt * DT + dt) * 64] = oacc[dt][qt];
      }
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float2 other = mx[qt * 64];
      const float top = fmaxf(m[qt], other.x);
      const float a0 = m[qt] == -INFINITY ? 0.f : fast_exp2(m[qt] - top);
      const float a1 = other.x == -INFINITY ? 0.f : fast_exp2(other.x - top);
      l[qt] = l[qt] * a0 + other.y * a1;
      m[qt] = top;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) oacc[dt][qt] = oacc[dt][qt] * a0 + ox[(qt * DT + dt) * 64] * a1;
    }
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int qi = qw + qt * 16 + lr;
    if (qi >= len) continue;
    T* const O = p.o.at<T>(start + qi, h);
    T* const low = p.o_low ? (T*)p.o_low + (O - (T*)p.o.p) : nullptr;
    const float inv = 1.f / l[qt];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (RAG && dt * 16 + lg * 4 >= p.d) continue;
      V4<T> o4;
#pragma unroll
      for (int e = 0; e < 4; ++e) o4.v[e] = (T)(oacc[dt][qt][e] * inv);
      *(V4<T>*)(O + dt * 16 + lg * 4) = o4;
      if (low) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o4.v[e] = (T)(oacc[dt][qt][e] * inv - to_f32(o4.v[e]));
        *(V4<T>*)(low + dt * 16 + lg * 4) = o4;
      }
    }
    if (lg == 0) lse[qi] = (m[qt] + log2f(l[qt])) * kLn2;
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// -D and -LSE log2(e) of every row: D / 8 lanes a row.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) packed_delta(PackedArgs p) {
  constexpr int CPR = D / 8, RPB = kThreads / CPR;
  const uint32_t row = blockIdx.x * (uint32_t)RPB + threadIdx.x / CPR;
  const int ch = threadIdx.x % CPR;
  const uint32_t total = (uint32_t)p.heads * (uint32_t)p.tokens, h = row / (uint32_t)p.tokens, t = row - h * (uint32_t)p.tokens;
  const bool there = row < total && (int)t >= p.head->begin && (int)t < p.head->end;
  float acc = 0.f;
  if (there && ch * 8 < p.d) {
    const T* po = p.o.at<T>(t, h) + ch * 8;
    const V8<T> o = *(const V8<T>*)po, g = *(const V8<T>*)(p.dout.at<T>(t, h) + ch * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc += to_f32(o.v[e]) * to_f32(g.v[e]);
    if (p.o_low) {
      const V8<T> l = *(const V8<T>*)((const T*)p.o_low + (po - (const T*)p.o.p));
#pragma unroll
      for (int e = 0; e < 8; ++e) acc += to_f32(l.v[e]) * to_f32(g.v[e]);
    }
  }
#pragma unroll
  for (int off = CPR / 2; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  if (there && ch == 0) {
    p.ndelta[row] = -acc;
    p.nlse2[row] = -p.lse[row] * kLog2e;
  }
}

// 16-key tiles of a wave: two would take all registers at 256 (794 spilled); at
// 192 they take 436 (16384 rows, 8 over 2 heads, in 4 sequences: 971 us, one 1100).
// Eight waves of one at 256 spill 28 (16384 rows, 16 over 4 heads, in 4 sequences:
// keys 2427 us and queries 970 in two launches, 2581 in one as it is).
template <int W>
constexpr int kKeyTiles = W > 192 ? 1 : 2;
template <int W>
constexpr int kKeyList = kKeyTiles<W> == 1 ? 1 : 0;
constexpr int kQueryTiles = 2;
// Sequences, or windows, of no more rows than this take what rounding took from dS
// to a product of its own (FINE; all their steps are masked ones): a gradient of
// few terms is off by its own rounding and by theirs, up to 1.9 times its own alone
// in sequences of 2 to 9 rows.  In longer ones it is 1.45 times, and the product a
// quarter of the queries' pass.  In a body of its own, and at 128 channels the keys
// in a launch of their own: in one kernel their loop took 1.09 times as long (1397
// us where it takes 1280), in one body 1.15.  Where both bodies share a kernel of two
// waves a SIMD (96 channels, and the queries at 128) the fine one's halves of a step
// are a loop: unrolled they spilled 6 to 11 registers of f16 (and 8 of bf16 at 72 to
// 88 channels); 300 sequences of 55 rows, 32 over 8 heads of 128, f16: queries 147 us,
// unrolled 163 (the keys, which have the registers, 154 and as a loop 163).  A
// launch of the fine queries with the fine keys, one wave a SIMD, took 398 us for both.
constexpr int kFine = 64;
__device__ __forceinline__ bool is_fine(const PackedArgs& p, const PackedTile& t) {
  return t.len <= kFine || (p.window > 0 && p.window <= kFine);
}

// dK and dV of a tile of keys, over the query heads [g0, g1) of its group.
template <typename T, int W, bool RAG, bool FINE>
__device__ __forceinline__ void dkv_body(const PackedArgs& p, const PackedTile& t, int hk, int g0, int g1, char* lds) {
  constexpr int D = kLayout<W>;
  typedef typename Mfma<T>::frag frag;
  typedef KvLayout<D> L;
  constexpr int RT = kKeyTiles<W>, KW = 16 * RT, KS = W / 32, DT = W / 16;
  constexpr int STAGE = 2 * L::TILE + 512;  // a Q and a dO tile, -LSE log2(e)[64], -D[64]
  const int lane = threadIdx.x & 63, wave = wave_id(), lr = lane & 15, lg = lane >> 4;
  const int start = t.start, len = t.len, group = p.heads / p.kv_heads;
  // (the list's number counts from the end: the first keys' tiles take longest)
  constexpr int KB = 4 * KW;
  const int tile = (len - 1) / KB - t.tile;
  const int k0 = tile * KB, kw = k0 + wave * KW;
  const int window = p.window > 0 ? min(p.window, len) : len;

  if constexpr (RAG) clear_lds(lds, 2 * STAGE);
  frag kf[RT][KS], vf[RT][KS];
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const int kj = kw + u * 16 + lr, row = start + min(kj, len - 1);
    load_frags<T, W, RAG>(p.k.at<T>(row, hk), kj < len, lg, p.d, p.sign, kf[u]);
    load_frags<T, W, RAG>(p.v.at<T>(row, hk), kj < len, lg, p.d, 1.f, vf[u]);
  }
  f32x4 dva[DT][RT], dka[DT][RT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int u = 0; u < RT; ++u) dva[dt][u] = dka[dt][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int qstart = k0 / 64 * 64;  // the steps that see the tile's keys
  const int qend = min(len, k0 + KB - 1 + window);
  const int nqb = (qend - qstart + 63) / 64, nsteps = nqb * (g1 - g0);
  const int sw = L::swz(lr);
  const TrOffsets<D> tro;
  TileLoad<W, 4, RAG> ql, dl;
  auto head_of = [&](int g) {
    const int h = hk * group + g;
    ql.init(p.q.at<T>(start, h), p.q.row * (int64_t)sizeof(T), p.d);
    dl.init(p.dout.at<T>(start, h), p.dout.row * (int64_t)sizeof(T), p.d);
  };
  int gload = g0, jload = 0;  // the next step to load
  auto issue = [&](char* st) {
    const int qb0 = qstart + jload * 64;
    ql.issue(qb0, len, st);
    dl.issue(qb0, len, st + L::TILE);
    if (wave < 2) {
      const float* src = (wave == 0 ? p.nlse2 : p.ndelta) + (int64_t)(hk * group + gload) * p.tokens + start + min(qb0 + lane, len - 1);
      dma_b32(src, lds_base_of(st + 2 * L::TILE + wave * 256));
    }
    if (++jload == nqb) {
      jload = 0;
      if (++gload < g1) head_of(gload);
    }
  };
  head_of(g0);
  issue(lds);
  int buf = 0, done = 0;
  auto step = [&](int j, auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const int qb0 = qstart + j * 64;
    __builtin_amdgcn_s_waitcnt(0xc07f & 0x3f70);  // vmcnt(0)
    __syncthreads();
    if (++done < nsteps) issue(lds + (buf ^ 1) * STAGE);
    const char* Qt = lds + buf * STAGE;
    const char* dOt = Qt + L::TILE;
    const float* lse_s = (const float*)(Qt + 2 * L::TILE);
    const float* del_s = lse_s + 64;
    buf ^= 1;
    if (MASK && (kw > qb0 + 63 || qb0 >= kw + KW - 1 + window || kw >= len)) return;  // no query sees the wave's keys
    const int kq = kw - qb0;  // the wave's first key minus the step's first query
    const float c = p.c;
    // query row qr sees the lane's key iff lo <= qr < lo + span: causal order,
    // window and the sequence's end in one unsigned compare; a dropped score's
    // exponent is -inf
    int lo[RT], span[RT];
    if constexpr (MASK)
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        const int kr = u * 16 + lr;
        lo[u] = max(0, kq + kr);
        span[u] = kw + kr < len ? max(0, min(len - qb0, min(64, kq + kr + window)) - lo[u]) : 0;
      }
#pragma unroll (FINE && W == 96 ? 1 : 2)
    for (int qs = 0; qs < 2; ++qs) {
      if (MASK && (qs * 32 + 31 < kq || qs * 32 >= kq + KW - 1 + window || qb0 + qs * 32 >= len)) continue;
      frag pb[RT], sb[RT], sl[FINE ? RT : 1];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int qt = 2 * qs + w;
        frag qa[KS], da[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int off = (qt * 16 + lr) * L::ROWB + (((ks * 4 + lg) ^ sw) << 4);
          qa[ks] = *(const frag*)(Qt + off);
          da[ks] = *(const frag*)(dOt + off);
        }
        const f32x4 l4 = *(const f32x4*)(lse_s + qt * 16 + 4 * lg), d4 = *(const f32x4*)(del_s + qt * 16 + 4 * lg);
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          f32x4 sa = {0.f, 0.f, 0.f, 0.f}, pa = d4;  // dP - D
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            sa = Mfma<T>::mma(qa[ks], kf[u][ks], sa);
            pa = Mfma<T>::mma(da[ks], vf[u][ks], pa);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = fmaf(sa[e], c, l4[e]);
            if constexpr (MASK) {
              const int qr = qt * 16 + 4 * lg + e;
              x = (unsigned)(qr - lo[u]) < (unsigned)span[u] ? x : -INFINITY;
            }
            const float pv = fast_exp2(x);
            pb[u][4 * w + e] = (T)pv;
            sb[u][4 * w + e] = (T)(pv * pa[e]);
            if constexpr (FINE) sl[u][4 * w + e] = (T)(pv * pa[e] - to_f32(sb[u][4 * w + e]));
          }
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const frag dof = tr_frag_at<T, D>(dOt, tro, dt, 2 * qs, 2 * qs + 1);
        const frag qtf = tr_frag_at<T, D>(Qt, tro, dt, 2 * qs, 2 * qs + 1);
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          dva[dt][u] = Mfma<T>::mma(dof, pb[u], dva[dt][u]);
          dka[dt][u] = Mfma<T>::mma(qtf, sb[u], dka[dt][u]);
          if constexpr (FINE) dka[dt][u] = Mfma<T>::mma(qtf, sl[u], dka[dt][u]);
        }
      }
    }
  };
  // masked [0, j1) (the causal diagonal), unmasked [j1, j2), masked [j2, nqb)
  int j1 = nqb, j2 = nqb;
  if (kw + KW <= len) {
    j1 = min(nqb, (max(0, kw + KW - 1 - qstart) + 63) / 64);
    j2 = max(j1, min(nqb, max(0, min(len, kw + window) - qstart) / 64));
  }
  for (int g = g0; g < g1; ++g) {
    int j = 0;
    for (; j < j1; ++j) step(j, BoolTag<true>{});
    if constexpr (!FINE)
      for (; j < j2; ++j) step(j, BoolTag<false>{});
    for (; j < nqb; ++j) step(j, BoolTag<true>{});
  }
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const int kj = kw + u * 16 + lr;
    if (kj >= len) continue;
    if (p.kv_part) {
      float* pk = p.kv_part + (((int64_t)g0 * p.kv_heads + hk) * p.tokens + start + kj) * D;
      const int64_t plane = (int64_t)p.heads * p.tokens * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        *(f32x4*)(pk + dt * 16 + lg * 4) = dka[dt][u];
        *(f32x4*)(pk + plane + dt * 16 + lg * 4) = dva[dt][u];
      }
      continue;
    }
    T* const dK = p.dk.at<T>(start + kj, hk);
    T* const dV = p.dv.at<T>(start + kj, hk);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (RAG && dt * 16 + lg * 4 >= p.d) continue;
      V4<T> k4, v4;
#pragma unroll
      for (int e = 0; e < 4; ++e) k4.v[e] = (T)(dka[dt][u][e] * p.scale), v4.v[e] = (T)dva[dt][u][e];
      *(V4<T>*)(dK + dt * 16 + lg * 4) = k4;
      *(V4<T>*)(dV + dt * 16 + lg * 4) = v4;
    }
  }
}

// dQ of a tile of 128 queries of one head.
template <typename T, int W, bool RAG, bool FINE>
__device__ __forceinline__ void dq_body(const PackedArgs& p, const PackedTile& t, int h, int hk, char* lds) {
  constexpr int D = kLayout<W>;
  typedef typename Mfma<T>::frag frag;
  typedef KvLayout<D> L;
  constexpr int RT = kQueryTiles, QW = 16 * RT, QB = 4 * QW, KS = W / 32, DT = W / 16;
  static_assert(QB == 128, "");
  constexpr int STAGE = 2 * L::TILE;
  const int lane = threadIdx.x & 63, wave = wave_id(), lr = lane & 15, lg = lane >> 4;
  const int start = t.start, len = t.len, q0 = t.tile * QB, qw = q0 + wave * QW;
  const int window = p.window > 0 ? min(p.window, len) : len;

  if constexpr (RAG) clear_lds(lds, 2 * STAGE);
  TileLoad<W, 4, RAG> kl, vl;
  kl.init(p.k.at<T>(start, hk), p.k.row * (int64_t)sizeof(T), p.d);
  vl.init(p.v.at<T>(start, hk), p.v.row * (int64_t)sizeof(T), p.d);
  const int kv_end = min(len, q0 + QB);
  const int jw = max(0, q0 - window + 1) / 64;
  kl.issue(jw * 64, len, lds);
  vl.issue(jw * 64, len, lds + L::TILE);

  frag qf[RT][KS], df[RT][KS];
  float lse2[RT], dlt[RT];
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const int qi = qw + u * 16 + lr, qc = min(qi, len - 1);
    load_frags<T, W, RAG>(p.q.at<T>(start + qc, h), qi < len, lg, p.d, p.sign, qf[u]);
    load_frags<T, W, RAG>(p.dout.at<T>(start + qc, h), qi < len, lg, p.d, 1.f, df[u]);
    lse2[u] = p.nlse2[(int64_t)h * p.tokens + start + qc];
    dlt[u] = p.ndelta[(int64_t)h * p.tokens + start + qc];
  }
  f32x4 dqa[DT][RT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int u = 0; u < RT; ++u) dqa[dt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int sw = L::swz(lr);
  const TrOffsets<D> tro;
  int buf = 0;
  auto step = [&](int j, auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const int kb0 = j * 64;
    __builtin_amdgcn_s_waitcnt(0xc07f & 0x3f70);  // vmcnt(0)
    __syncthreads();
    if (kb0 + 64 < kv_end) {
      char* nx = lds + (buf ^ 1) * STAGE;
      kl.issue(kb0 + 64, len, nx);
      vl.issue(kb0 + 64, len, nx + L::TILE);
    }
    const char* Kt = lds + buf * STAGE;
    const char* Vt = Kt + L::TILE;
    buf ^= 1;
    if (MASK && (kb0 > qw + QW - 1 || kb0 + 63 < qw - window + 1 || qw >= len)) return;
    const int qk = qw - kb0;  // the wave's first query minus the step's first key
    const float c = p.c;
    int lim[RT], lo[RT];  // key rows lo .. lim - 1 are visible to the lane's query
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const int qr = u * 16 + lr;
      lim[u] = qw + qr < len ? qk + qr + 1 : 0;
      lo[u] = qk + qr - window + 1;
    }
#pragma unroll (FINE && (W == 96 || W == 128) ? 1 : 2)
    for (int ks2 = 0; ks2 < 2; ++ks2) {
      if (MASK && (ks2 * 32 > qk + QW - 1 || ks2 * 32 + 31 < qk - window + 1)) continue;
      frag sb[RT], sl[FINE ? RT : 1];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int kt = 2 * ks2 + w;
        frag ka[KS], va[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int off = (kt * 16 + lr) * L::ROWB + (((ks * 4 + lg) ^ sw) << 4);
          ka[ks] = *(const frag*)(Kt + off);
          va[ks] = *(const frag*)(Vt + off);
        }
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          f32x4 sa = {0.f, 0.f, 0.f, 0.f}, pa = {dlt[u], dlt[u], dlt[u], dlt[u]};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            sa = Mfma<T>::mma(ka[ks], qf[u][ks], sa);
            pa = Mfma<T>::mma(va[ks], df[u][ks], pa);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = fmaf(sa[e], c, lse2[u]);
            if constexpr (MASK) {
              const int key = kt * 16 + 4 * lg + e;
              x = key < lim[u] && key >= lo[u] ? x : -INFINITY;
            }
            const float sv = fast_exp2(x) * pa[e];
            sb[u][4 * w + e] = (T)sv;
            if constexpr (FINE) sl[u][4 * w + e] = (T)(sv - to_f32(sb[u][4 * w + e]));
          }
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const frag ktf = tr_frag_at<T, D>(Kt, tro, dt, 2 * ks2, 2 * ks2 + 1);
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          dqa[dt][u] = Mfma<T>::mma(ktf, sb[u], dqa[dt][u]);
          if constexpr (FINE) dqa[dt][u] = Mfma<T>::mma(ktf, sl[u], dqa[dt][u]);
        }
      }
    }
  };
  const int nkb = (kv_end + 63) / 64;
  // masked [jw, jl) (the window's edge), unmasked [jl, ju), masked [ju, nkb)
  const int jl = min(nkb, max(jw, (max(0, qw + QW - window) + 63) / 64));
  const int ju = qw + QW <= len ? max(jl, min(nkb, (qw + 1) / 64)) : jl;
  int j = jw;
  for (; j < jl; ++j) step(j, BoolTag<true>{});
  if constexpr (!FINE)
    for (; j < ju; ++j) step(j, BoolTag<false>{});
  for (; j < nkb; ++j) step(j, BoolTag<true>{});
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const int qi = qw + u * 16 + lr;
    if (qi >= len) continue;
    T* const dQ = p.dq.at<T>(start + qi, h);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (RAG && dt * 16 + lg * 4 >= p.d) continue;
      V4<T> q4;
#pragma unroll
      for (int e = 0; e < 4; ++e) q4.v[e] = (T)(dqa[dt][u][e] * p.scale);
      *(V4<T>*)(dQ + dt * 16 + lg * 4) = q4;
    }
  }
}

// KIND 0, both in one launch: the first nkv blocks take keys, one of a K/V
// head's or, where their gradients go through partials, one of a query head's;
// the rest take queries.  1: keys alone, but for FINE tiles, which 3 takes (4.8 us
// where there are none; 1 is left out where the call can have no others), 2: queries
// alone.  At head_dim 128 the keys' blocks need 381 registers, a wave a SIMD, and
// the queries' 251, two; in one launch both run at the first ([16384 rows, 32 over 8, 128] in 4 sequences:
// 2370 us, 1335 + 774 in two).  Four tiles of keys a wave, two waves a block,
// spill (4.9 ms, 39 registers of 512 short with the sums pinned in AGPRs); four of
// queries take 960.  At 64 and 96 both run at two in one launch (96 channels
// 570 us of 16384 rows, 12 heads, in 4 sequences; 564 in two, 781 as 128).
template <typename T, int W, bool RAG, int KIND>
__global__ void __launch_bounds__(kThreads, W <= 96 || (W == 128 && KIND == 2) ? 2 : 1) packed_bwd(PackedArgs p, uint32_t nkv) {
  constexpr int D = kLayout<W>;
  char* const lds = packed_lds;
  const int group = p.heads / p.kv_heads;
  if (KIND % 2 || (KIND == 0 && blockIdx.x < nkv)) {
    const PackedAt at = packed_at(p.tiles[kKeyList<W>], p.head->count[kKeyList<W>], blockIdx.x, p.kv_part ? p.heads : p.kv_heads, p.kv_heads);
    if (!at.live || (KIND == 3 && at.t.tile < 0 && !p.all_fine)) return;
    const int g = p.kv_part ? at.h - at.hk * group : 0;
    if (at.t.tile < 0) {
      if (g == 0) zero_rows<T>(p.dk, at.t, at.hk, p.d), zero_rows<T>(p.dv, at.t, at.hk, p.d);
      return;
    }
    const int g1 = p.kv_part ? g + 1 : group;
    if (is_fine(p, at.t)) {
      if constexpr (KIND != 1) dkv_body<T, W, RAG, true>(p, at.t, at.hk, g, g1, lds);
    } else {
      if constexpr (KIND != 3) dkv_body<T, W, RAG, false>(p, at.t, at.hk, g, g1, lds);
    }
    return;
  }
  if constexpr (KIND % 2 == 0) {
    const PackedAt at = packed_at(p.tiles[0], p.head->count[0], blockIdx.x - nkv, p.heads, p.kv_heads);
    if (!at.live) return;
    if (at.t.tile < 0) return zero_rows<T>(p.dq, at.t, at.h, p.d);
    if (is_fine(p, at.t)) return dq_body<T, W, RAG, true>(p, at.t, at.h, at.hk, lds);
    dq_body<T, W, RAG, false>(p, at.t, at.h, at.hk, lds);
  }
}

// dK and dV from the f32 partials of a group's query heads, added in head order.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) packed_sum(PackedArgs p) {
  const int64_t i4 = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = i4 / (D / 4), hk = row / p.tokens;
  const int t = (int)(row - hk * p.tokens), d = (int)(i4 - row * (D / 4)) * 4;
  if (hk >= p.kv_heads || d >= p.d || t < p.head->begin || t >= p.head->end) return;
  const int64_t plane = (int64_t)p.heads * p.tokens * D;
  f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sv = sk;
  const int group = p.heads / p.kv_heads;
#pragma unroll 4
  for (int g = 0; g < group; ++g) {
    const float* pk = p.kv_part + (((int64_t)g * p.kv_heads + hk) * p.tokens + t) * D + d;
    sk += *(const f32x4*)pk, sv += *(const f32x4*)(pk + plane);
  }
  V4<T> k4, v4;
#pragma unroll
  for (int e = 0; e < 4; ++e) k4.v[e] = (T)(sk[e] * p.scale), v4.v[e] = (T)sv[e];
  *(V4<T>*)(p.dk.at<T>(t, hk) + d) = k4;
  *(V4<T>*)(p.dv.at<T>(t, hk) + d) = v4;
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Opts a kernel into more than 64 KB of LDS, once for each device that is
// current at a launch.
struct Reserved {
  std::atomic<uint64_t> devices{0};
  int operator()(const void* kernel, int bytes, const char* what) {
    if (bytes <= 65536) return MI355X_OK;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == hipSuccess && (devices.load(std::memory_order_relaxed) & bit)) return MI355X_OK;
    if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail(MI355X_ELAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, bytes, hipGetErrorString(e));
    devices.fetch_or(bit, std::memory_order_relaxed);
    return MI355X_OK;
  }
};

struct Launch {
  int64_t sequences, tokens;
  hipStream_t s;
  int64_t cap(int rows) const { return packed_cap(sequences, tokens, rows); }
};

constexpr int64_t kMostThreads = 1ll << 32;

template <typename T, int W, bool RAG, int NW, int QPW, int KH>
int fwd_start(const PackedArgs& a, const Launch& l) {
  constexpr int bytes = 4 * KvLayout<kLayout<W>>::TILE;
  auto k = packed_fwd<T, W, RAG, NW, QPW, KH>;
  static Reserved reserve;
  const int rc = reserve((const void*)k, bytes, "mi355x_packed_attn_fwd");
  if (rc) return rc;
  const int64_t blocks = l.cap(NW / KH * QPW) * a.heads;
  MI_REQUIRE(blocks * 64 * NW < kMostThreads, "mi355x_packed_attn_fwd: %lld blocks", (long long)blocks);
  k<<<(unsigned)blocks, 64 * NW, bytes, l.s>>>(a);
  return check_launch("mi355x_packed_attn_fwd");
}

// Above 128 channels a block fills a CU, with 8 waves of 16 queries: 128 queries
// where that gives 512 blocks, else 64, the keys of a step in two halves (256
// channels, 4096 rows in 3 sequences: 8 heads 71 us and 59, 16 heads 95 and 106;
// 16384 rows in 30, 4 heads, 66 and 82.  Four waves of 32 queries read half as
// much from LDS, one a SIMD: 826 us where 8 take 746 and halves 878).
template <typename T, int W, bool RAG>
int fwd_launch(const PackedArgs& a, const Launch& l) {
  if constexpr (W <= 128) return fwd_start<T, W, RAG, 4, 32, 1>(a, l);
  else if (l.tokens / 128 * a.heads >= 512) return fwd_start<T, W, RAG, 8, 16, 1>(a, l);
  else return fwd_start<T, W, RAG, 8, 16, 2>(a, l);
}

template <typename T, int D>
int sum_launch(const PackedArgs& a, const Launch& l) {
  const int64_t sums = (int64_t)a.kv_heads * a.tokens * (D / 4);
  MI_REQUIRE(sums < kMostThreads - kThreads, "mi355x_packed_attn_bwd: too many rows and heads");
  packed_sum<T, D><<<ceil_div(sums, kThreads), kThreads, 0, l.s>>>(a);
  return check_launch("mi355x_packed_attn_bwd");
}

template <int D>
constexpr int kBwdLds = 2 * (2 * KvLayout<D>::TILE + 512);

template <typename T, int W, bool RAG>
int bwd_launch(PackedArgs a, const Launch& l) {
  constexpr int D = kLayout<W>;
  constexpr bool SPLIT = W == 128;
  auto k0 = packed_bwd<T, W, RAG, SPLIT ? 1 : 0>, k1 = packed_bwd<T, W, RAG, SPLIT ? 2 : 0>, k2 = packed_bwd<T, W, RAG, SPLIT ? 3 : 0>;
  static Reserved reserve0, reserve1, reserve2;
  int rc = reserve0((const void*)k0, kBwdLds<D>, "mi355x_packed_attn_bwd");
  if (!rc) rc = reserve1((const void*)k1, kBwdLds<D>, "mi355x_packed_attn_bwd");
  if (!rc) rc = reserve2((const void*)k2, kBwdLds<D>, "mi355x_packed_attn_bwd");
  if (rc) return rc;
  const int64_t nkv = l.cap(kPackedRows[kKeyList<W>]) * (a.kv_part ? a.heads : a.kv_heads), nq = l.cap(128) * a.heads;
  const int64_t rows = (int64_t)a.heads * a.tokens;
  MI_REQUIRE((nkv + nq) * kThreads < kMostThreads && rows * (D / 4) < kMostThreads - kThreads,
             "mi355x_packed_attn_bwd: too many rows and heads");
  a.all_fine = a.tokens <= kFine || (a.window > 0 && a.window <= kFine);
  packed_delta<T, D><<<ceil_div(rows, kThreads / (D / 8)), kThreads, 0, l.s>>>(a);
  if (SPLIT) {
    if (!a.all_fine) k0<<<(unsigned)nkv, kThreads, kBwdLds<D>, l.s>>>(a, (uint32_t)nkv);
    k2<<<(unsigned)nkv, kThreads, kBwdLds<D>, l.s>>>(a, (uint32_t)nkv);
    k1<<<(unsigned)nq, kThreads, kBwdLds<D>, l.s>>>(a, 0);
  } else {
    k0<<<(unsigned)(nkv + nq), kThreads, kBwdLds<D>, l.s>>>(a, (uint32_t)nkv);
  }
  return a.kv_part ? sum_launch<T, D>(a, l) : check_launch("mi355x_packed_attn_bwd");
}

int layout_of(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
int width_of(int64_t d) { return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

#define MI_PACKED_WIDTH(FN, T, W, a, l) (a).d == W ? FN<T, W, false>(a, l) : FN<T, W, true>(a, l)
#define MI_PACKED(FN, T, a, l)                                   \
  switch (width_of((a).d)) {                                     \
    case 64: return MI_PACKED_WIDTH(FN, T, 64, a, l);            \
    case 96: return MI_PACKED_WIDTH(FN, T, 96, a, l);            \
    case 128: return MI_PACKED_WIDTH(FN, T, 128, a, l);          \
    case 192: return MI_PACKED_WIDTH(FN, T, 192, a, l);          \
    default: return MI_PACKED_WIDTH(FN, T, 256, a, l);           \
  }

int check_shape(const char* what, int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d, double scale,
                int64_t window, int dtype) {
  MI_REQUIRE(sequences >= 0 && sequences < (1ll << 30) && tokens >= 0 && tokens < (1ll << 30) - 1024, "%s: %lld sequences of %lld rows",
             what, (long long)sequences, (long long)tokens);
  MI_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads < 65536, "%s: %lld heads over %lld K/V heads", what,
             (long long)heads, (long long)kv_heads);
  MI_REQUIRE(window >= 0, "%s: window %lld", what, (long long)window);
  MI_REQUIRE(fabs(scale) < 1e38, "%s: scale %g", what, scale);
  if (d <= 0 || d > 256 || d % 8) return fail(MI355X_EUNSUPPORTED, "%s: head_dim %lld (a multiple of 8 up to 256)", what, (long long)d);
  if (dtype != MI355X_BF16 && dtype != MI355X_F16 && dtype != MI355X_F32)
    return fail(MI355X_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  MI_REQUIRE(heads * tokens < (1ll << 31), "%s: heads x rows must be below 2^31", what);
  return MI355X_OK;
}

// Scores are formed as (sign q) k times c > 0, so that a row's maximum can be
// taken before the product with c; without a scale all are 0 and c is not.
void set_scale(PackedArgs& a, double scale) {
  a.scale = (float)scale, a.c = (float)(fabs(scale) * 1.4426950408889634);
  a.sign = a.c < 1e-37f ? 0.f : scale > 0 ? 1.f : -1.f;
  if (a.sign == 0.f) a.c = 1.f;
}

// The f32 kernels' arguments: strides of rows and heads, one batch.
AttnF32 f32_args(const PackedArgs& a) {
  AttnF32 f{};
  f.o = (float*)a.o.p, f.o_s = a.o.row, f.o_h = a.o.head, f.lse = a.lse;
  f.q = (const float*)a.q.p, f.q_s = a.q.row, f.q_h = a.q.head;
  f.k = (const float*)a.k.p, f.k_s = a.k.row, f.k_h = a.k.head;
  f.v = (const float*)a.v.p, f.v_s = a.v.row, f.v_h = a.v.head;
  f.dout = (const float*)a.dout.p, f.do_s = a.dout.row, f.do_h = a.dout.head;
  f.dq = (float*)a.dq.p, f.dq_s = a.dq.row, f.dq_h = a.dq.head;
  f.dk = (float*)a.dk.p, f.dk_s = a.dk.row, f.dk_h = a.dk.head;
  f.dv = (float*)a.dv.p, f.dv_s = a.dv.row, f.dv_h = a.dv.head;
  f.delta = a.ndelta, f.B = 1, f.H = a.heads, f.Sq = f.Skv = a.tokens;
  f.scale = a.scale, f.scale_log2 = a.scale * kLog2e, f.causal = 1, f.group = 1, f.window = a.window;
  f.kv_part = a.kv_part, f.kv_plane = (int64_t)a.heads * a.tokens * layout_of(a.d), f.d = a.d;
  return f;
}

// Rows that are read and written 16 bytes at a time.
bool wide(const void* p, const int64_t* th, size_t es) {
  return p && (uintptr_t)p % 16 == 0 && th[0] * (int64_t)es % 16 == 0 && th[1] * (int64_t)es % 16 == 0 && th[0] >= 0 &&
         th[1] >= 0 && th[0] * (int64_t)es <= kMostRowBytes;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi355x_packed_attn_fwd(void* o, const int64_t* o_th, void* o_low, float* lse, const void* q, const int64_t* q_th,
                                      const void* k, const int64_t* k_th, const void* v, const int64_t* v_th, const void* plan,
                                      int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d,
                                      double scale, int64_t window, int dtype, mi355x_stream_t stream) {
  const char* what = "mi355x_packed_attn_fwd";
  const int rc = check_shape(what, sequences, tokens, heads, kv_heads, d, scale, window, dtype);
  if (rc) return rc;
  if (tokens == 0) return MI355X_OK;
  MI_REQUIRE(lse && plan && (uintptr_t)plan % 16 == 0, "%s: lse or plan missing", what);
  const size_t es = dtype_size(dtype);
  MI_REQUIRE(wide(o, o_th, es) && wide(q, q_th, es) && wide(k, k_th, es) && wide(v, v_th, es) && (uintptr_t)o_low % 16 == 0,
             "%s: rows must be 16-byte aligned, less than 64 MB apart", what);
  PackedArgs a{};
  a.q = {q, q_th[0], q_th[1]}, a.k = {k, k_th[0], k_th[1]}, a.v = {v, v_th[0], v_th[1]}, a.o = {o, o_th[0], o_th[1]};
  a.o_low = o_low, a.lse = lse, a.head = (const PackedHeader*)plan;
  for (int i = 0; i < 2; ++i) a.tiles[i] = packed_list(plan, sequences, tokens, kPackedRows[i]);
  a.tokens = (int)tokens, a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.d = (int)d;
  a.window = (int)std::min<int64_t>(window, tokens);
  set_scale(a, scale);
  const Launch l{sequences, tokens, (hipStream_t)stream};
  if (dtype == MI355X_F32) return attn_f32_packed(f32_args(a), {a.head, a.tiles[1], l.cap(64), (uint32_t)heads, (uint32_t)kv_heads}, false, l.s);
  if (dtype == MI355X_BF16) MI_PACKED(fwd_launch, bf16, a, l);
  MI_PACKED(fwd_launch, f16, a, l);
}

// Whether a K/V head's query heads go to blocks of their own, whose partials are
// added after them.  In f32 always; in 16 bits below two blocks a CU, where one for
// all of a group would leave CUs idle (bf16 forward and backward, one block a group
// against one a head: 16384 rows in 16 sequences, 32 over 2 heads of 64 684 and 584
// us; 8192 rows in 4, 32 over 8 of 128 747 and 844; 16384 in 4, 16 over 4 of 256
// 3533 and 3740).
static bool splits_group(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d, int dtype) {
  return heads > kv_heads && (dtype == MI355X_F32 || (tokens / kPackedRows[d > 192] + 1) * kv_heads < 512);
}

extern "C" int64_t mi355x_packed_attn_bwd_workspace_bytes_for(int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                              int64_t d, int dtype) {
  const int64_t terms = 2 * heads * tokens * (int64_t)sizeof(float) + 512;
  return splits_group(tokens, heads, kv_heads, d, dtype) ? terms + 2 * heads * tokens * layout_of(d) * (int64_t)sizeof(float) : terms;
}

extern "C" int64_t mi355x_packed_attn_bwd_workspace_bytes(int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                          int64_t d) {
  return mi355x_packed_attn_bwd_workspace_bytes_for(sequences, tokens, heads, kv_heads, d, MI355X_F32);
}

extern "C" int mi355x_packed_attn_bwd(void* dq, const int64_t* dq_th, void* dk, const int64_t* dk_th, void* dv,
                                      const int64_t* dv_th, const void* dout, const int64_t* do_th, const void* q,
                                      const int64_t* q_th, const void* k, const int64_t* k_th, const void* v, const int64_t* v_th,
                                      const void* o, const int64_t* o_th, const void* o_low, const float* lse, const void* plan,
                                      int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d,
                                      double scale, int64_t window, int dtype, void* workspace, int64_t ws_bytes,
                                      mi355x_stream_t stream) {
  const char* what = "mi355x_packed_attn_bwd";
  const int rc = check_shape(what, sequences, tokens, heads, kv_heads, d, scale, window, dtype);
  if (rc) return rc;
  if (tokens == 0) return MI355X_OK;
  MI_REQUIRE(lse && plan && (uintptr_t)plan % 16 == 0, "%s: lse or plan missing", what);
  const size_t es = dtype_size(dtype);
  MI_REQUIRE(wide(o, o_th, es) && wide(q, q_th, es) && wide(k, k_th, es) && wide(v, v_th, es) && wide(dout, do_th, es) &&
                 wide(dq, dq_th, es) && wide(dk, dk_th, es) && wide(dv, dv_th, es) && (uintptr_t)o_low % 16 == 0,
             "%s: rows must be 16-byte aligned, less than 64 MB apart", what);
  const int64_t need = mi355x_packed_attn_bwd_workspace_bytes_for(sequences, tokens, heads, kv_heads, d, dtype);
  if (!workspace || ws_bytes < need)
    return fail(MI355X_EWORKSPACE, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes, (long long)need);
  PackedArgs a{};
  a.q = {q, q_th[0], q_th[1]}, a.k = {k, k_th[0], k_th[1]}, a.v = {v, v_th[0], v_th[1]}, a.o = {o, o_th[0], o_th[1]};
  a.dout = {dout, do_th[0], do_th[1]}, a.dq = {dq, dq_th[0], dq_th[1]}, a.dk = {dk, dk_th[0], dk_th[1]}, a.dv = {dv, dv_th[0], dv_th[1]};
  a.o_low = o_low, a.lse = (float*)lse, a.head = (const PackedHeader*)plan;
  for (int i = 0; i < 2; ++i) a.tiles[i] = packed_list(plan, sequences, tokens, kPackedRows[i]);
  a.tokens = (int)tokens, a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.d = (int)d;
  a.window = (int)std::min<int64_t>(window, tokens);
  set_scale(a, scale);
  a.ndelta = (float*)(((uintptr_t)workspace + 15) & ~(uintptr_t)15);
  a.nlse2 = a.ndelta + heads * tokens;
  if (splits_group(tokens, heads, kv_heads, d, dtype))
    a.kv_part = (float*)(((uintptr_t)(a.nlse2 + heads * tokens) + 255) & ~(uintptr_t)255);
  const Launch l{sequences, tokens, (hipStream_t)stream};
  if (dtype == MI355X_F32) {
    const int r = attn_f32_packed(f32_args(a), {a.head, a.tiles[1], l.cap(64), (uint32_t)heads, (uint32_t)kv_heads}, true, l.s);
    if (r || !a.kv_part) return r;
    const int w = layout_of(d);
    return w == 64 ? sum_launch<float, 64>(a, l) : w == 128 ? sum_launch<float, 128>(a, l) : sum_launch<float, 256>(a, l);
  }
  if (dtype == MI355X_BF16) MI_PACKED(bwd_launch, bf16, a, l);
  MI_PACKED(bwd_launch, f16, a, l);
}
