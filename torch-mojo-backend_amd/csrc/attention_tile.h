// What the attention kernels of 16-bit types on matrix cores share
// (attention.hip, attention_packed.hip): the layout of tiles in LDS, their loads
// and transposing reads, and reductions over a wave's lane groups.
#pragma once
#include "attention_window.h"
#include "common.h"
#include "mfma.h"

#ifndef ATTN_ASM_DMA
#define ATTN_ASM_DMA 1
#endif

namespace mi {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ typename Mfma<T>::frag zero_frag() {
  typename Mfma<T>::frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
  return f;
}

// Reductions over the four 16-lane groups of a wave (the key rows of an
// S^T tile): v_permlane16_swap / v_permlane32_swap with both operands = x
// leave x's partner row (lane +-16, then +-32) in the second result.
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
// 2^x on the transcendental unit (results below 2^-126 flush to zero, which
// softmax weights never miss).
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

typedef const void __attribute__((address_space(1)))* gptr_t;
typedef void __attribute__((address_space(3)))* lptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int D>
struct KvLayout {
  static constexpr int ROWB = D * 2;          // bytes per row
  static constexpr int CH = D / 8;            // 16-byte chunks per row
  static constexpr int TILE = 64 * ROWB;      // one 64-row tile
  static constexpr int RPI = 1024 / ROWB;     // rows per 1 KB load instruction
  // Chunk swizzle of row r, chosen from LDS bank-conflict counter
  // measurements of the two read patterns: 16-byte fragment reads (16
  // consecutive rows at one chunk) and ds_read_b64_tr_b16 reads (rows
  // 4g + j, adjacent chunks c, c ^ 1).  Both run without bank conflicts.
  //   D = 64 (128-byte rows):  r & 7
  //   D = 128 (256-byte rows): bit 0 = r3, bits 1-2 = r0-r1, bit 3 = r2 ^ r3
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (D == 256) return row & 15;  // 512-byte rows: 16 rows at one chunk hit 16 bank groups
    return D == 64 ? (row & 7)
                   : (((row >> 3) & 1) | ((row & 3) << 1) | ((((row >> 2) ^ (row >> 3)) & 1) << 3));
  }
  // byte offset of element (row, col) in a swizzled tile
  static __device__ __forceinline__ int off(int row, int col) {
    return row * ROWB + (((col >> 3) ^ swz(row)) << 4) + ((col & 7) << 1);
  }
};

__host__ __device__ inline int64_t ceil_div64(int64_t a, int64_t b) { return a <= 0 ? 0 : (a + b - 1) / b; }


template <bool B>
struct BoolTag {
  static constexpr bool value = B;
};

// This lane's byte offsets of tr_frag's reads at tile row 0, one per
// head-dim block dt.  Row t0*16 + r has the swizzle of r (it uses only the
// row's low four bits), so tr_frag(tile, dt, t0, t1) reads tile +
// t0*16*ROWB + o[dt] and tile + t1*16*ROWB + o[dt]: with the offsets kept
// in registers the per-step address arithmetic folds into immediates.
template <int D>
struct TrOffsets {
  int o[D / 16];
  __device__ __forceinline__ TrOffsets() {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, src = lane & 15;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[dt] = KvLayout<D>::off(4 * g + (src >> 2), dt * 16 + 4 * (src & 3));
  }
};

template <typename T, int D>
__device__ __forceinline__ typename Mfma<T>::frag tr_frag_at(const char* tile, const TrOffsets<D>& to, int dt,
                                                             int t0, int t1) {
  constexpr int RB = 16 * KvLayout<D>::ROWB;
  s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + t0 * RB + to.o[dt]));
  s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + t1 * RB + to.o[dt]));
  typename Mfma<T>::frag f;
  short* fs = (short*)&f;
#pragma unroll
  for (int e = 0; e < 4; ++e) fs[e] = a[e], fs[4 + e] = b[e];
  return f;
}

// Tile loader (K/V in the forward and dQ pass, Q/dO in the dK/dV pass):
// each thread's byte offsets within a full tile are computed once, so a tile
// costs one scalar row-offset product plus one 64-bit add per load (a 64-bit
// vector multiply per load, as recomputing them would take, runs at a
// quarter of the VALU rate).  Rows past the end (only in the last tile)
// reload the last row; their scores are masked.
template <int D, int NW>
struct KvTileLoad {
  typedef KvLayout<D> L;
  static constexpr int IT = L::TILE / 1024 / NW;  // 1 KB load instructions per thread
  const char* g;
  int64_t rs;
  int64_t off[IT];   // r * rs + chunk * 16
  static __device__ __forceinline__ int row_of(int it) {
    return (it * NW + wave_id()) * L::RPI + (int)(threadIdx.x & 63) / L::CH;
  }
  static __device__ __forceinline__ int coff_of(int row) {
    return (((int)(threadIdx.x & 63) % L::CH) ^ L::swz(row)) * 16;
  }
  __device__ __forceinline__ void init(const char* base, int64_t rs_bytes) {
    g = base;
    rs = rs_bytes;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int r = row_of(it);
      off[it] = r * rs + coff_of(r);
    }
  }
  __device__ __forceinline__ void issue(int64_t row0, int64_t nrows, char* dst) const {
    const int wave = wave_id();
    if (row0 + 64 <= nrows) {
      const char* tb = g + row0 * rs;
#pragma unroll
      for (int it = 0; it < IT; ++it) load(tb + off[it], dst + (it * NW + wave) * 1024);
    } else {
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int r = row_of(it);
        const int64_t gr = min(row0 + r, nrows - 1);
        load(g + gr * rs + coff_of(r), dst + (it * NW + wave) * 1024);
      }
    }
  }
  static __device__ __forceinline__ void load(const char* src, char* dst) {
#if ATTN_ASM_DMA
    dma_b128(src, lds_base_of(dst));
#else
    __builtin_amdgcn_global_load_lds((gptr_t)src, (lptr_t)dst, 16, 0, 0);
#endif
  }
};

// How far a row's maximum may exceed the softmax's reference before that moves.
constexpr float kSlack = 8.f;

}  // namespace
}  // namespace mi
