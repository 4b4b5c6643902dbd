// What the kernels of the 8-bit products share: the call's arguments, the
// matrix instruction and fragments read straight from memory.
#pragma once

#include "fp8_common.h"
#include "gemm_tile.h"

namespace sph {

struct Fp8Args {
  int64_t m, n, k;
  const uint8_t* x;
  int64_t ldx;
  const float* xs;
  int64_t xs_row, xs_blk;
  const uint8_t* w;
  int64_t ldw;
  const float* ws;
  int64_t ws_row, ws_blk;
  const void* bias;
  void* d;
  int64_t ldd;
  int whole_lines;  // every row of d begins on 128 bytes
  int tiles_m, tiles_n;
  // K split: `splits` workgroups of kslice blocks each per tile, fp32 sums of
  // split s at part + s * m * pitch (pitch: n rounded up to 4).
  int splits, kslice;
  float* part;
};

// Tiles and K slices of a product (host).
struct Fp8Plan {
  enum Kernel { kStream = SPH_FP8_STREAM, kRing = SPH_FP8_RING, kTiles = SPH_FP8_TILES } kernel = kStream;
  int cfg = 0, splits = 1, kslice = 0;
  int64_t bytes = 0;  // of workspace
  double us = 0;
  // where not 0: this plan's columns (rows); the others are a product of their own
  int64_t n1 = 0, m1 = 0;
};
struct Fp8Tile {
  int m, n, per_cu;
};
int launch_fp8_stream(bool bf16, const Fp8Args& p, hipStream_t st);
Fp8Plan fp8_ring_plan(int64_t m, int64_t n, int64_t k, int64_t max_bytes);
Fp8Tile fp8_ring_tile(int cfg);
int launch_fp8_ring(bool bf16, Fp8Args p, const Fp8Plan& plan, hipStream_t st);

namespace {

using fp8::kGroup;

typedef int i32x8 __attribute__((ext_vector_type(8)));


__device__ inline i32x8 frag(u32x4 lo, u32x4 hi) {
  return __builtin_shufflevector(__builtin_bit_cast(i32x4, lo), __builtin_bit_cast(i32x4, hi), 0, 1,
                                 2, 3, 4, 5, 6, 7);
}

// (Scale operands of 0 select the unscaled form of the instruction.)
__device__ inline f32x4 mfma_block(i32x8 a, i32x8 b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0,
                                                          0, 0, 0);
}

// 4 bytes per lane from rsrc[voff] into LDS at lds_addr + 4 * lane, with the five
// wait states that a resource just written by a vector instruction takes: its
// base moves with every block.
__device__ inline void dma4(i32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds_addr), "v"(voff), "s"(rsrc)
               : "memory", "m0");
}

// v with zeros from byte `left` on.
__device__ inline u32x4 keep_bytes(u32x4 v, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int nb = left - 4 * i;
    v[i] &= nb >= 4 ? ~0u : nb <= 0 ? 0u : (1u << (8 * nb)) - 1u;
  }
  return v;
}

template <typename T>
__device__ inline uint32_t pack2(float a, float b) {
  return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, Num<T>::from_f(a))) |
         (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, Num<T>::from_f(b))) << 16);
}

// 16 codes at row[p], zeros from K on.  `row` and p are multiples of 16 bytes,
// so a chunk that begins inside the row is read whole: it cannot leave the page.
__device__ inline u32x4 load_chunk(const uint8_t* row, int64_t p, int64_t k) {
  const u32x4 v = *reinterpret_cast<const u32x4*>(row + (p < k ? p : 0));
  return keep_bytes(v, static_cast<int>(k - p));
}

// The operand of block b for 16 rows: lane l holds row l % 16, chunks l / 16
// and l / 16 + 4 of the block (any order of K serves that both operands share).
__device__ inline i32x8 load_frag(const uint8_t* row, int64_t b, int64_t k, int g4) {
  const int64_t p = b * kGroup + 16 * g4;
  return frag(load_chunk(row, p, k), load_chunk(row, p + 64, k));
}

// 8 consecutive results of one row, the last row piece element by element.
template <typename T>
__device__ inline void store_row8(const Fp8Args& p, int64_t row, int64_t col, u32x4 v) {
  if (row >= p.m || col >= p.n) return;
  T* dp = static_cast<T*>(p.d) + row * p.ldd + col;
  if (col + 8 <= p.n) {
    if (p.whole_lines)
      __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(dp));
    else
      *reinterpret_cast<u32x4_any*>(dp) = v;
  } else {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (col + c < p.n) dp[c] = e[c];
  }
}

// Four consecutive results of one row, with bias.
template <typename T>
__device__ inline void store_row4(const Fp8Args& p, int64_t row, int64_t col, f32x4 v) {
  if (row >= p.m || col >= p.n) return;
  const T* bias = static_cast<const T*>(p.bias);
  T* dp = static_cast<T*>(p.d) + row * p.ldd + col;
  const int nc = static_cast<int>(min(static_cast<int64_t>(4), p.n - col));
  if (bias != nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < nc) v[e] += Num<T>::to_f(bias[col + e]);
  }
  if (nc == 4) {
    typedef u32x2 u32x2_any2 __attribute__((aligned(2)));
    *reinterpret_cast<u32x2_any2*>(dp) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < nc) dp[e] = Num<T>::from_f(v[e]);
  }
}

// A wave's tiles, with bias, to D: tile (i, j) holds columns col0 + 16 i + 4 g4
// .. + 3 of row row0 + 16 j + r16 in lane 16 g4 + r16.  v_permlane16_swap
// exchanges the odd 16-lane rows of one tile with the even ones of the next, so
// that a lane holds 8 consecutive columns and a store covers 64 bytes of a row,
// without LDS or a barrier.  Rows that begin on cache lines (128 bytes) leave by
// streaming stores (4096 x 16384 x 4096 in 256-row tiles 267 us without, 249 with);
// other rows need the cache to join their pieces (4000 x 6200 x 2048 86 us with,
// 61 without; 24 x 49155 x 4096 50 and 43).
template <typename T, int TN, int TM>
__device__ inline void store_tiles(const Fp8Args& p, f32x4 (&acc)[TN][TM], int64_t row0,
                                   int64_t col0, int r16, int g4) {
  static_assert(TN % 2 == 0, "tiles go out in pairs");
  const T* bias = static_cast<const T*>(p.bias);
#pragma unroll
  for (int i = 0; i < TN; i += 2) {
    f32x4 b[2] = {};
    if (bias != nullptr) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t col = col0 + 16 * (i + h) + 4 * g4 + e;
          b[h][e] = col < p.n ? Num<T>::to_f(bias[col]) : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const f32x4 u = acc[i][j] + b[0], w = acc[i + 1][j] + b[1];
      const auto lo = __builtin_amdgcn_permlane16_swap(pack2<T>(u[0], u[1]), pack2<T>(w[0], w[1]), false, false);
      const auto hi = __builtin_amdgcn_permlane16_swap(pack2<T>(u[2], u[3]), pack2<T>(w[2], w[3]), false, false);
      store_row8<T>(p, row0 + 16 * j + r16, col0 + 16 * (i + (g4 & 1)) + 8 * (g4 >> 1),
                    u32x4{lo[0], hi[0], lo[1], hi[1]});
    }
  }
}

}  // namespace
}  // namespace sph
