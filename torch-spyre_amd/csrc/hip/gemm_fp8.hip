// Products of OCP e4m3 codes with a scale for each block of 128, on gfx950's
// 8-bit matrix cores:
//
//   D[i, j] = sum_b xs[i, b] ws[j / 128, b] sum_{p in block b} X[i, p] W[j, p] + bias[j]
//
// v_mfma_f32_16x16x128_f8f6f4 takes one whole block of K, so its fp32 result is
// the inner sum; one FMA per element then scales it and adds it to the fp32
// accumulator.  W is the MFMA's first operand: a lane then holds 4 consecutive
// columns j of one row i, all its elements of a 16-row tile share one scale
// xs[i, b] ws[j / 128, b], and that product is one multiplication per tile.
#include "fp8_common.h"
#include "gemm_tile.h"

namespace sph {
namespace {

using fp8::kGroup;

typedef int i32x8 __attribute__((ext_vector_type(8)));

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
  int tiles_m, tiles_n;
};

__device__ inline i32x8 frag(u32x4 lo, u32x4 hi) {
  return __builtin_shufflevector(__builtin_bit_cast(i32x4, lo), __builtin_bit_cast(i32x4, hi), 0, 1,
                                 2, 3, 4, 5, 6, 7);
}

// (Scale operands of 0 select the unscaled form of the instruction.)
__device__ inline f32x4 mfma_block(i32x8 a, i32x8 b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0,
                                                          0, 0, 0);
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

// ---------------------------------------------------------------------------
// Large products: tiles of BN of W's rows by 256 of X's, direct global -> LDS
// loads, the layout of the 16-bit direct-load kernel (a row's block of 128
// codes is 8 chunks of 16 bytes, chunk c of row r at slot c ^ ((r >> 1) & 7)).
//
//   * 8 waves (2 along W's rows, 4 along X's), each TN x 4 MFMA tiles.  A K step
//     is one block: TN * 4 MFMAs of 32 cycles, each followed LAG MFMAs later by
//     its 4 FMAs, so the matrix core runs while the vector ALU scales.
//   * Registers, not LDS, limit the overlap (TN * 16 accumulators of 256), so
//     the fragments are not double-buffered as a whole: W's go through a ring
//     of 4, each slot refilled after its last use; an X fragment is refilled
//     for the next step right after its use by the last row of tiles.
//   * The barrier that hands over the stages comes before MFMA XB, where every
//     fragment of the present stage has been read; after it come the reads of
//     the next stage and the loads of the block after it into the stage just
//     left.
//   * Scales come by ordinary loads, two steps ahead, and are multiplied
//     right behind the barrier's wait, so that the wait which the compiler adds
//     for them finds nothing left in flight.
// ---------------------------------------------------------------------------
namespace dl8 {
constexpr uint32_t kOutside = 0x80000000u;  // past every buffer resource
constexpr int TM = 4, LAG = 2;
template <int TN_, int WN_, int WM_>
struct Cfg {
  static constexpr int TN = TN_, WN = WN_, WM = WM_, NW = WN * WM, NT = NW * 64;
  static constexpr int WTN = TN * 16, BN = WN * WTN, BM = WM * TM * 16, NMF = TN * TM;
  static constexpr int W_BYTES = BN * kGroup, X_BYTES = BM * kGroup, STAGE = W_BYTES + X_BYTES;
  static constexpr int LW = W_BYTES / 1024 / NW, LX = X_BYTES / 1024 / NW, L = LW + LX;
  static_assert(LW * NW * 1024 == W_BYTES && LX * NW * 1024 == X_BYTES, "load lines");
  static constexpr int XB = (TN - 3) * TM;  // the last W fragment is read 4 MFMAs before
  static_assert(NMF - XB >= L, "loads fit behind the barrier");
  static constexpr int SP = WTN + 8;  // epilogue pitch (elements)
  static_assert(NW * 16 * SP * 2 <= 2 * STAGE, "epilogue slabs fit");
};
}  // namespace dl8

template <typename T, int TN_, int WN_, int WM_>
__global__ void __launch_bounds__(WN_ * WM_ * 64) gemm_fp8_dl_kernel(const Fp8Args p) {
  using namespace dl8;
  using C = Cfg<TN_, WN_, WM_>;
  constexpr int TN = C::TN, STAGE = C::STAGE, NMF = C::NMF, WM = C::WM, BM = C::BM, NT = C::NT;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  int tm, tn;
  tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wn = wave / WM, wm = wave % WM, r16 = lane & 15, g4 = lane >> 4;
  const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * C::BN;
  const int k = static_cast<int>(p.k), ldx = static_cast<int>(p.ldx), ldw = static_cast<int>(p.ldw);
  const int ksteps = k / kGroup;  // whole blocks
  const int xrows = static_cast<int>(min(static_cast<int64_t>(BM), p.m - m0));
  const int wrows = static_cast<int>(min(static_cast<int64_t>(C::BN), p.n - n0));
  const i32x4 rx = buffer_rsrc(p.x + m0 * p.ldx, static_cast<uint32_t>((xrows - 1) * ldx + ksteps * kGroup));
  const i32x4 rw = buffer_rsrc(p.w + n0 * p.ldw, static_cast<uint32_t>((wrows - 1) * ldw + ksteps * kGroup));
  // Lane offsets of this wave's load lines (8 rows of 8 chunks each) 0 and 1;
  // lines two apart differ by 16 rows.  Rows past the last lie outside the
  // resource.
  uint32_t vw[2], vx[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int rw_ = (wave * C::LW + i) * 8 + (lane >> 3), rx_ = (wave * C::LX + i) * 8 + (lane >> 3);
    vw[i] = static_cast<uint32_t>(rw_ * ldw + (((lane & 7) ^ ((rw_ >> 1) & 7)) << 4));
    vx[i] = static_cast<uint32_t>(rx_ * ldx + (((lane & 7) ^ ((rx_ >> 1) & 7)) << 4));
  }
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPH_LDS char*)(lds)));
  // Load line l (W's first) of block t into stage st & 1.
  auto dma = [&](int t, int st, int l) __attribute__((always_inline)) {
    const uint32_t sb = lds_base + (st & 1) * STAGE;
    const bool is_w = l < C::LW;
    const int h = is_w ? l : l - C::LW, line = wave * (is_w ? C::LW : C::LX) + h;
    dma16(is_w ? rw : rx,
          __builtin_amdgcn_readfirstlane(sb + (is_w ? 0 : C::W_BYTES) + line * 1024),
          (is_w ? vw[h & 1] : vx[h & 1]) + (h >> 1) * 16 * (is_w ? ldw : ldx),
          __builtin_amdgcn_readfirstlane(t * kGroup));
  };
  const int sw = (g4 ^ ((r16 >> 1) & 7)) << 4;
  const int woff = (wn * C::WTN + r16) * kGroup, xoff = C::W_BYTES + (wm * 64 + r16) * kGroup;
  auto read = [&](int st, int off, int tile) __attribute__((always_inline)) {
    const char* q = lds + (st & 1) * STAGE + off + tile * 16 * kGroup;
    return frag(*reinterpret_cast<const u32x4*>(q + sw), *reinterpret_cast<const u32x4*>(q + (sw ^ 64)));
  };
  // Scales: this lane's row of each X tile, and the wave's block of W.
  const float* xsb = p.xs + m0 * p.xs_row;
  uint32_t xso[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j)
    xso[j] = static_cast<uint32_t>(min(wm * 64 + 16 * j + r16, xrows - 1)) * static_cast<uint32_t>(p.xs_row);
  const int64_t wblk = min((n0 + wn * C::WTN) / kGroup, (p.n - 1) / kGroup);
  const float* wsb = p.ws + wblk * p.ws_row;
  int zero;  // keeps the load of W's scale off the scalar unit, whose waits would cover LDS reads
  asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
  float xr[TM], wr, sc[TM];
  auto load_scales = [&](int t) __attribute__((always_inline)) {
    t = min(t, ksteps - 1);
#pragma unroll
    for (int j = 0; j < TM; ++j) xr[j] = (xsb + t * p.xs_blk)[xso[j]];
    wr = (wsb + t * p.ws_blk)[zero];
  };

  f32x4 acc[TN][TM], P[LAG];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto scale_add = [&](int x) __attribute__((always_inline)) {
    f32x4& a = acc[x / TM][x % TM];
    const f32x4 v = P[x % LAG];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = fmaf(v[e], sc[x % TM], a[e]);
  };

  load_scales(0);
#pragma unroll
  for (int l = 0; l < C::L; ++l) dma(0, 0, l);
  if (ksteps > 1) {
#pragma unroll
    for (int l = 0; l < C::L; ++l) dma(1, 1, l);
    wait_vmcnt<C::L>();
  } else {
    wait_vmcnt<0>();
  }
#pragma unroll
  for (int j = 0; j < TM; ++j) sc[j] = xr[j] * wr;
  load_scales(1);
  __syncthreads();
  i32x8 wf[4], xf[TM];
#pragma unroll
  for (int i = 0; i < 4; ++i) wf[i] = read(0, woff, i);
#pragma unroll
  for (int j = 0; j < TM; ++j) xf[j] = read(0, xoff, j);

  for (int ks = 0; ks < ksteps; ++ks) {
    const int tnext = min(ks + 2, ksteps - 1);
#pragma unroll
    for (int x = 0; x < NMF; ++x) {
      const int i = x / TM, j = x % TM;
      if (x == C::XB) {
        wait_vmcnt<0>();
        wait_lgkmcnt0();
#pragma unroll
        for (int q = 0; q < TM; ++q) {
          xr[q] *= wr;
          asm volatile("" : "+v"(xr[q]));
        }
        __syncthreads();
      }
      if (x >= LAG) scale_add(x - LAG);
      P[x % LAG] = mfma_block(wf[i & 3], xf[j]);
      // W's tile i + 4 of this block, else the next block's tile of the slot
      if (j == TM - 1)
        wf[i & 3] = i + 4 < TN ? read(ks, woff, i + 4) : read(ks + 1, woff, i & 3);
      if (i == TN - 1) xf[j] = read(ks + 1, xoff, j);
      if (x >= C::XB && x - C::XB < C::L) dma(tnext, ks, x - C::XB);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int x = NMF - LAG; x < NMF; ++x) scale_add(x);
#pragma unroll
    for (int q = 0; q < TM; ++q) sc[q] = xr[q];
    load_scales(ks + 2);
  }

  // A partial last block: straight from memory.
  if (k % kGroup != 0) {
    i32x8 xt[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int64_t row = m0 + min(wm * 64 + 16 * j + r16, xrows - 1);
      xt[j] = load_frag(p.x + row * p.ldx, ksteps, k, g4);
      sc[j] = (xsb + ksteps * p.xs_blk)[xso[j]] * (wsb + ksteps * p.ws_blk)[0];
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const int64_t row = n0 + min(wn * C::WTN + 16 * i + r16, wrows - 1);
      const i32x8 wt = load_frag(p.w + row * p.ldw, ksteps, k, g4);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        P[0] = mfma_block(wt, xt[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(P[0][e], sc[j], acc[i][j][e]);
      }
    }
  }

  // Lane: columns 4 g4 .. + 3 of W tile i, row r16 of X tile j.  16 rows at a
  // time through the wave's own LDS slab, so that stores cover whole lines.
  wait_vmcnt<0>();
  wait_lgkmcnt0();
  __syncthreads();
  constexpr int SP = C::SP, CPO = C::WTN / 8;
  T* slab = reinterpret_cast<T*>(lds) + wave * (16 * SP);
  const T* bias = static_cast<const T*>(p.bias);
  T* D = static_cast<T*>(p.d);
  const int64_t col0 = n0 + wn * C::WTN, row0 = m0 + wm * (TM * 16);
  if (bias != nullptr) {
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t col = col0 + 16 * i + 4 * g4 + e;
        if (col < p.n) b[e] = Num<T>::to_f(bias[col]);
      }
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] += b[e];
    }
  }
#pragma unroll
  for (int j = 0; j < TM; ++j) {
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      u32x2 v;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        v[e] = pack2<T>(acc[i][j][2 * e], acc[i][j][2 * e + 1]);
      *reinterpret_cast<u32x2*>(slab + r16 * SP + 16 * i + 4 * g4) = v;
    }
    wait_lgkmcnt0();
#pragma unroll
    for (int q = lane; q < 16 * CPO; q += 64) {
      const int rr = q / CPO, cc = (q % CPO) * 8;
      const int64_t row = row0 + 16 * j + rr, col = col0 + cc;
      if (row >= p.m || col >= p.n) continue;
      const u32x4 v = *reinterpret_cast<const u32x4*>(slab + rr * SP + cc);
      T* dp = D + row * p.ldd + col;
      if (col + 8 <= p.n) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(dp));
      } else {
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (col + c < p.n) dp[c] = e[c];
      }
    }
    wait_lgkmcnt0();
  }
}

// A wave computes 16 columns of W's rows by 64 rows of X, straight from memory.
template <typename T>
__global__ void __launch_bounds__(256) gemm_fp8_kernel(const Fp8Args p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g4 = lane >> 4;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 64;
  if (n0 >= p.n) return;
  const uint8_t* wr = p.w + min(n0 + r16, p.n - 1) * p.ldw;
  const uint8_t* xr[4];
  const float* xs[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = min(m0 + 16 * j + r16, p.m - 1);
    xr[j] = p.x + row * p.ldx;
    xs[j] = p.xs + row * p.xs_row;
  }
  const float* ws = p.ws + n0 / kGroup * p.ws_row;
  const int64_t nb = (p.k + kGroup - 1) / kGroup;
  f32x4 acc[4] = {};
  for (int64_t b = 0; b < nb; ++b) {
    const i32x8 wf = load_frag(wr, b, p.k, g4);
    const float wscale = ws[b * p.ws_blk];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 s = mfma_block(wf, load_frag(xr[j], b, p.k, g4));
      const float sc = xs[j][b * p.xs_blk] * wscale;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(s[e], sc, acc[j][e]);
    }
  }
  const T* bias = static_cast<const T*>(p.bias);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = m0 + 16 * j + r16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t col = n0 + 4 * g4 + e;
      if (row < p.m && col < p.n)
        static_cast<T*>(p.d)[row * p.ldd + col] =
            Num<T>::from_f(acc[j][e] + (bias ? Num<T>::to_f(bias[col]) : 0.f));
    }
  }
}

template <typename T, int TN, int WN, int WM>
int launch_dl(Fp8Args p, hipStream_t stream) {
  using C = dl8::Cfg<TN, WN, WM>;
  p.tiles_m = static_cast<int>(ceil_div(p.m, C::BM));
  p.tiles_n = static_cast<int>(ceil_div(p.n, C::BN));
  gemm_fp8_dl_kernel<T, TN, WN, WM><<<p.tiles_m * p.tiles_n, C::NT, 0, stream>>>(p);
  return check_launch("sph_gemm_fp8");
}

template <typename T>
int launch(const Fp8Args& p, hipStream_t stream) {
  if (p.k >= kGroup && p.m > 128) return launch_dl<T, 8, 2, 4>(p, stream);
  const dim3 grid(static_cast<uint32_t>(ceil_div(p.n, 64)), static_cast<uint32_t>(ceil_div(p.m, 64)));
  gemm_fp8_kernel<T><<<grid, 256, 0, stream>>>(p);
  return check_launch("sph_gemm_fp8");
}

}  // namespace
}  // namespace sph

using namespace sph;

extern "C" int64_t sph_gemm_fp8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  (void)m, (void)n, (void)k;
  return 0;
}

extern "C" int sph_gemm_fp8(sph_dtype dtype, int64_t m, int64_t n, int64_t k, const void* x,
                            int64_t ldx, const float* x_scale, int64_t x_scale_row_stride,
                            int64_t x_scale_group_stride, const void* w, int64_t ldw,
                            const float* w_scale, int64_t w_scale_row_stride,
                            int64_t w_scale_group_stride, const void* bias, void* d, int64_t ldd,
                            void* workspace, int64_t workspace_bytes, sph_stream_t stream) {
  (void)workspace, (void)workspace_bytes;
  SPH_REQUIRE(m >= 0 && n >= 0 && k >= 0, SPH_ERR_INVALID_ARG, "sph_gemm_fp8: negative size");
  SPH_REQUIRE(dtype == SPH_F16 || dtype == SPH_BF16, SPH_ERR_UNSUPPORTED,
              "sph_gemm_fp8: dtype must be F16 or BF16");
  if (m == 0 || n == 0) return SPH_OK;
  SPH_REQUIRE(d != nullptr, SPH_ERR_INVALID_ARG, "sph_gemm_fp8: null output");
  SPH_REQUIRE(m == 1 || ldd >= n, SPH_ERR_INVALID_ARG, "sph_gemm_fp8: ldd is less than n");
  if (k > 0) {
    SPH_REQUIRE(x != nullptr && w != nullptr && x_scale != nullptr && w_scale != nullptr,
                SPH_ERR_INVALID_ARG, "sph_gemm_fp8: null operand");
    SPH_REQUIRE((m == 1 || ldx >= k) && (n == 1 || ldw >= k), SPH_ERR_INVALID_ARG,
                "sph_gemm_fp8: ldx or ldw is less than k");
    SPH_REQUIRE(x_scale_row_stride >= 0 && x_scale_group_stride >= 0 && w_scale_row_stride >= 0 &&
                    w_scale_group_stride >= 0,
                SPH_ERR_INVALID_ARG, "sph_gemm_fp8: negative scale stride");
    SPH_REQUIRE((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) % 16 == 0 &&
                    (m == 1 || ldx % 16 == 0) && (n == 1 || ldw % 16 == 0),
                SPH_ERR_UNSUPPORTED, "sph_gemm_fp8: rows of x and w must be 16-byte aligned");
  }
  SPH_REQUIRE(k <= INT32_MAX / 512 && ldx <= INT32_MAX / 512 && ldw <= INT32_MAX / 512,
              SPH_ERR_TOO_LARGE, "sph_gemm_fp8: k, ldx or ldw above 4194303");
  SPH_REQUIRE(m <= INT32_MAX && n <= INT32_MAX, SPH_ERR_TOO_LARGE,
              "sph_gemm_fp8: m or n above 2^31 - 1");
  SPH_REQUIRE(ceil_div(m, 64) <= 65535, SPH_ERR_TOO_LARGE, "sph_gemm_fp8: too many rows");
  Fp8Args p{m,
                  n,
                  k,
                  static_cast<const uint8_t*>(x),
                  ldx,
                  x_scale,
                  x_scale_row_stride,
                  x_scale_group_stride,
                  static_cast<const uint8_t*>(w),
                  ldw,
                  w_scale,
                  w_scale_row_stride,
                  w_scale_group_stride,
                  bias,
                  d,
                  ldd,
                  0,
                  0};
  const hipStream_t st = as_stream(stream);
  return dtype == SPH_F16 ? launch<half_t>(p, st) : launch<bf16_t>(p, st);
}
