// 8-bit products whose rows do not fill the CUs with 256-row tiles: decode
// batches, short and ragged prompts.
//
//   * Tiles of BM of X's rows by BN of W's on 4 or 8 waves (2 along X's rows), one
//     to three workgroups per CU; a ring of ST LDS stages of KB blocks of K each,
//     ST - 1 of them in flight (direct loads, 128 codes a row, chunk c of row r
//     at slot c ^ ((r >> 1) & 7)).
//   * The blocks' scales ride in the same stage by one 4-byte load per lane: the
//     first waves fetch X's, the others W's (one value), so they are covered by
//     the same wait and barrier and need no registers in flight.
//   * K is split over workgroups until the chip is full: fp32 sums in a caller's
//     workspace, added in a fixed order by a second kernel.
//
// A step of one block costs a small tile some 600 cycles of latency (wait,
// barrier, LDS, MFMA, FMA) whatever its size, so the small tiles take two blocks
// a step (256 x 4096 x 4096 in 32 x 64 tiles 12.1 us, 15.1 with one) and the
// larger ones 8 waves (777 x 6144 x 4096 in 128 x 128 tiles 32.0 us, 39.8 on 4).
// Few rows are bound by reading W (24 x 49155 x 4096 45 us, 39.7 at copy rate), the
// others by what is in flight into LDS (333 x 4096 x 12800 34.6 us: 9.5 TB/s from
// the caches, the matrix cores busy 21 %).  (Operands of three products in turn, so
// in part from the caches; with W from memory 256 x 4096 x 4096 17.4, 777 x 6144 x
// 4096 35.9, 333 x 4096 x 12800 38.4.)  Asking for W's lines three or six
// steps ahead made all of them slower (44.8 and 43.5 us in the run whose time
// without was 38.6), 192 x 128 and 256 x 128 tiles no faster (35.2, 40.7).
#include <algorithm>

#include "gemm_fp8.h"

namespace sph {
namespace {

namespace ring8 {
constexpr uint32_t kOutside = 0x80000000u;  // past every buffer resource

template <int BM_, int BN_, int NW_, int KB_, int ST_>
struct Cfg {
  static constexpr int BM = BM_, BN = BN_, KB = KB_, ST = ST_, NW = NW_, WN = NW / 2, WTM = BM / 2, WTN = BN / WN;
  static constexpr int TM = WTM / 16, TN = WTN / 16;
  static constexpr int X_BYTES = BM * kGroup, W_BYTES = BN * kGroup, S_BYTES = NW * 256;
  static constexpr int BLK = X_BYTES + W_BYTES + S_BYTES, STAGE = KB * BLK;
  static constexpr int LX = X_BYTES / 1024 / NW, LW = W_BYTES / 1024 / NW, LB = LX + LW + 1, L = KB * LB;
  static constexpr int XSW = (BM + 63) / 64;  // waves that fetch X's scales
  static_assert(LX * NW * 1024 == X_BYTES && LW * NW * 1024 == W_BYTES, "load lines");
  static_assert(XSW < NW && BN <= kGroup && TN % 2 == 0, "scales, one block of W, tile pairs");
  static_assert((ST - 2) * L < 64, "vmcnt range");
};
}  // namespace ring8

template <int ST, int L>
__device__ inline void wait_blocks(int blocks) {
  static_assert(ST <= 4, "at most two blocks in flight behind the one awaited");
  if constexpr (ST >= 4) {
    if (blocks >= 2) return wait_vmcnt<2 * L>();
  }
  if constexpr (ST >= 3) {
    if (blocks >= 1) return wait_vmcnt<L>();
  }
  wait_vmcnt<0>();
}

template <typename T, int BM_, int BN_, int NW_, int KB_, int ST_>
__global__ void __launch_bounds__(NW_ * 64) gemm_fp8_ring_kernel(const Fp8Args p) {
  using C = ring8::Cfg<BM_, BN_, NW_, KB_, ST_>;
  constexpr int BM = C::BM, BN = C::BN, KB = C::KB, ST = C::ST, TM = C::TM, TN = C::TN;
  __shared__ __attribute__((aligned(1024))) char lds[ST * C::STAGE];
  // Workgroup -> (tile, K slice): a contiguous run per XCD, row tiles of one
  // panel of W next to each other.
  int id = blockIdx.x;
  {
    const int total = gridDim.x, q = total >> 3, r = total & 7, x = id & 7;
    id = x * q + min(x, r) + (id >> 3);
  }
  const int tm = id % p.tiles_m;
  id /= p.tiles_m;
  const int split = id % p.splits, tn = id / p.splits;
  const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
  const int k = static_cast<int>(p.k), nbf = k / kGroup;
  const int kb0 = split * p.kslice, nblk = min(p.kslice, nbf - kb0), ksteps = (nblk + KB - 1) / KB;
  const int ldx = static_cast<int>(p.ldx), ldw = static_cast<int>(p.ldw);
  const int xrows = static_cast<int>(min(static_cast<int64_t>(BM), p.m - m0));
  const int wrows = static_cast<int>(min(static_cast<int64_t>(BN), p.n - n0));
  const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = wave / C::WN, wn = wave % C::WN;
  const i32x4 rx = buffer_rsrc(p.x + m0 * p.ldx, static_cast<uint32_t>((xrows - 1) * ldx + nbf * kGroup));
  const i32x4 rw = buffer_rsrc(p.w + n0 * p.ldw, static_cast<uint32_t>((wrows - 1) * ldw + nbf * kGroup));
  uint32_t vx[C::LX], vw[C::LW];
#pragma unroll
  for (int i = 0; i < C::LX; ++i) {
    const int r = (wave * C::LX + i) * 8 + (lane >> 3);
    vx[i] = r < xrows ? static_cast<uint32_t>(r * ldx + (((lane & 7) ^ ((r >> 1) & 7)) << 4)) : ring8::kOutside;
  }
#pragma unroll
  for (int i = 0; i < C::LW; ++i) {
    const int r = (wave * C::LW + i) * 8 + (lane >> 3);
    vw[i] = r < wrows ? static_cast<uint32_t>(r * ldw + (((lane & 7) ^ ((r >> 1) & 7)) << 4)) : ring8::kOutside;
  }
  // Scales: this wave's source, step per block, and lane offset.
  const bool sx = wave < C::XSW;
  const float* sbase = sx ? p.xs + m0 * p.xs_row : p.ws + n0 / kGroup * p.ws_row;
  const int64_t sblk = sx ? p.xs_blk : p.ws_blk;
  const uint32_t sbytes = sx ? (static_cast<uint32_t>(xrows - 1) * static_cast<uint32_t>(p.xs_row) + 1) * 4 : 4;
  const uint32_t vs = sx ? static_cast<uint32_t>(min(wave * 64 + lane, xrows - 1)) * static_cast<uint32_t>(p.xs_row) * 4 : 0;
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPH_LDS char*)(lds)));

  auto issue = [&](int t, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const uint32_t sb = lds_base + slot * C::STAGE + b * C::BLK;
      const int kb = min(kb0 + t * KB + b, nbf - 1);  // (a block past the slice is not used)
#pragma unroll
      for (int i = 0; i < C::LX; ++i)
        dma16(rx, __builtin_amdgcn_readfirstlane(sb + (wave * C::LX + i) * 1024), vx[i],
              __builtin_amdgcn_readfirstlane(kb * kGroup));
#pragma unroll
      for (int i = 0; i < C::LW; ++i)
        dma16(rw, __builtin_amdgcn_readfirstlane(sb + C::X_BYTES + (wave * C::LW + i) * 1024), vw[i],
              __builtin_amdgcn_readfirstlane(kb * kGroup));
      dma4(buffer_rsrc(sbase + kb * sblk, sbytes),
           __builtin_amdgcn_readfirstlane(sb + C::X_BYTES + C::W_BYTES + wave * 256), vs);
    }
  };

  const int sw = (g4 ^ ((r16 >> 1) & 7)) << 4;
  const int xoff = (wm * C::WTM + r16) * kGroup, woff = C::X_BYTES + (wn * C::WTN + r16) * kGroup;
  const int soff = C::X_BYTES + C::W_BYTES;
  f32x4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int t = 0; t < ST - 1 && t < ksteps; ++t) issue(t, t);
  int slot = 0;
  for (int ks = 0; ks < ksteps; ++ks) {
    // block ks has landed once only later blocks' loads are outstanding; the
    // barrier also means that every wave is done with the slot of block ks - 1
    wait_blocks<ST, C::L>(min(ST - 2, ksteps - 1 - ks));
    wait_lgkmcnt0();
    __syncthreads();
    if (ks + ST - 1 < ksteps) issue(ks + ST - 1, slot == 0 ? ST - 1 : slot - 1);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      if (b > 0 && ks * KB + b >= nblk) break;
      const char* sp = lds + slot * C::STAGE + b * C::BLK;
      const float wsc = *reinterpret_cast<const float*>(sp + soff + (C::NW - 1) * 256);
      float sc[TM];
      i32x8 xf[TM], wf[TN];
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        sc[j] = *reinterpret_cast<const float*>(sp + soff + (wm * C::WTM + 16 * j + r16) * 4) * wsc;
        const char* q = sp + xoff + j * 16 * kGroup;
        xf[j] = frag(*reinterpret_cast<const u32x4*>(q + sw), *reinterpret_cast<const u32x4*>(q + (sw ^ 64)));
      }
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const char* q = sp + woff + i * 16 * kGroup;
        wf[i] = frag(*reinterpret_cast<const u32x4*>(q + sw), *reinterpret_cast<const u32x4*>(q + (sw ^ 64)));
      }
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const f32x4 s = mfma_block(wf[i], xf[j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(s[e], sc[j], acc[i][j][e]);
        }
    }
    slot = slot + 1 == ST ? 0 : slot + 1;
  }

  const int64_t row0 = m0 + wm * C::WTM, col0 = n0 + wn * C::WTN;
  if (k % kGroup != 0 && split == p.splits - 1) {  // the partial last block
    const int64_t xbase = m0 + xrows - 1, wbase = n0 + wrows - 1;
    i32x8 xf[TM];
    float sc[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int64_t row = min(row0 + 16 * j + r16, xbase);
      xf[j] = load_frag(p.x + row * p.ldx, nbf, k, g4);
      sc[j] = p.xs[row * p.xs_row + nbf * p.xs_blk] * p.ws[n0 / kGroup * p.ws_row + nbf * p.ws_blk];
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const i32x8 wf = load_frag(p.w + min(col0 + 16 * i + r16, wbase) * p.ldw, nbf, k, g4);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const f32x4 s = mfma_block(wf, xf[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(s[e], sc[j], acc[i][j][e]);
      }
    }
  }
  if (p.splits == 1) return store_tiles<T, TN, TM>(p, acc, row0, col0, r16, g4);
  const int64_t pitch = (p.n + 3) & ~static_cast<int64_t>(3);
  float* W = p.part + static_cast<int64_t>(split) * p.m * pitch;
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int64_t col = col0 + 16 * i + 4 * g4;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int64_t row = row0 + 16 * j + r16;
      if (row < p.m && col < pitch) *reinterpret_cast<f32x4*>(W + row * pitch + col) = acc[i][j];
    }
  }
}

// Adds the K slices' sums in slice order, then bias: 4 columns a thread.
template <typename T>
__global__ void __launch_bounds__(256) gemm_fp8_reduce(const Fp8Args p) {
  const int64_t nq = (p.n + 3) >> 2, idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (idx >= p.m * nq) return;
  const int64_t row = idx / nq, col = (idx - row * nq) * 4, step = p.m * nq * 4;
  const float* W = p.part + row * nq * 4 + col;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) v += *reinterpret_cast<const f32x4*>(W + s * step);
  store_row4<T>(p, row, col, v);
}

template <typename T, int BM, int BN, int NW, int KB, int ST>
int launch_ring8(Fp8Args& p, hipStream_t st) {
  p.tiles_m = static_cast<int>(ceil_div(p.m, BM));
  p.tiles_n = static_cast<int>(ceil_div(p.n, BN));
  const int64_t grid = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  if (const int rc = fp8::check_grid("sph_gemm_fp8", grid, NW * 64)) return rc;
  gemm_fp8_ring_kernel<T, BM, BN, NW, KB, ST><<<static_cast<unsigned>(grid), NW * 64, 0, st>>>(p);
  if (p.splits > 1)
    gemm_fp8_reduce<T><<<static_cast<unsigned>(ceil_div(p.m * ceil_div(p.n, 4), 256)), 256, 0, st>>>(p);
  return check_launch("sph_gemm_fp8");
}

// Tile configurations: per_cu workgroups share a CU (LDS), each with `fly` blocks
// in flight; us of a round of workgroups beside its blocks of K, of the launch,
// and per block of K with 1, 2 or 3 workgroups on the CU; us of the reduce's
// launch and TB/s of its sums; TB/s of the tiles' traffic from the caches and of
// the operands from memory.  Fitted to 7300 timings of 1 to 4400 rows by 256 to
// 49155 columns, K 256 to 25600, 1 to 16 slices, the weights of most of them read
// from HBM as a model's layers are (rms error 6 to 8 %).  The plan that the fitted
// times choose is 2 % slower than the fastest kernel and slices of a product on
// average over 1494 products of up to 70 rows and 490 of few columns (30 % at most:
// 12 x 4046 x 22672; 16 x 4096 x 12800 14 %, 16.7 us in 5 slices and 14.6 in 8), 3 %
// over 420 of 200 to 9000 rows and K to 2600 (50 % at most: 5904 x 7360 x 256, whose
// stores the rounds of small tiles leave out).
struct RingCfg {
  int bm, bn, kb, per_cu, fly;
  double round, launch, blk[3], reduce, sums, traffic, mem;
};
constexpr RingCfg kRing[] = {
    {32, 64, 2, 3, 2, 0.32, 2.2, {0.378, 0.511, 0.53}, 2.9, 4.1, 33.0, 5.14},
    {64, 128, 1, 2, 2, 0.1, 3.36, {0.439, 0.818, 0}, 2.45, 5.3, 15.4, 5.5},
    {128, 128, 1, 2, 1, 2.1, 1.8, {0.852, 1.11, 0}, 2.5, 6.1, 15.2, 5.0},
    {128, 128, 1, 1, 2, 2.2, 2.2, {0.578, 0, 0}, 2.4, 5.6, 10.9, 5.5}};
constexpr int kRingCfgs = sizeof(kRing) / sizeof(kRing[0]);

template <typename T>
int launch_cfg(Fp8Args& p, int cfg, hipStream_t st) {
  switch (cfg) {
    case 0: return launch_ring8<T, 32, 64, 4, 2, 2>(p, st);
    case 1: return launch_ring8<T, 64, 128, 8, 1, 3>(p, st);
    case 2: return launch_ring8<T, 128, 128, 8, 1, 2>(p, st);
    default: return launch_ring8<T, 128, 128, 8, 1, 3>(p, st);
  }
}

}  // namespace

Fp8Plan fp8_ring_plan(int64_t m, int64_t n, int64_t k, int64_t max_bytes) {
  Fp8Plan best;
  best.us = 1e30;
  constexpr int64_t kCUs = 256;
  const int64_t nbf = k / kGroup, pitch = (n + 3) / 4 * 4;
  const double mem_mb = static_cast<double>(m * k + n * k + 2 * m * n) * 1e-6;
  for (int c = 0; c < kRingCfgs; ++c) {
    const RingCfg& f = kRing[c];
    // (up to 32 rows no 128-row tiles: 4 x 25600 x 4096 27.8 us, 26.9 in 64-row tiles)
    if (m <= 32 && f.bm > 64) continue;
    const int64_t tiles = ceil_div(m, f.bm) * ceil_div(n, f.bn), slots = kCUs * f.per_cu;
    for (int s = 1; s <= 16; ++s) {
      // at least 2 blocks a slice, no more slices than two rounds hold
      if (s > 1 && (tiles * s > 2 * slots || nbf < 2 * s)) break;
      const int64_t slice = ceil_div(nbf, s);
      if (ceil_div(nbf, slice) != s) continue;  // every slice has blocks
      const int64_t bytes = s > 1 ? s * m * pitch * 4 : 0;
      if (bytes > max_bytes) continue;
      const int64_t wgs = tiles * s, full = wgs / slots, rest = wgs % slots;
      const double blocks = static_cast<double>(ceil_div(slice, f.kb) * f.kb);
      // a round is no faster than the caches serve its tiles, the whole no faster
      // than what is in flight arrives (1.3 us) and the operands come from memory
      const double block_bytes = static_cast<double>((f.bm + f.bn) * kGroup);
      const auto served = [&](int64_t w) {
        return static_cast<double>(w * slice) * block_bytes / (f.traffic * 1e6);
      };
      double us = static_cast<double>(full) *
                  std::max(f.round + blocks * f.blk[f.per_cu - 1], served(slots));
      if (rest > 0)
        us += std::max(0.7 * f.round + blocks * f.blk[(rest - 1) / kCUs], served(rest));
      const double fly = static_cast<double>(std::min(wgs, slots) * f.fly) * block_bytes;
      us = std::max({us, static_cast<double>((m + n) * k) / fly * 1.3, mem_mb / f.mem});
      us += f.launch;
      if (s > 1) us += f.reduce + 2.0 * static_cast<double>(bytes) / (f.sums * 1e6);
      if (us < best.us) {
        best.kernel = Fp8Plan::kRing;
        best.cfg = c;
        best.splits = s;
        best.kslice = static_cast<int>(slice);
        best.bytes = bytes;
        best.us = us;
      }
    }
  }
  return best;
}

Fp8Tile fp8_ring_tile(int cfg) { return {kRing[cfg].bm, kRing[cfg].bn, kRing[cfg].per_cu}; }

int launch_fp8_ring(bool bf16, Fp8Args p, const Fp8Plan& plan, hipStream_t st) {
  p.splits = plan.splits;
  p.kslice = plan.kslice;
  return bf16 ? launch_cfg<bf16_t>(p, plan.cfg, st) : launch_cfg<half_t>(p, plan.cfg, st);
}

}  // namespace sph
