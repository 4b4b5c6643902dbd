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
#include <algorithm>

#include "gemm_fp8.h"

namespace sph {
namespace {

// ---------------------------------------------------------------------------
// Large products: persistent workgroups, one per CU, over tiles of BN of W's
// rows by 256 of X's, direct global -> LDS loads in the layout of the 16-bit
// direct-load kernel (a row's block of 128 codes is 8 chunks of 16 bytes, chunk c
// of row r at slot c ^ ((r >> 1) & 7)).
//
//   * 8 waves (2 along W's rows, 4 along X's), each TN x 4 MFMA tiles.  A K step
//     is one block: TN * 4 MFMAs of 32 cycles, each followed LAG MFMAs later by
//     its 4 FMAs, so the matrix core runs while the vector ALU scales.
//   * Registers limit the overlap (TN * 16 accumulators of 256), so the
//     fragments are not double-buffered as a whole: W's go through a ring of 4,
//     each slot refilled after its last use; an X fragment is refilled for the
//     next step right after its use by the last row of tiles.
//   * The barrier that hands over the stages comes before MFMA XB, where every
//     fragment of the present stage has been read; after it come the reads of
//     the next stage and the loads of the block after it into the stage just
//     left.  That stream of blocks runs on into the next tile, so a tile's first
//     blocks land while the one before is finished and stored.
//   * A block's scales ride in its stage: waves 0 to 3 fetch X's, 4 and 5 those
//     of W's first 128 rows (of a 192-row tile: its first block), 6 and 7 the
//     next.
//
// 4096 x 25600 x 4096: 417 to 430 us, 2000 to 2060 TFLOP/s.  Bound by the chip's
// power and the tiles' way through LDS together: the clock stands at 2.05 GHz
// (2.35 without the loads), the matrix cores are busy 53 % of it, and of the time
// 90 us go with the direct loads and 48 with the stores (327 and 369 us without);
// matrix instructions and scaling alone reach 3600 TFLOP/s.  X's fragments
// straight from memory to registers, past LDS: 645 us (192-row tiles, 448 as here).
// ---------------------------------------------------------------------------
namespace dl8 {
constexpr int TM = 4, LAG = 2, WN = 2, WM = 4, NW = 8, NT = 512, BM = 256;
template <int TN_>
struct Cfg {
  static constexpr int TN = TN_, WTN = TN * 16, BN = WN * WTN, NMF = TN * TM;
  static constexpr int W_BYTES = BN * kGroup, X_BYTES = BM * kGroup, S_BYTES = NW * 256;
  static constexpr int STAGE = W_BYTES + X_BYTES + S_BYTES;
  static constexpr int LW = W_BYTES / 1024 / NW, LX = X_BYTES / 1024 / NW, L = LW + LX;
  static_assert(LW * NW * 1024 == W_BYTES && LX * NW * 1024 == X_BYTES, "load lines");
  // The barrier: behind the present block's last W fragment (read after row of
  // tiles TN - 5), before the next block's first (read after row TN - 4).
  static constexpr int XB = (TN - 4) * TM + TM - 1;
  static_assert(NMF - XB > L, "loads fit behind the barrier");
  // Tiles of a wave that certainly share W's block: all of 128 rows, pairs of
  // the 96 that begin on multiples of 32 in a block.
  static constexpr int NC = TN == 8 ? 1 : TN / 2, CT = TN / NC;
  static_assert(TN == 8 || TN == 6, "256- or 192-row tiles of W");
};
}  // namespace dl8

template <typename T, int TN_>
__global__ void __launch_bounds__(dl8::NT) gemm_fp8_dl_kernel(const Fp8Args p) {
  using namespace dl8;
  using C = Cfg<TN_>;
  constexpr int TN = C::TN, STAGE = C::STAGE, NMF = C::NMF, BN = C::BN, NC = C::NC;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wn = wave / WM, wm = wave % WM;
  const int k = static_cast<int>(p.k), ldx = static_cast<int>(p.ldx), ldw = static_cast<int>(p.ldw);
  const int ksteps = k / kGroup;  // K is whole blocks, at least 2
  const int ntiles = p.tiles_m * p.tiles_n;
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPH_LDS char*)(lds)));
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
  // Where the load stream stands: its tile's resources and block.
  struct Stream {
    i32x4 rx, rw, rs;
    const float* sb;
    int64_t sblk;
    uint32_t sbytes, vs;
    int t, tile;
  } ld;
  auto open = [&](int tile) __attribute__((always_inline)) {
    int tm, tn;
    tile_of(tile, p.tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
    const int xrows = static_cast<int>(min(static_cast<int64_t>(BM), p.m - m0));
    const int wrows = static_cast<int>(min(static_cast<int64_t>(BN), p.n - n0));
    ld.rx = buffer_rsrc(p.x + m0 * p.ldx, static_cast<uint32_t>((xrows - 1) * ldx + ksteps * kGroup));
    ld.rw = buffer_rsrc(p.w + n0 * p.ldw, static_cast<uint32_t>((wrows - 1) * ldw + ksteps * kGroup));
    if (wave < 4) {
      ld.sb = p.xs + m0 * p.xs_row;
      ld.sblk = p.xs_blk;
      ld.sbytes = (static_cast<uint32_t>(xrows - 1) * static_cast<uint32_t>(p.xs_row) + 1) * 4;
    } else {
      const int64_t b = min(n0 / kGroup + (wave >> 1) - 2, (p.n - 1) / kGroup);
      ld.sb = p.ws + b * p.ws_row;
      ld.sblk = p.ws_blk;
      ld.sbytes = 4;
    }
    ld.t = 0;
    ld.tile = tile;
  };
  // (rows past the last read zeros: their results are not stored)
  const uint32_t vs = wave < 4 ? static_cast<uint32_t>(wave * 64 + lane) * static_cast<uint32_t>(p.xs_row) * 4 : 0;
  // Load line l (W's first; L: the scales) of the stream's block into stage st & 1.
  auto dma = [&](int st, int l) __attribute__((always_inline)) {
    const uint32_t sb = lds_base + (st & 1) * STAGE;
    if (l == C::L) {
      dma4(buffer_rsrc(ld.sb + ld.t * ld.sblk, ld.sbytes),
           __builtin_amdgcn_readfirstlane(sb + C::W_BYTES + C::X_BYTES + wave * 256), vs);
      return;
    }
    const bool is_w = l < C::LW;
    const int h = is_w ? l : l - C::LW, line = wave * (is_w ? C::LW : C::LX) + h;
    uint32_t v = is_w ? vw[h & 1] : vx[h & 1];
    asm volatile("" : "+v"(v));  // the sum below is not worth a register across the loop
    dma16(is_w ? ld.rw : ld.rx,
          __builtin_amdgcn_readfirstlane(sb + (is_w ? 0 : C::W_BYTES) + line * 1024),
          v + (h >> 1) * 16 * (is_w ? ldw : ldx), __builtin_amdgcn_readfirstlane(ld.t * kGroup));
  };
  // On to the next block; past the last tile the last block is loaded again
  // (nobody uses it), so the loop has no branches around loads.
  auto next_block = [&]() __attribute__((always_inline)) {
    if (ld.t + 1 < ksteps)
      ++ld.t;
    else if (ld.tile + static_cast<int>(gridDim.x) < ntiles)
      open(ld.tile + gridDim.x);
  };

  const int sw = (g4 ^ ((r16 >> 1) & 7)) << 4;
  const int woff = (wn * C::WTN + r16) * kGroup, xoff = C::W_BYTES + (wm * 64 + r16) * kGroup;
  auto read = [&](int st, int off, int tile) __attribute__((always_inline)) {
    const char* q = lds + (st & 1) * STAGE + off + tile * 16 * kGroup;
    return frag(*reinterpret_cast<const u32x4*>(q + sw), *reinterpret_cast<const u32x4*>(q + (sw ^ 64)));
  };

  f32x4 acc[TN][TM], P[LAG];
  float sc[NC][TM], xr[TM], wr[NC];
  int wb[NC];  // where the scale of each class of tiles lies
  auto read_scales = [&](int st) __attribute__((always_inline)) {
    const char* q = lds + (st & 1) * STAGE + C::W_BYTES + C::X_BYTES;
#pragma unroll
    for (int j = 0; j < TM; ++j) xr[j] = *reinterpret_cast<const float*>(q + (wm * 64 + 16 * j + r16) * 4);
#pragma unroll
    for (int c = 0; c < NC; ++c) wr[c] = *reinterpret_cast<const float*>(q + wb[c]);
  };
  auto set_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < TM; ++j) sc[c][j] = xr[j] * wr[c];
  };
  auto scale_add = [&](int x) __attribute__((always_inline)) {
    f32x4& a = acc[x / TM][x % TM];
    const f32x4 v = P[x % LAG];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = fmaf(v[e], sc[x / TM / C::CT][x % TM], a[e]);
  };
  // Scales of W's rows of this wave's tiles in the tile that begins at row n0.
  auto place = [&](int64_t n0) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int first = static_cast<int>(n0 % kGroup) + wn * C::WTN + c * C::CT * 16;
      wb[c] = (first < kGroup ? 4 : 6) * 256;
    }
  };

  int tile = blockIdx.x;
  open(tile);
#pragma unroll
  for (int l = 0; l <= C::L; ++l) dma(0, l);
  next_block();
#pragma unroll
  for (int l = 0; l <= C::L; ++l) dma(1, l);
  wait_vmcnt<C::L + 1>();
  __syncthreads();
  i32x8 wf[4], xf[TM];
#pragma unroll
  for (int i = 0; i < 4; ++i) wf[i] = read(0, woff, i);
#pragma unroll
  for (int j = 0; j < TM; ++j) xf[j] = read(0, xoff, j);
  int st = 0, stored = 0;
  for (;;) {
    int tm, tn;
    tile_of(tile, p.tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
    place(n0);
    read_scales(st);
    set_scales();
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int ks = 0; ks < ksteps; ++ks, ++st) {
      next_block();
#pragma unroll
      for (int x = 0; x < NMF; ++x) {
        const int i = x / TM, j = x % TM;
        if (x == C::XB) {
          // this wave's loads of the next block have landed (behind them a
          // tile's first step may still have its predecessor's stores under way)
          asm volatile(
              "s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lstored%=\n\ts_waitcnt vmcnt(0)\n.Lstored%=:\n\t"
              "s_waitcnt vmcnt(%1) lgkmcnt(0)"
              :
              : "s"(__builtin_amdgcn_readfirstlane(stored)), "n"(TN / 2 * TM)
              : "memory", "scc");
          __syncthreads();
        }
        if (x >= LAG) scale_add(x - LAG);
        P[x % LAG] = mfma_block(wf[i & 3], xf[j]);
        // W's tile i + 4 of this block, else the next block's tile of the slot
        if (j == TM - 1)
          wf[i & 3] = i + 4 < TN ? read(st, woff, i + 4) : read(st + 1, woff, i & 3);
        if (i == TN - 1) xf[j] = read(st + 1, xoff, j);
        if (x == NMF - TM - 1) read_scales(st + 1);
        if (x >= C::XB && x - C::XB <= C::L) dma(st, x - C::XB);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int x = NMF - LAG; x < NMF; ++x) scale_add(x);
      set_scales();
      stored = 0;
    }
    // (the lane number anew: addresses of the stores kept over the K loop would
    // cost registers there)
    int l = lane;
    asm volatile("" : "+v"(l));
    store_tiles<T, TN, TM>(p, acc, m0 + wm * (TM * 16), n0 + wn * C::WTN, l & 15, l >> 4);
    tile += gridDim.x;
    if (tile >= ntiles) break;
    // a whole tile's stores are TN / 2 * TM instructions
    stored = m0 + BM <= p.m && n0 + BN <= p.n;
  }
  wait_vmcnt<0>();  // the last loads land before the LDS is given back
}

constexpr int64_t kTileCUs = 256;

template <typename T, int TN>
int launch_dl(Fp8Args p, hipStream_t stream) {
  using C = dl8::Cfg<TN>;
  p.tiles_m = static_cast<int>(ceil_div(p.m, dl8::BM));
  p.tiles_n = static_cast<int>(ceil_div(p.n, C::BN));
  const int grid = std::min<int>(p.tiles_m * p.tiles_n, kTileCUs);
  gemm_fp8_dl_kernel<T, TN><<<grid, dl8::NT, 0, stream>>>(p);
  return check_launch("sph_gemm_fp8");
}

// us of `tiles` 256- (c = 0) or 192-row tiles: the launch, and per round what it
// takes beside its blocks and per block, with few and with all CUs at work (they
// share the chip's power).
double tiles_us(int c, int64_t tiles, int64_t k) {
  constexpr double kLaunch = 0.5, kRound[2] = {5.8, 5.0}, kFew[2] = {1.21, 1.01},
                   kAll[2] = {1.62, 1.36};
  const double nb = static_cast<double>(k / kGroup);
  const int64_t full = tiles / kTileCUs, rest = tiles % kTileCUs;
  double us = kLaunch + static_cast<double>(full) * (kRound[c] + nb * kAll[c]);
  if (rest > 0)
    us += kRound[c] + nb * (kFew[c] + (kAll[c] - kFew[c]) * static_cast<double>(rest) / kTileCUs);
  return us;
}

// us of a streamed product: the launch, what a workgroup takes beside its bytes,
// and the bytes of the fullest CU (W's from memory, X's from the caches).  Fitted to
// 1246 timings of 1 to 70 rows by 64 to 40000 columns, K 128 to 26000, each with W
// from HBM, in which it comes within 1.6 of the fastest kernel (rms error 8 %).
double stream_us(int64_t m, int64_t n, int64_t k) {
  constexpr double kLaunch = 2.33, kWorkgroup = 0.0013, kCuKB = 22.8, kX = 0.47;
  const int64_t wgs = ceil_div(n, 16) * ceil_div(m, 16);
  const double rows = 16 + kX * static_cast<double>(std::min<int64_t>(m, 16));
  return kLaunch + kWorkgroup * static_cast<double>(wgs) +
         static_cast<double>(ceil_div(wgs, kTileCUs) * k) * rows * 1e-3 / kCuKB;
}

// The kernel of a product (one MI355X, W from memory, us).
//   Streamed rows, where one pass of workgroups over 16 rows each of X and W and
// 4 blocks a wave is the whole product: 512 workgroups and K of 4096 at most,
// above 16 rows (W read more than once, from the caches) half of their product.
//     1 x 6144 x 4096 8.2 (ring 9.6), 16 x 4096 x 4096 7.0 (9.0), 16 x 8192 x 4096
//     11.1 (11.4), 16 x 12288 x 4096 15.5 (14.3), 64 x 2048 x 2048 6.3 (7.5), 512 x
//     256 x 4096 10.0 (9.0)
//   Elsewhere too where its fitted time is 5 % below the ring's: of 1494 products of
// up to 70 rows 67 stream by this, 0.73 to 1.12 (on average 0.89) of the time of
// the kernel they had by the limits above and K to 12800 for up to 8 rows:
//     4 x 4096 x 12800 13.5 (ring 16.0), 4 x 4096 x 14336 14.9 (17.6), 1 x 9152 x 1664
//     6.1 (8.3), but 16 x 4096 x 12800 17.5 (16.7) and 4 x 5120 x 12800 22.6 (18.2)
//   Others the kernel whose fitted time is the least:
//     16 x 25600 x 4096 ring 24.3 (streamed 30.8), 333 x 4096 x 12800 ring 38.4 (192-
//     row tiles 131), 2048 x 6144 x 4096 192-row tiles 52.8 (256-row 60.6, ring 76),
//     1500 x 25600 x 4096 256-row tiles 175 (ring 192)
//   Large tiles that would leave most of a last round of workgroups idle take whole
// rounds alone and leave the other rows (or columns) to a second product, where
// the fitted times gain 13 %: 2048 x 25600 x 4096 210, whole 233; 13 such products
// of random sizes took 0.90 to 1.12 (on average 0.97) of the fastest single kernel.
// A rest of few rows or columns that is streamed is counted as nothing: short K,
// where this happens, takes a single kernel longer than fitted (its stores), by more
// than the rest.  Six such splits took 0.90 to 1.04 (on average 0.96) of the fastest
// single kernel, 4100 x 4096 x 256 15.9 and 16.8, 8200 x 4096 x 384 27.7 and 26.6;
// with the rest's time counted, the plan left them to slower kernels (19.2, 38.0).
// With less to gain splitting pays little or nothing: 4096 x 25600 x 4096 410 and 425,
// 1500 x 25600 x 4096 170 and 175, 4000 x 6200 x 2048 65.3 and 66.7, though 2600 x
// 6144 x 4096 74 and 79 (ring).
Fp8Plan fp8_plan(int64_t m, int64_t n, int64_t k, int64_t max_bytes, bool whole = false) {
  const int64_t wgs = ceil_div(n, 16) * ceil_div(m, 16);
  const Fp8Plan stream{Fp8Plan::kStream, 0, 1, 0, 0, stream_us(m, n, k)};
  if (k < kGroup ||
      (wgs <= 512 && k <= 32 * kGroup && wgs * k <= (m <= 16 ? 1 << 21 : 1 << 20)))
    return stream;
  Fp8Plan best = fp8_ring_plan(m, n, k, max_bytes);
  if (stream.us < 0.95 * best.us) best = stream;
  if (k < 2 * kGroup || k % kGroup != 0) return best;
  for (int c = 0; c < 2; ++c) {
    const int64_t bn = c == 0 ? 256 : 192, tm = ceil_div(m, dl8::BM), tn = ceil_div(n, bn);
    const double us = tiles_us(c, tm * tn, k);
    if (us < best.us) best = Fp8Plan{Fp8Plan::kTiles, c, 1, 0, 0, us};
    const int64_t full = tm * tn / kTileCUs * kTileCUs;
    if (whole || full == 0 || full == tm * tn) continue;
    const int64_t unit = c == 0 ? 256 : 384;  // whole tiles and whole blocks of W
    const int64_t n1 = full / tm * bn / unit * unit, m1 = full / tn * dl8::BM;
    for (const bool cols : {true, false}) {
      const int64_t done = cols ? n1 : m1;
      if (done == 0 || done >= (cols ? n : m)) continue;
      const Fp8Plan rest = cols ? fp8_plan(m, n - done, k, max_bytes, true)
                                : fp8_plan(m - done, n, k, max_bytes, true);
      // (a streamed rest counts nothing, see above)
      const double both = tiles_us(c, cols ? tm * (done / bn) : done / dl8::BM * tn, k) +
                          (rest.kernel == Fp8Plan::kStream ? 0 : rest.us);
      if (both < 0.87 * best.us) {
        best = Fp8Plan{Fp8Plan::kTiles, c, 1, 0, rest.bytes, both};
        (cols ? best.n1 : best.m1) = done;
      }
    }
  }
  return best;
}

int launch(bool bf16, const Fp8Args& p, const Fp8Plan& plan, hipStream_t st) {
  if (plan.kernel == Fp8Plan::kStream) return launch_fp8_stream(bf16, p, st);
  if (plan.kernel == Fp8Plan::kRing) return launch_fp8_ring(bf16, p, plan, st);
  if (plan.cfg == 1) return bf16 ? launch_dl<bf16_t, 6>(p, st) : launch_dl<half_t, 6>(p, st);
  return bf16 ? launch_dl<bf16_t, 8>(p, st) : launch_dl<half_t, 8>(p, st);
}

int check_sizes(const char* what, int64_t m, int64_t n, int64_t k) {
  SPH_REQUIRE(k <= INT32_MAX / 512, SPH_ERR_TOO_LARGE, std::string(what) + ": k above 4194303");
  SPH_REQUIRE(m <= 16 * 65535 && n <= INT32_MAX && m * n <= (int64_t{1} << 40), SPH_ERR_TOO_LARGE,
              std::string(what) + ": more than 1048560 rows, 2^31 - 1 columns or 2^40 results");
  return SPH_OK;
}

int run(bool bf16, const Fp8Args& p, int64_t max_bytes, hipStream_t st) {
  const Fp8Plan plan = fp8_plan(p.m, p.n, p.k, max_bytes);
  if (plan.m1 == 0 && plan.n1 == 0) return launch(bf16, p, plan, st);
  Fp8Args first = p, rest = p;
  if (plan.n1 > 0) {
    first.n = plan.n1;
    rest.n -= plan.n1;
    rest.w += plan.n1 * p.ldw;
    rest.ws += plan.n1 / kGroup * p.ws_row;
    if (p.bias != nullptr) rest.bias = static_cast<const uint16_t*>(p.bias) + plan.n1;
    rest.d = static_cast<uint16_t*>(p.d) + plan.n1;
  } else {
    first.m = plan.m1;
    rest.m -= plan.m1;
    rest.x += plan.m1 * p.ldx;
    rest.xs += plan.m1 * p.xs_row;
    rest.d = static_cast<uint16_t*>(p.d) + plan.m1 * p.ldd;
  }
  if (const int rc = launch(bf16, first, plan, st)) return rc;
  return launch(bf16, rest, fp8_plan(rest.m, rest.n, rest.k, max_bytes, true), st);
}

}  // namespace
}  // namespace sph

using namespace sph;

extern "C" int64_t sph_gemm_fp8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || check_sizes("sph_gemm_fp8", m, n, k) != SPH_OK) return 0;
  return fp8_plan(m, n, k, INT64_MAX).bytes;
}

extern "C" int sph_gemm_fp8_plan(int64_t m, int64_t n, int64_t k, int64_t workspace_bytes,
                                 int32_t* plan) {
  SPH_REQUIRE(m > 0 && n > 0 && k > 0 && plan != nullptr, SPH_ERR_INVALID_ARG,
              "sph_gemm_fp8_plan: sizes must be positive");
  if (const int rc = check_sizes("sph_gemm_fp8_plan", m, n, k)) return rc;
  const Fp8Plan p = fp8_plan(m, n, k, workspace_bytes);
  const Fp8Tile t = p.kernel == Fp8Plan::kStream  ? Fp8Tile{16, 16, 4}
                    : p.kernel == Fp8Plan::kRing ? fp8_ring_tile(p.cfg)
                                                 : Fp8Tile{dl8::BM, p.cfg == 0 ? 256 : 192, 1};
  plan[0] = p.kernel;
  plan[1] = t.m;
  plan[2] = t.n;
  plan[3] = p.splits;
  plan[4] = t.per_cu;
  plan[5] = static_cast<int32_t>(p.n1 > 0 ? p.n1 : p.m1);
  plan[6] = p.n1 > 0 ? 1 : p.m1 > 0 ? 2 : 0;
  return SPH_OK;
}

extern "C" int sph_gemm_fp8(sph_dtype dtype, int64_t m, int64_t n, int64_t k, const void* x,
                            int64_t ldx, const float* x_scale, int64_t x_scale_row_stride,
                            int64_t x_scale_group_stride, const void* w, int64_t ldw,
                            const float* w_scale, int64_t w_scale_row_stride,
                            int64_t w_scale_group_stride, const void* bias, void* d, int64_t ldd,
                            void* workspace, int64_t workspace_bytes, sph_stream_t stream) {
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
  if (const int rc = check_sizes("sph_gemm_fp8", m, n, k)) return rc;
  SPH_REQUIRE(ldx <= INT32_MAX / 512 && ldw <= INT32_MAX / 512, SPH_ERR_TOO_LARGE,
              "sph_gemm_fp8: ldx or ldw above 4194303");
  SPH_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, SPH_ERR_UNSUPPORTED,
              "sph_gemm_fp8: workspace must be 16-byte aligned");
  SPH_REQUIRE(m == 1 || k == 0 || x_scale_row_stride <= (1 << 21), SPH_ERR_TOO_LARGE,
              "sph_gemm_fp8: x_scale_row_stride above 2097152");
  Fp8Args p{};
  p.m = m;
  p.n = n;
  p.k = k;
  p.x = static_cast<const uint8_t*>(x);
  p.ldx = ldx;
  p.xs = x_scale;
  p.xs_row = x_scale_row_stride;
  p.xs_blk = x_scale_group_stride;
  p.w = static_cast<const uint8_t*>(w);
  p.ldw = ldw;
  p.ws = w_scale;
  p.ws_row = w_scale_row_stride;
  p.ws_blk = w_scale_group_stride;
  p.bias = bias;
  p.d = d;
  p.ldd = ldd;
  p.whole_lines = reinterpret_cast<uintptr_t>(d) % 128 == 0 && ldd % 64 == 0;
  p.splits = 1;
  p.part = static_cast<float*>(workspace);
  return run(dtype == SPH_BF16, p, workspace != nullptr ? workspace_bytes : 0, as_stream(stream));
}
