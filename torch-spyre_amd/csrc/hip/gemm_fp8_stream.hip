// 8-bit products of few rows (decode steps), and of K below one block: bound by
// reading W once.
//
//   * A workgroup takes 16 of W's rows and 16 of X's; its 8 waves take the
//     blocks of K in turn (together whole stretches of a row), 4 blocks in flight
//     per wave, straight into registers: the MFMA operand layout is 16 bytes a
//     lane of 16 rows, which loads as it lies.
//   * X's rows past M repeat the last; the matrix cores have an order of
//     magnitude to spare, so one row costs the same as 16.
//   * The waves' sums are added through LDS in a fixed order.
//
// 1 x 4096 x 4096 5.3 us (3.3 at copy rate), 1 x 6144 x 4096 8.0 (4.9), 16 x 4096 x
// 4096 6.5 (operands of three products in turn; with W from memory 5.7, 8.2 and
// 7.0).  From the same sweep: 16 waves of 2 blocks 5.3, 8.0 and 6.9, 32 of W's
// rows a workgroup 6.1, 8.4 and 7.1, 4 waves of 8 blocks 5.9 and 8.5.
#include <type_traits>

#include "gemm_fp8.h"

namespace sph {
namespace {

namespace st8 {
constexpr int NW = 8, U = 4;
}

template <typename T>
__global__ void __launch_bounds__(st8::NW * 64) gemm_fp8_stream_kernel(const Fp8Args p) {
  using namespace st8;
  __shared__ f32x4 red[NW][64];
  const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16, m0 = static_cast<int64_t>(blockIdx.y) * 16;
  const int k = static_cast<int>(p.k), nbf = k / kGroup;
  const int64_t xrow = min(m0 + r16, p.m - 1);
  const uint8_t* wr = p.w + min(n0 + r16, p.n - 1) * p.ldw;
  const uint8_t* xr = p.x + xrow * p.ldx;
  const float* xs = p.xs + xrow * p.xs_row;
  const float* ws = p.ws + n0 / kGroup * p.ws_row;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](i32x8 wf, i32x8 xf, float sc) __attribute__((always_inline)) {
    const f32x4 s = mfma_block(wf, xf);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(s[e], sc, acc[e]);
  };
  auto blocks = [&](int b0, auto nu) __attribute__((always_inline)) {
    constexpr int NU = decltype(nu)::value;
    u32x4 wv[NU][2], xv[NU][2];
    float sx[NU], sw[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        wv[u][h] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4*>(wr + (b0 + u * NW) * kGroup + 16 * g4 + 64 * h));
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        xv[u][h] = *reinterpret_cast<const u32x4*>(xr + (b0 + u * NW) * kGroup + 16 * g4 + 64 * h);
      sx[u] = xs[(b0 + u * NW) * p.xs_blk];
      sw[u] = ws[(b0 + u * NW) * p.ws_blk];
    }
#pragma unroll
    for (int u = 0; u < NU; ++u)
      add(frag(wv[u][0], wv[u][1]), frag(xv[u][0], xv[u][1]), sx[u] * sw[u]);
  };
  int b = wave;
  for (; b + (U - 1) * NW < nbf; b += U * NW) blocks(b, std::integral_constant<int, U>{});
  for (; b < nbf; b += NW) blocks(b, std::integral_constant<int, 1>{});
  if (k % kGroup != 0 && nbf % NW == wave)  // the partial last block
    add(load_frag(wr, nbf, k, g4), load_frag(xr, nbf, k, g4), xs[nbf * p.xs_blk] * ws[nbf * p.ws_blk]);
  red[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
  f32x4 v = red[0][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) v += red[w][lane];
  store_row4<T>(p, m0 + r16, n0 + 4 * g4, v);
}

}  // namespace

int launch_fp8_stream(bool bf16, const Fp8Args& p, hipStream_t st) {
  if (const int rc = fp8::check_grid("sph_gemm_fp8", ceil_div(p.n, 16), st8::NW * 64)) return rc;
  const dim3 grid(static_cast<unsigned>(ceil_div(p.n, 16)), static_cast<unsigned>(ceil_div(p.m, 16)));
  if (bf16)
    gemm_fp8_stream_kernel<bf16_t><<<grid, st8::NW * 64, 0, st>>>(p);
  else
    gemm_fp8_stream_kernel<half_t><<<grid, st8::NW * 64, 0, st>>>(p);
  return check_launch("sph_gemm_fp8");
}

}  // namespace sph
