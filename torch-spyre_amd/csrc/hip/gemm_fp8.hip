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
#include "gemm_common.h"

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

// 16 codes at row[p], zeros from K on.  `row` and p are multiples of 16 bytes,
// so a chunk that begins inside the row is read whole: it cannot leave the page.
__device__ inline u32x4 load_chunk(const uint8_t* row, int64_t p, int64_t k) {
  if (p >= k) return zero4();
  u32x4 v = *reinterpret_cast<const u32x4*>(row + p);
  if (p + 16 > k) {
    const int left = static_cast<int>(k - p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int nb = left - 4 * i;
      v[i] = nb >= 4 ? v[i] : nb <= 0 ? 0u : v[i] & ((1u << (8 * nb)) - 1u);
    }
  }
  return v;
}

// The operand of block b for 16 rows: lane l holds row l % 16, chunks l / 16
// and l / 16 + 4 of the block (any order of K serves that both operands share).
__device__ inline i32x8 load_frag(const uint8_t* row, int64_t b, int64_t k, int g4) {
  const int64_t p = b * kGroup + 16 * g4;
  return frag(load_chunk(row, p, k), load_chunk(row, p + 64, k));
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
  const Fp8Args p{m,
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
                  ldd};
  const dim3 grid(static_cast<uint32_t>(ceil_div(n, 64)), static_cast<uint32_t>(ceil_div(m, 64)));
  if (dtype == SPH_F16)
    gemm_fp8_kernel<half_t><<<grid, 256, 0, as_stream(stream)>>>(p);
  else
    gemm_fp8_kernel<bf16_t><<<grid, 256, 0, as_stream(stream)>>>(p);
  return check_launch("sph_gemm_fp8");
}
