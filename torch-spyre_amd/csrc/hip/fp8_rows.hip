// Rows to OCP e4m3 codes with one fp32 scale per group of 128 columns
// (gfx950): plain values, RMSNorm (with the residual's addition) and
// silu(gate) * up, each in one pass over its inputs.
//
// A group's scale is s = amax / 448 with amax = max(max |v|, 2^-100) and its
// codes are e4m3(v * (448 / amax)), rounded to nearest even by
// v_cvt_pk_fp8_f32.  |v| * (448 / amax) is at most 448 (1 + 2^-22), below the
// 464 from which that instruction would give NaN, so nothing is clamped.  A
// group that holds an infinity or a NaN gets it as its scale.
//
// All of them are bound by memory: 16 lanes hold a group, 8 columns each (one
// 16-byte load of 16-bit values, one 8-byte store of codes), and the largest
// magnitude goes over the 16 lanes by DPP, without LDS.  At the rate of a large
// copy (5.14 TB/s) and here, operands from memory: 4096 x 12800 in blocks 30.6 and
// 30.7 us (of fp32 51.0 and 45.6), 8192 x 4096 to codes 19.6 and 21.4, to norm and
// codes 19.6 and 30.7, with residual 45.7 and 49.8, silu of 2048 x 12800 25.5 and
// 27.5, of 8192 x 4096 32.6 and 33.5.
#include "fp8_common.h"

namespace sph {
namespace {

using fp8::kGroup;
using fp8::kLeastBits;
using fp8::kTop;

constexpr int kLanes = kGroup / 8;  // lanes of a group

typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// Columns [c0, c0 + 8) of a row, zeros from `cols` on.
template <typename T>
__device__ inline void load_cols(const T* __restrict__ row, int64_t c0, int64_t cols,
                                 float (&v)[8]) {
  if (c0 + 8 <= cols) {
    load8u<T>(row + c0, v);
  } else {
    const int n = c0 < cols ? static_cast<int>(cols - c0) : 0;
    load8_partial<T>(row + c0, n, 0.f, v);
  }
}

__device__ inline uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ inline uint32_t amax8(const float (&v)[8]) {
  uint32_t m = mag(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max(m, mag(v[i]));
  return m;
}

// Largest over the 16 lanes of a group (a DPP row): neighbours, pairs, then
// the mirrored half row and row.
template <int CTRL>
__device__ inline uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
__device__ inline uint32_t group_max(uint32_t m) {
  m = max(m, dpp<0xB1>(m));   // quad_perm 1 0 3 2
  m = max(m, dpp<0x4E>(m));   // quad_perm 2 3 0 1
  m = max(m, dpp<0x141>(m));  // row_half_mirror
  return max(m, dpp<0x140>(m));  // row_mirror
}

// The codes of 8 values, v * r each.
__device__ inline uint2 codes8(const float (&v)[8], float r) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * r, v[1] * r, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * r, v[3] * r, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * r, v[5] * r, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * r, v[7] * r, hi, true);
  return make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}

__device__ inline void store_codes(uint8_t* __restrict__ row, int64_t c0, int64_t cols, uint2 w) {
  if (c0 + 8 <= cols) {
    // (streaming: 4096 x 12800 in blocks 33.8 us without, 30.7 with)
    __builtin_nontemporal_store(u32x2_any{w.x, w.y}, reinterpret_cast<u32x2_any*>(row + c0));
  } else {
    const uint64_t b = (static_cast<uint64_t>(w.y) << 32) | w.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < cols) row[c0 + i] = static_cast<uint8_t>(b >> (8 * i));
  }
}

// Where the codes and scales go: row r's codes at q + r * ldq, the scale of its
// group g at scale + r * sr + g * sg.
struct Out {
  uint8_t* q;
  int64_t ldq;
  float* scale;
  int64_t sr, sg;
};

// What a group is made of: plain values, or silu(gate) * up with up `cols`
// columns behind gate.
template <typename T>
struct Values {
  const T* x;
  int64_t ld;
  __device__ inline void load(int64_t row, int64_t c0, int64_t cols, float (&v)[8]) const {
    load_cols<T>(x + row * ld, c0, cols, v);
  }
};

// silu(g) = g / (1 + t) for g >= 0, g t / (1 + t) below, t = exp(-|g|) = 2^n 2^f, n + f =
// -|g| log2(e), n whole: f keeps its relative precision for large |g| (log2(e) in two
// parts), and the divisor stays in [1, 2].  (As g / (1 + exp(-g)) 1.5 % faster, but
// the reciprocal flushes subnormal results: 0 from g = -87.3 on.)  The division is a
// reciprocal (1 ulp) and one correction by its remainder; without it values near a
// tie fall to the other code twice as often, for 3 % of the time of 2048 x 12800;
// the library's expf and an IEEE division cost 22 %.
__device__ inline float silu_fast(float g) {
  const float c = fminf(fabsf(g), 150.f);  // (past 150 t is 0 in fp32)
  const float n = rintf(c * -1.44269502f);
  const float f = fmaf(c, -1.92596299e-8f, fmaf(c, -1.44269502f, -n));
  const float t = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n));
  const float a = g < 0.f ? g * t : g;
  const float d = 1.f + t, r = __builtin_amdgcn_rcpf(d);
  return a * fmaf(fmaf(-d, r, 1.f), r, r);
}

template <typename T>
struct SiluMul {
  const T* x;
  int64_t ld;
  __device__ inline void load(int64_t row, int64_t c0, int64_t cols, float (&v)[8]) const {
    float u[8];
    load_cols<T>(x + row * ld, c0, cols, v);
    load_cols<T>(x + row * ld + cols, c0, cols, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = silu_fast(v[i]) * u[i];
  }
};

// Groups of 1 x 128.  A wave takes one group of 4 consecutive rows, a workgroup
// 16 rows, so the scales that it writes lie side by side where a group's scales
// of all rows do (sr = 1).  (Two groups a wave with their loads ahead: 5 % slower.)
// Workgroups go along a row's groups first: with operands from memory 8192 x 4096 to
// codes 21.4 us, 24.0 with the rows first; silu of 2048 x 12800 27.5 and 29.3, of
// 8192 x 4096 33.5 and 41.2; from the caches the same up to 2048 x 12800 (23.2 and
// 23.4), 42.8 and 41.6 at 4096 x 12800.
template <typename S>
__global__ void __launch_bounds__(256) fp8_groups_kernel(S src, Out o, int64_t rows, int64_t cols) {
  const int l16 = threadIdx.x % kLanes, r16 = threadIdx.x / kLanes;
  const int64_t g = blockIdx.x, nr = (rows + 15) / 16;
  for (int64_t rb = blockIdx.y; rb < nr; rb += gridDim.y) {
    const int64_t row = rb * 16 + r16, c0 = g * kGroup + l16 * 8;
    if (row >= rows) return;
    float v[8];
    src.load(row, c0, cols, v);
    const float amax = __uint_as_float(max(group_max(amax8(v)), kLeastBits));
    store_codes(o.q + row * o.ldq, c0, cols, codes8(v, kTop / amax));
    if (l16 == 0) o.scale[row * o.sr + g * o.sg] = amax / kTop;
  }
}

// Blocks of 128 x 128: a workgroup holds one block in registers (8 passes of
// 16 rows) between finding its largest magnitude and rounding it.
template <typename T>
__global__ void __launch_bounds__(256) fp8_blocks_kernel(Values<T> src, Out o, int64_t rows,
                                                         int64_t cols) {
  __shared__ uint32_t red[4];
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kGroup + threadIdx.x % kLanes * 8;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kGroup + threadIdx.x / kLanes;
  float v[8][8];
  uint32_t m = kLeastBits;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (r0 + 16 * i < rows) {
      src.load(r0 + 16 * i, c0, cols, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
    m = max(m, amax8(v[i]));
  }
  m = group_max(m);
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16)));
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32)));
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = m;
  __syncthreads();
  const float amax = __uint_as_float(max(max(red[0], red[1]), max(red[2], red[3])));
  const float r = kTop / amax;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (r0 + 16 * i < rows) store_codes(o.q + (r0 + 16 * i) * o.ldq, c0, cols, codes8(v[i], r));
  if (threadIdx.x == 0) o.scale[blockIdx.y * o.sr + blockIdx.x * o.sg] = amax / kTop;
}

// ---------------------------------------------------------------------------
// RMSNorm to codes.  y = h * rstd * w with rstd = rsqrt(mean(h^2) + eps) > 0,
// one number for the row, so amax|y| = rstd * amax|h w| and the codes,
// e4m3(y * 448 / amax|y|) = e4m3(h w * (448 / amax|h w|)), do not depend on
// rstd: they are formed while the sum of squares is still under way, and only
// the scales wait for it.  h w of two 16-bit values is exact in fp32.
// ---------------------------------------------------------------------------
struct NormArgs {
  const void *x, *residual, *w;
  void* h;
  int64_t ldx, ldr, ldh;
  int64_t rows, cols;
  float eps;
  Out o;
};

// h = x + residual r of columns [c0, c0 + 8), rounded to T and stored.
template <typename T>
__device__ inline void add_residual(const NormArgs& p, int64_t row, int64_t c0, bool store,
                                    const float (&r)[8], float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = Num<T>::to_f(Num<T>::from_f(v[j] + r[j]));
  if (!store) return;
  T* hp = static_cast<T*>(p.h) + row * p.ldh + c0;
  if (c0 + 8 <= p.cols)
    store8u<T>(hp, v);
  else
    store8_partial<T>(hp, c0 < p.cols ? static_cast<int>(p.cols - c0) : 0, v);
}

template <typename W>
__device__ inline void times_weight(const NormArgs& p, int64_t c0, float (&v)[8]) {
  if (p.w == nullptr) return;
  float w[8];
  load_cols<W>(static_cast<const W*>(p.w), c0, p.cols, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= w[j];
}

// Consecutive rows to one XCD (workgroups go round over the 8): the scales of a
// group lie row by row, and a line of them is then merged in one L2.
__device__ inline int64_t row_block(int64_t blocks) {
  const int64_t id = blockIdx.x, q = blocks >> 3, r = blocks & 7, x = id & 7;
  return x * q + min(x, r) + (id >> 3);
}

// TPR threads hold a row, VPT chunks of 8 columns each; 256 / TPR rows a
// workgroup below 256.
template <typename T, typename W, int TPR, int VPT>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) fp8_rmsnorm_kernel(const NormArgs p) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
  __shared__ float red[NT / kWave];
  const int t = threadIdx.x % TPR;
  const int64_t blocks = (p.rows + RPB - 1) / RPB;
  const int64_t at = row_block(blocks) * RPB + threadIdx.x / TPR;
  const bool valid = at < p.rows;
  const int64_t row = valid ? at : p.rows - 1;
  float v[VPT][8], r[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    load_cols<T>(static_cast<const T*>(p.x) + row * p.ldx, (i * TPR + t) * 8, p.cols, v[i]);
  if (p.residual != nullptr) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      load_cols<T>(static_cast<const T*>(p.residual) + row * p.ldr, (i * TPR + t) * 8, p.cols, r[i]);
#pragma unroll
    for (int i = 0; i < VPT; ++i) add_residual<T>(p, row, (i * TPR + t) * 8, valid, r[i], v[i]);
  }
  float ss = 0.f, amax[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c0 = (i * TPR + t) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
    times_weight<W>(p, c0, v[i]);
    amax[i] = __uint_as_float(max(group_max(amax8(v[i])), kLeastBits));
    if (valid) store_codes(p.o.q + row * p.o.ldq, c0, p.cols, codes8(v[i], kTop / amax[i]));
  }
  ss = group_reduce<SumOp, TPR>(ss, red);
  const float rstd = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
  if (!valid || t % kLanes != 0) return;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c0 = (i * TPR + t) * 8;
    if (c0 < p.cols) p.o.scale[row * p.o.sr + c0 / kGroup * p.o.sg] = amax[i] * rstd / kTop;
  }
}

// Rows of any length: the groups' largest magnitudes wait in LDS for the sum.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) fp8_rmsnorm_long_kernel(const NormArgs p) {
  constexpr int NT = 1024;
  extern __shared__ float amax[];
  __shared__ float red[NT / kWave];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int passes = static_cast<int>((p.cols + NT * 8 - 1) / (NT * 8));
  float ss = 0.f;
  for (int i = 0; i < passes; ++i) {
    const int64_t c0 = (static_cast<int64_t>(i) * NT + t) * 8;
    float v[8], r[8];
    load_cols<T>(static_cast<const T*>(p.x) + row * p.ldx, c0, p.cols, v);
    if (p.residual != nullptr) {
      load_cols<T>(static_cast<const T*>(p.residual) + row * p.ldr, c0, p.cols, r);
      add_residual<T>(p, row, c0, true, r, v);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
    times_weight<W>(p, c0, v);
    const float a = __uint_as_float(max(group_max(amax8(v)), kLeastBits));
    store_codes(p.o.q + row * p.o.ldq, c0, p.cols, codes8(v, kTop / a));
    if (t % kLanes == 0 && c0 < p.cols) amax[c0 / kGroup] = a;
  }
  ss = group_reduce<SumOp, NT>(ss, red);
  const float rstd = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
  const int ng = static_cast<int>((p.cols + kGroup - 1) / kGroup);
  for (int g = t; g < ng; g += NT) p.o.scale[row * p.o.sr + g * p.o.sg] = amax[g] * rstd / kTop;
}

// Rows, columns and strides common to the entry points below.
int check_out(const char* what, int64_t rows, int64_t cols, const Out& o) {
  SPH_REQUIRE(rows >= 0 && cols >= 0, SPH_ERR_INVALID_ARG, std::string(what) + ": negative size");
  SPH_REQUIRE(rows == 0 || cols == 0 || (o.q != nullptr && o.scale != nullptr),
              SPH_ERR_INVALID_ARG, std::string(what) + ": null output");
  SPH_REQUIRE(rows <= 1 || o.ldq >= cols, SPH_ERR_INVALID_ARG,
              std::string(what) + ": ldq is less than the columns");
  SPH_REQUIRE(o.sr >= 0 && o.sg >= 0, SPH_ERR_INVALID_ARG,
              std::string(what) + ": negative scale stride");
  SPH_REQUIRE(rows <= int64_t{1} << 48 && cols <= INT32_MAX, SPH_ERR_TOO_LARGE,
              std::string(what) + ": too many rows or columns");
  return SPH_OK;
}

template <typename S>
int launch_groups(const char* what, const S& src, const Out& o, int64_t rows, int64_t cols,
                  hipStream_t stream) {
  const int64_t ng = fp8::groups(cols), nr = ceil_div(rows, 16);
  if (const int rc = fp8::check_grid(what, ng, 256)) return rc;
  const dim3 grid(static_cast<uint32_t>(ng), static_cast<uint32_t>(nr < 65535 ? nr : 65535));
  fp8_groups_kernel<S><<<grid, 256, 0, stream>>>(src, o, rows, cols);
  return check_launch(what);
}

template <typename T>
int quantize(const void* x, int64_t ldx, int64_t rows, int64_t cols, int64_t block_rows,
             const Out& o, hipStream_t stream) {
  const Values<T> src{static_cast<const T*>(x), ldx};
  if (block_rows == 1) return launch_groups("sph_quantize_fp8", src, o, rows, cols, stream);
  SPH_REQUIRE(ceil_div(rows, kGroup) <= 65535, SPH_ERR_TOO_LARGE,
              "sph_quantize_fp8: more than 65535 blocks of 128 rows");
  if (const int rc = fp8::check_grid("sph_quantize_fp8", fp8::groups(cols), 256)) return rc;
  const dim3 grid(static_cast<uint32_t>(fp8::groups(cols)),
                  static_cast<uint32_t>(ceil_div(rows, kGroup)));
  fp8_blocks_kernel<T><<<grid, 256, 0, stream>>>(src, o, rows, cols);
  return check_launch("sph_quantize_fp8");
}

template <typename T, typename W, int TPR, int VPT>
int launch_rmsnorm(const NormArgs& p, hipStream_t stream) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  const int64_t wgs = ceil_div(p.rows, NT / TPR);
  if (const int rc = fp8::check_grid("sph_rmsnorm_fp8", wgs, NT)) return rc;
  fp8_rmsnorm_kernel<T, W, TPR, VPT><<<static_cast<uint32_t>(wgs), NT, 0, stream>>>(p);
  return check_launch("sph_rmsnorm_fp8");
}

template <typename T, typename W>
int rmsnorm(const NormArgs& p, hipStream_t stream) {
  // One chunk of 8 columns a thread wherever a workgroup holds the row: 8192 x
  // 4096 (with residual) 49.8 us on 512 threads, 52.3 on 256 of two chunks, 66.7
  // on 64 of eight; 1000 x 16384 25.1 by passes, 26.7 on 1024 threads of two.
  if (p.cols <= 512) return launch_rmsnorm<T, W, 64, 1>(p, stream);
  if (p.cols <= 1024) return launch_rmsnorm<T, W, 64, 2>(p, stream);
  if (p.cols <= 2048) return launch_rmsnorm<T, W, 256, 1>(p, stream);
  if (p.cols <= 4096) return launch_rmsnorm<T, W, 512, 1>(p, stream);
  if (p.cols <= 8192) return launch_rmsnorm<T, W, 1024, 1>(p, stream);
  if (const int rc = fp8::check_grid("sph_rmsnorm_fp8", p.rows, 1024)) return rc;
  fp8_rmsnorm_long_kernel<T, W><<<static_cast<uint32_t>(p.rows), 1024,
                                  static_cast<size_t>(fp8::groups(p.cols)) * 4, stream>>>(p);
  return check_launch("sph_rmsnorm_fp8");
}

}  // namespace
}  // namespace sph

using namespace sph;

extern "C" int sph_quantize_fp8(sph_dtype dtype, const void* x, int64_t ldx, int64_t rows,
                                int64_t cols, int64_t block_rows, void* q, int64_t ldq,
                                float* scale, int64_t scale_row_stride,
                                int64_t scale_group_stride, sph_stream_t stream) {
  const Out o{static_cast<uint8_t*>(q), ldq, scale, scale_row_stride, scale_group_stride};
  if (const int rc = check_out("sph_quantize_fp8", rows, cols, o)) return rc;
  SPH_REQUIRE(block_rows == 1 || block_rows == kGroup, SPH_ERR_INVALID_ARG,
              "sph_quantize_fp8: block_rows must be 1 or 128");
  SPH_REQUIRE(rows <= 1 || ldx >= cols, SPH_ERR_INVALID_ARG,
              "sph_quantize_fp8: ldx is less than the columns");
  SPH_REQUIRE(dtype == SPH_F16 || dtype == SPH_BF16 || dtype == SPH_F32, SPH_ERR_UNSUPPORTED,
              "sph_quantize_fp8: dtype must be F16, BF16 or F32");
  if (rows == 0 || cols == 0) return SPH_OK;
  SPH_REQUIRE(x != nullptr, SPH_ERR_INVALID_ARG, "sph_quantize_fp8: null input");
  const hipStream_t s = as_stream(stream);
  if (dtype == SPH_F16) return quantize<half_t>(x, ldx, rows, cols, block_rows, o, s);
  if (dtype == SPH_BF16) return quantize<bf16_t>(x, ldx, rows, cols, block_rows, o, s);
  return quantize<float>(x, ldx, rows, cols, block_rows, o, s);
}

extern "C" int sph_silu_mul_fp8(sph_dtype dtype, const void* gu, int64_t ld, int64_t rows,
                                int64_t cols, void* q, int64_t ldq, float* scale,
                                int64_t scale_row_stride, int64_t scale_group_stride,
                                sph_stream_t stream) {
  const Out o{static_cast<uint8_t*>(q), ldq, scale, scale_row_stride, scale_group_stride};
  if (const int rc = check_out("sph_silu_mul_fp8", rows, cols, o)) return rc;
  SPH_REQUIRE(rows <= 1 || ld >= 2 * cols, SPH_ERR_INVALID_ARG,
              "sph_silu_mul_fp8: ld is less than the gate and up columns");
  if (const int rc = fp8::check_grid("sph_silu_mul_fp8", ceil_div(rows, 16), 256)) return rc;
  SPH_REQUIRE(dtype == SPH_F16 || dtype == SPH_BF16, SPH_ERR_UNSUPPORTED,
              "sph_silu_mul_fp8: dtype must be F16 or BF16");
  if (rows == 0 || cols == 0) return SPH_OK;
  SPH_REQUIRE(gu != nullptr, SPH_ERR_INVALID_ARG, "sph_silu_mul_fp8: null input");
  const hipStream_t s = as_stream(stream);
  if (dtype == SPH_F16)
    return launch_groups("sph_silu_mul_fp8", SiluMul<half_t>{static_cast<const half_t*>(gu), ld}, o,
                         rows, cols, s);
  return launch_groups("sph_silu_mul_fp8", SiluMul<bf16_t>{static_cast<const bf16_t*>(gu), ld}, o,
                       rows, cols, s);
}

extern "C" int sph_rmsnorm_fp8(sph_dtype dtype, sph_dtype w_dtype, const void* x, int64_t ldx,
                               const void* residual, int64_t ld_residual, const void* weight,
                               void* h_out, int64_t ld_h, int64_t rows, int64_t cols, float eps,
                               void* q, int64_t ldq, float* scale, int64_t scale_row_stride,
                               int64_t scale_group_stride, sph_stream_t stream) {
  const Out o{static_cast<uint8_t*>(q), ldq, scale, scale_row_stride, scale_group_stride};
  if (const int rc = check_out("sph_rmsnorm_fp8", rows, cols, o)) return rc;
  SPH_REQUIRE(fp8::groups(cols) <= 8192, SPH_ERR_TOO_LARGE,
              "sph_rmsnorm_fp8: rows of more than 1048576 columns");
  SPH_REQUIRE(rows <= 1 || ldx >= cols, SPH_ERR_INVALID_ARG,
              "sph_rmsnorm_fp8: ldx is less than the columns");
  SPH_REQUIRE(dtype == SPH_F16 || dtype == SPH_BF16, SPH_ERR_UNSUPPORTED,
              "sph_rmsnorm_fp8: dtype must be F16 or BF16");
  SPH_REQUIRE(weight == nullptr || w_dtype == SPH_F32 || w_dtype == dtype, SPH_ERR_UNSUPPORTED,
              "sph_rmsnorm_fp8: w_dtype must be F32 or the activation dtype");
  if (rows == 0 || cols == 0) return SPH_OK;
  SPH_REQUIRE(x != nullptr, SPH_ERR_INVALID_ARG, "sph_rmsnorm_fp8: null input");
  if (residual != nullptr) {
    SPH_REQUIRE(h_out != nullptr, SPH_ERR_INVALID_ARG,
                "sph_rmsnorm_fp8: a residual needs h_out for the sum");
    SPH_REQUIRE(rows <= 1 || (ld_residual >= cols && ld_h >= cols), SPH_ERR_INVALID_ARG,
                "sph_rmsnorm_fp8: ld_residual or ld_h is less than the columns");
  }
  const NormArgs p{x,    residual, weight, h_out, ldx, ld_residual, ld_h,
                   rows, cols,     eps,    o};
  const hipStream_t s = as_stream(stream);
  const bool wf = weight != nullptr && w_dtype == SPH_F32;
  if (dtype == SPH_F16) return wf ? rmsnorm<half_t, float>(p, s) : rmsnorm<half_t, half_t>(p, s);
  return wf ? rmsnorm<bf16_t, float>(p, s) : rmsnorm<bf16_t, bf16_t>(p, s);
}
