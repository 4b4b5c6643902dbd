// A step's projection rows on their way into a paged KV cache: for every token
// the query and key heads are normalised (RMSNorm over the head, optional) and
// rotated to the token's position, keys and values are written to the token's slot, and
// the queries are returned.
//
//   y = x rsqrt(mean x^2 + eps) w            (x itself without norm weights)
//   out = y cos[p] + rot(y) sin[p],  rot(y) = (-y2, y1) for the halves y1, y2
//
// Everything in fp32 from the 16-bit inputs, rounded once at the end; values are
// copied.  A slot below 0 marks a padding row: nothing of it is appended, its
// queries are zeros and its position is not looked at.  A slot or position
// outside its range sets the error word and is treated like padding.
//
// Bound by memory: every element is read and written once.  With 32 query and 2 x 8 further
// heads of 128, fp16, 8192 tokens take 42.2 us (206 MB, 4.9 TB/s; a copy of 1 GiB runs at 5.0),
// 2331 with norms 15.3 (3.9 TB/s), up to 120 the host's call, 5.3 (the kernel 2.6 to 3.7).
// A workgroup takes 2048 elements of one token, so that one token already has several and
// none walks: D / 8 lanes hold a head in 16-byte chunks; the rotation's partner is half a head
// away and comes by a lane exchange, the mean by log2(D / 8) of them.  Rows and cache rows may begin at any element (16-byte
// accesses off their natural alignment).
#include "sph_common.h"

namespace sph {
namespace {

constexpr int kAppendThreads = 256;
constexpr int32_t kPagedIndex = 3;  // error code: slot or position out of range

struct AppendArgs {
  const void* qkv;
  int64_t ld_qkv;
  const void* cos;
  const void* sin;
  int64_t ld_cos, ld_sin, n_positions;
  const int64_t* positions;
  const int64_t* slots;
  const void* q_norm;  // [D] or null
  const void* k_norm;
  float eps;
  void* kc;
  int64_t k_sp, k_sh, k_ss;  // element strides: page, head, position in the page
  void* vc;
  int64_t v_sp, v_sh, v_ss;
  int64_t n_pages, page;
  void* q;  // [tokens, H, D]
  int64_t tokens;
  int nh, nkv, groups;  // groups: workgroups per token
  int32_t* err;
};

// TT: the tables' type, W: the norm weights'.
template <typename T, typename TT, typename W, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs p) {
  constexpr int L = D / 8;  // lanes per head
  const int lane = threadIdx.x % L;
  const int64_t token = blockIdx.x / p.groups;
  const int head = (blockIdx.x % p.groups) * (kAppendThreads / L) + threadIdx.x / L;
  // (whole heads leave together: the lane exchanges below stay inside a head)
  if (head >= p.nh + 2 * p.nkv) return;
  const int c = lane * 8;
  const int64_t slot = p.slots[token];
  const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
  float x[8];
  load8u<T>(static_cast<const T*>(p.qkv) + token * p.ld_qkv + static_cast<int64_t>(head) * D + c, x);
  const int64_t pos = slot >= 0 ? p.positions[token] : 0;
  bool ok = slot >= 0;
  if (ok && (slot >= p.n_pages * p.page || pos < 0 || pos >= p.n_positions)) {
    ok = false;
    if (lane == 0 && head == 0 && p.err != nullptr) *p.err = kPagedIndex;
  }
  T* to = static_cast<T*>(p.q) + (token * p.nh + head) * D;
  if (!ok) {
    if (is_q) {
      const float z[8] = {};
      store8u<T>(to + c, z);
    }
    return;
  }
  if (!is_q) {
    const int64_t pg = slot / p.page, at = slot % p.page;
    to = is_v ? static_cast<T*>(p.vc) + pg * p.v_sp + (head - p.nh - p.nkv) * p.v_sh + at * p.v_ss
              : static_cast<T*>(p.kc) + pg * p.k_sp + (head - p.nh) * p.k_sh + at * p.k_ss;
  }
  if (!is_v) {
    const W* w = static_cast<const W*>(is_q ? p.q_norm : p.k_norm);
    if (w != nullptr) {
      float s = 0.f, wf[8];
      load8u<W>(w + c, wf);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x[e], x[e], s);
      s = wave_reduce<SumOp, L>(s);
      const float r = 1.f / sqrtf(s * (1.f / D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * r * wf[e];
    }
    float cs[8], sn[8];
    load8u<TT>(static_cast<const TT*>(p.cos) + pos * p.ld_cos + c, cs);
    load8u<TT>(static_cast<const TT*>(p.sin) + pos * p.ld_sin + c, sn);
    const float sign = lane < L / 2 ? -1.f : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = __shfl_xor(x[e], L / 2, L);
      x[e] = fmaf(sign * other, sn[e], x[e] * cs[e]);
    }
  }
  store8u<T>(to + c, x);
}

}  // namespace
}  // namespace sph

extern "C" int sph_paged_append(
    sph_dtype dtype, sph_dtype table_dtype, sph_dtype norm_dtype, int64_t tokens, int64_t n_heads,
    int64_t n_kv_heads, int64_t head_dim, const void* qkv, int64_t ld_qkv, const void* cos,
    int64_t ld_cos, const void* sin, int64_t ld_sin, int64_t n_positions, const int64_t* positions,
    const int64_t* slots, const void* q_norm, const void* k_norm, float eps, void* k_cache,
    int64_t k_stride_p, int64_t k_stride_h, int64_t k_stride_s, void* v_cache, int64_t v_stride_p,
    int64_t v_stride_h, int64_t v_stride_s, int64_t n_pages, int64_t page_size, void* q,
    int32_t* error_word, sph_stream_t stream) {
  using namespace sph;
  SPH_REQUIRE(dtype == SPH_F16 || dtype == SPH_BF16, SPH_ERR_UNSUPPORTED,
              "paged append: dtype must be F16 or BF16");
  SPH_REQUIRE(table_dtype == dtype || table_dtype == SPH_F32, SPH_ERR_UNSUPPORTED,
              "paged append: tables must have the rows' type or F32");
  SPH_REQUIRE(norm_dtype == dtype || norm_dtype == SPH_F32, SPH_ERR_UNSUPPORTED,
              "paged append: norm weights must have the rows' type or F32");
  SPH_REQUIRE(head_dim == 64 || head_dim == 128, SPH_ERR_UNSUPPORTED,
              "paged append: head_dim must be 64 or 128");
  SPH_REQUIRE(tokens >= 0 && n_heads > 0 && n_kv_heads > 0 && n_positions >= 0 && n_pages >= 0 &&
                  page_size > 0,
              SPH_ERR_INVALID_ARG, "paged append: bad sizes");
  if (tokens == 0) return SPH_OK;
  SPH_REQUIRE(n_heads < (1 << 20) && n_kv_heads < (1 << 20) && page_size < (1LL << 31) &&
                  n_pages < (1LL << 31),
              SPH_ERR_TOO_LARGE, "paged append: at most 2^20 heads, 2^31 pages of 2^31 positions");
  SPH_REQUIRE(qkv != nullptr && q != nullptr && positions != nullptr && slots != nullptr &&
                  ((cos != nullptr && sin != nullptr) || n_positions == 0) &&
                  ((k_cache != nullptr && v_cache != nullptr) || n_pages == 0),
              SPH_ERR_INVALID_ARG, "paged append: null pointer");
  SPH_REQUIRE(tokens == 1 || ld_qkv >= (n_heads + 2 * n_kv_heads) * head_dim, SPH_ERR_INVALID_ARG,
              "paged append: leading dimension too small");
  const int64_t per = kAppendThreads / (head_dim / 8);
  const int64_t groups = ceil_div(n_heads + 2 * n_kv_heads, per);
  // a launch holds 2^32 threads
  SPH_REQUIRE(tokens < (1LL << 24) && tokens * groups < (1LL << 24), SPH_ERR_TOO_LARGE,
              "paged append: at most 2^24 groups of heads over the tokens");
  AppendArgs a{qkv, ld_qkv, cos, sin, ld_cos, ld_sin, n_positions, positions, slots, q_norm, k_norm,
               eps, k_cache, k_stride_p, k_stride_h, k_stride_s, v_cache, v_stride_p, v_stride_h,
               v_stride_s, n_pages, page_size, q, tokens, static_cast<int>(n_heads),
               static_cast<int>(n_kv_heads), static_cast<int>(groups), error_word};
  const dim3 grid(static_cast<unsigned>(tokens * groups));
  hipStream_t st = as_stream(stream);
  auto go = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    if (table_dtype == SPH_F32) {
      if (norm_dtype == SPH_F32) paged_append_kernel<T, float, float, D><<<grid, kAppendThreads, 0, st>>>(a);
      else paged_append_kernel<T, float, T, D><<<grid, kAppendThreads, 0, st>>>(a);
    } else {
      if (norm_dtype == SPH_F32) paged_append_kernel<T, T, float, D><<<grid, kAppendThreads, 0, st>>>(a);
      else paged_append_kernel<T, T, T, D><<<grid, kAppendThreads, 0, st>>>(a);
    }
  };
  auto by_dim = [&](auto t) {
    if (head_dim == 128) go(t, std::integral_constant<int, 128>{});
    else go(t, std::integral_constant<int, 64>{});
  };
  if (dtype == SPH_F16) by_dim(half_t{});
  else by_dim(bf16_t{});
  return check_launch("sph_paged_append");
}
