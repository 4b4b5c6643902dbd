// Serving from a paged KV cache on spyre tensors: torch.ops.spyre.paged_append,
// paged_attention and sample (schemas and the formulas for other devices:
// torch_spyre/_inductor/serving.py).  Registered here, not through Python
// kernels, for the host time of a call (ops_fp8.cpp).
//
// No reference function corresponds: the reference has no KV cache and no sampling.
#include <ATen/MemoryOverlap.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>

#include "spyre_ops_common.h"

namespace spyre {
namespace {

bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

void check_device(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on ", t.device(),
              ", expected ", like.device());
}

// A 1-D tensor of `n` values of one type, contiguous.
at::Tensor vec(const at::Tensor& t, int64_t n, at::ScalarType dtype, const at::Tensor& like,
               const char* op, const char* name) {
  check_device(t, like, op, name);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.scalar_type() == dtype, op, ": ", name,
              " must be [", n, "] of ", dtype, ", got ", t.sizes(), " of ", t.scalar_type());
  return contiguous_on_device(t);
}

void check_strided(const at::Tensor& t, const char* what) {
  if (t.numel() > 0)
    check_extent(t, t.data_ptr(), t.dim(), t.sizes().data(), t.strides().data(), t.element_size(),
                 what);
}

// The caches of a call: [pages, n_kv_heads, page_size, head_dim], dim stride 1.
void check_caches(const at::Tensor& k, const at::Tensor& v, const at::Tensor& like, int64_t dim,
                  const char* op) {
  check_device(k, like, op, "k_cache");
  check_device(v, like, op, "v_cache");
  TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes() && k.size(1) > 0 && k.size(2) > 0, op,
              ": k_cache and v_cache must be [pages, n_kv_heads, page_size, head_dim], got ",
              k.sizes(), " and ", v.sizes());
  TORCH_CHECK(k.scalar_type() == like.scalar_type() && v.scalar_type() == like.scalar_type(), op,
              ": the caches must have the type ", like.scalar_type());
  TORCH_CHECK(dim < 0 || k.size(3) == dim, op, ": the caches' head_dim must be ", dim, ", got ",
              k.size(3));
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, op, ": head_dim must be 64 or 128 on spyre, got ",
              k.size(3));
  TORCH_CHECK(k.numel() == 0 || (k.stride(3) == 1 && v.stride(3) == 1), op,
              ": the caches' last dimension must have stride 1");
  check_strided(k, "k_cache");
  check_strided(v, "v_cache");
}

// The kernel writes `t` past the dispatcher: its version rises here, so that a backward pass
// which saved it before raises instead of taking the new values.  (Inference tensors have no
// version and are saved by none.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::Tensor paged_append(const at::Tensor& qkv_in, const at::Tensor& cos_in,
                        const at::Tensor& sin_in, const at::Tensor& positions_in,
                        const at::Tensor& slots_in, at::Tensor& k_cache, at::Tensor& v_cache,
                        int64_t n_heads, const std::optional<at::Tensor>& q_norm_in,
                        const std::optional<at::Tensor>& k_norm_in, double eps) {
  const char* op = "paged_append";
  const at::ScalarType dt = qkv_in.scalar_type();
  TORCH_CHECK(half_type(dt), "paged_append: qkv must be fp16 or bf16, got ", dt);
  check_caches(k_cache, v_cache, qkv_in, -1, op);
  at::assert_no_internal_overlap(k_cache);
  at::assert_no_internal_overlap(v_cache);
  at::assert_no_overlap(k_cache, v_cache);
  // (a workgroup would read what another has written)
  for (const at::Tensor* in : {&qkv_in, &cos_in, &sin_in, &positions_in, &slots_in}) {
    at::assert_no_overlap(k_cache, *in);
    at::assert_no_overlap(v_cache, *in);
  }
  const int64_t kv = k_cache.size(1), page = k_cache.size(2), d = k_cache.size(3);
  TORCH_CHECK(n_heads > 0 && qkv_in.dim() == 2 && qkv_in.size(1) == (n_heads + 2 * kv) * d,
              "paged_append: qkv must be [tokens, (n_heads + 2 n_kv_heads) * head_dim] = [tokens, ",
              (n_heads + 2 * kv) * d, "], got ", qkv_in.sizes());
  const int64_t tokens = qkv_in.size(0);
  check_device(cos_in, qkv_in, op, "cos");
  check_device(sin_in, qkv_in, op, "sin");
  TORCH_CHECK(cos_in.dim() == 2 && cos_in.size(1) == d && sin_in.sizes() == cos_in.sizes() &&
                  sin_in.scalar_type() == cos_in.scalar_type() &&
                  (cos_in.scalar_type() == dt || cos_in.scalar_type() == at::kFloat),
              "paged_append: cos and sin must be [positions, ", d, "] of qkv's type or fp32");
  c10::DeviceGuard guard(qkv_in.device());
  const at::Tensor positions = vec(positions_in, tokens, at::kLong, qkv_in, op, "positions");
  const at::Tensor slots = vec(slots_in, tokens, at::kLong, qkv_in, op, "slots");
  at::Tensor norms[2];
  at::ScalarType nt = dt;
  for (int i = 0; i < 2; ++i) {
    const auto& in = i == 0 ? q_norm_in : k_norm_in;
    if (!in.has_value() || !in->defined()) continue;
    nt = in->scalar_type();
    TORCH_CHECK(nt == dt || nt == at::kFloat,
                "paged_append: norm weights must have qkv's type or fp32, got ", nt);
    TORCH_CHECK(i == 0 || !norms[0].defined() || norms[0].scalar_type() == nt,
                "paged_append: q_norm and k_norm must have one type");
    at::assert_no_overlap(k_cache, *in);
    at::assert_no_overlap(v_cache, *in);
    norms[i] = vec(*in, d, nt, qkv_in, op, i == 0 ? "q_norm" : "k_norm");
  }
  const at::Tensor qkv =
      qkv_in.numel() == 0 ||
              (qkv_in.stride(1) == 1 && (tokens == 1 || qkv_in.stride(0) >= qkv_in.size(1)))
          ? qkv_in
          : contiguous_on_device(qkv_in);
  const at::Tensor cos = cos_in.stride(1) == 1 ? cos_in : contiguous_on_device(cos_in);
  const at::Tensor sin = sin_in.stride(1) == 1 ? sin_in : contiguous_on_device(sin_in);
  check_strided(qkv, "qkv");
  check_strided(cos, "cos");
  check_strided(sin, "sin");
  at::Tensor q = empty_spyre({tokens, n_heads, d}, dt, qkv.device());
  written(k_cache);
  written(v_cache);
  if (tokens == 0) return q;
  const int dev = qkv.get_device();
  SPYRE_SPH_CHECK(sph_paged_append(
      to_sph(dt), to_sph(cos.scalar_type()), to_sph(nt), tokens, n_heads, kv, d, qkv.data_ptr(),
      qkv.stride(0), cos.data_ptr(), cos.stride(0), sin.data_ptr(), sin.stride(0), cos.size(0),
      positions.data_ptr<int64_t>(), slots.data_ptr<int64_t>(),
      norms[0].defined() ? norms[0].data_ptr() : nullptr,
      norms[1].defined() ? norms[1].data_ptr() : nullptr, static_cast<float>(eps),
      k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
      v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
      k_cache.size(0), page, q.data_ptr(), device_error_word(dev), stream(dev)));
  return q;
}

at::Tensor paged_attention(const at::Tensor& q_in, const at::Tensor& k_cache,
                           const at::Tensor& v_cache, const at::Tensor& table_in,
                           const at::Tensor& lens_in, const at::Tensor& starts_in, double scale,
                           const std::optional<at::Tensor>& mask_in) {
  const char* op = "paged_attention";
  const at::ScalarType dt = q_in.scalar_type();
  TORCH_CHECK(half_type(dt), "paged_attention: q must be fp16 or bf16, got ", dt);
  TORCH_CHECK(q_in.dim() == 3, "paged_attention: q must be [tokens, n_heads, head_dim], got ",
              q_in.sizes());
  check_caches(k_cache, v_cache, q_in, q_in.size(2), op);
  const int64_t tokens = q_in.size(0), heads = q_in.size(1), d = q_in.size(2);
  const int64_t kv = k_cache.size(1), page = k_cache.size(2);
  TORCH_CHECK(heads > 0 && heads % kv == 0, "paged_attention: ", heads,
              " query heads are no multiple of ", kv, " KV heads");
  TORCH_CHECK(scale > 0 && std::isfinite(scale),
              "paged_attention: scale must be positive and finite, got ", scale);
  check_device(table_in, q_in, op, "block_table");
  TORCH_CHECK(table_in.dim() == 2 && table_in.scalar_type() == at::kLong,
              "paged_attention: block_table must be [sequences, pages] of int64, got ",
              table_in.sizes(), " of ", table_in.scalar_type());
  const int64_t batch = table_in.size(0), width = table_in.size(1);
  c10::DeviceGuard guard(q_in.device());
  const at::Tensor lens = vec(lens_in, batch, at::kLong, q_in, op, "seq_lens");
  const at::Tensor starts = vec(starts_in, batch + 1, at::kLong, q_in, op, "q_starts");
  const at::Tensor table =
      table_in.numel() == 0 || table_in.stride(1) == 1 ? table_in : contiguous_on_device(table_in);
  at::Tensor mask;
  if (mask_in.has_value() && mask_in->defined()) {
    check_device(*mask_in, q_in, op, "mask");
    TORCH_CHECK(mask_in->dim() == 2 && mask_in->size(0) == tokens &&
                    mask_in->scalar_type() == at::kBool,
                "paged_attention: mask must be [", tokens, ", new tokens] of bool, got ",
                mask_in->sizes(), " of ", mask_in->scalar_type());
    mask = mask_in->numel() == 0 || (mask_in->stride(1) == 1 &&
                                     (tokens == 1 || mask_in->stride(0) >= mask_in->size(1)))
               ? *mask_in
               : contiguous_on_device(*mask_in);
    check_strided(mask, "mask");
  }
  const at::Tensor q = q_in.stride(2) == 1 ? q_in : contiguous_on_device(q_in);
  check_strided(q, "q");
  check_strided(table, "block_table");
  at::Tensor out = empty_spyre({tokens, heads, d}, dt, q.device());
  if (tokens == 0) return out;
  if (batch == 0) return out.zero_();
  const int64_t bytes =
      sph_paged_attention_workspace_bytes(tokens, batch, heads, kv, d, width * page);
  const at::Tensor ws = empty_spyre({bytes}, at::kByte, q.device());
  // (a mask without columns is none without a pointer: any other, never read)
  const uint8_t* mp = !mask.defined() ? nullptr
                                      : static_cast<const uint8_t*>(
                                            mask.numel() ? mask.data_ptr() : out.data_ptr());
  const int dev = q.get_device();
  SPYRE_SPH_CHECK(sph_paged_attention(
      to_sph(dt), tokens, batch, heads, kv, d, q.data_ptr(), q.stride(0), q.stride(1),
      k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
      v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2), k_cache.size(0),
      page, table.numel() ? table.data_ptr<int64_t>() : nullptr, table.stride(0), width,
      lens.data_ptr<int64_t>(), starts.data_ptr<int64_t>(), mp,
      mask.defined() ? std::max(mask.stride(0), mask.size(1)) : 0,
      mask.defined() ? mask.size(1) : 0, static_cast<float>(scale), out.data_ptr(), ws.data_ptr(),
      bytes, device_error_word(dev), stream(dev)));
  return out;
}

at::Tensor sample(const at::Tensor& logits_in, const at::Tensor& uniform_in,
                  const std::optional<at::Tensor>& temperature_in,
                  const std::optional<at::Tensor>& top_k_in,
                  const std::optional<at::Tensor>& top_p_in,
                  const std::optional<at::Tensor>& min_p_in) {
  const char* op = "sample";
  const at::ScalarType dt = logits_in.scalar_type();
  TORCH_CHECK(half_type(dt) || dt == at::kFloat, "sample: logits must be fp16, bf16 or fp32, got ",
              dt);
  TORCH_CHECK(logits_in.dim() == 2 && logits_in.size(1) > 0,
              "sample: logits must be [rows, vocabulary], got ", logits_in.sizes());
  const int64_t rows = logits_in.size(0), vocab = logits_in.size(1);
  c10::DeviceGuard guard(logits_in.device());
  const at::Tensor uniform = vec(uniform_in, rows, at::kFloat, logits_in, op, "uniform");
  auto optional = [&](const std::optional<at::Tensor>& t, at::ScalarType type, const char* name) {
    return t.has_value() && t->defined() ? vec(*t, rows, type, logits_in, op, name) : at::Tensor();
  };
  const at::Tensor temperature = optional(temperature_in, at::kFloat, "temperature");
  const at::Tensor top_k = optional(top_k_in, at::kLong, "top_k");
  const at::Tensor top_p = optional(top_p_in, at::kFloat, "top_p");
  const at::Tensor min_p = optional(min_p_in, at::kFloat, "min_p");
  const at::Tensor logits =
      vocab == 1 || logits_in.stride(1) == 1 ? logits_in : contiguous_on_device(logits_in);
  check_strided(logits, "logits");
  at::Tensor tokens = empty_spyre({rows}, at::kLong, logits.device());
  if (rows == 0) return tokens;
  SPYRE_SPH_CHECK(sph_sample(
      to_sph(dt), rows, vocab, logits.data_ptr(), logits.stride(0), uniform.data_ptr<float>(),
      temperature.defined() ? temperature.data_ptr<float>() : nullptr,
      top_k.defined() ? top_k.data_ptr<int64_t>() : nullptr,
      top_p.defined() ? top_p.data_ptr<float>() : nullptr,
      min_p.defined() ? min_p.data_ptr<float>() : nullptr, tokens.data_ptr<int64_t>(),
      stream(logits.get_device())));
  return tokens;
}

}  // namespace

TORCH_LIBRARY_IMPL(spyre, PrivateUse1, m) {
  m.impl("paged_append", TORCH_FN(paged_append));
  m.impl("paged_attention", TORCH_FN(paged_attention));
  m.impl("sample", TORCH_FN(sample));
}

TORCH_LIBRARY_IMPL(spyre, AutogradPrivateUse1, m) {
  for (const char* name : {"paged_append", "paged_attention", "sample"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_gradients>());
}

}  // namespace spyre
