// The 8-bit serving operators on spyre tensors: torch.ops.spyre.quantize_fp8,
// rms_norm_fp8, add_rms_norm_fp8, silu_mul_fp8 and mm_fp8 (schemas and the
// formulas for other devices: torch_spyre/_inductor/customops.py).
//
// They are registered here, not through Python kernels, because a decode step
// makes a call every few microseconds: the Python custom_op wrapper alone takes
// 11 us a call on the host, this path 3 to 4.
//
// No reference function corresponds: the reference has no 8-bit types.
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/library.h>

#include <limits>

#include "spyre_ops_common.h"

namespace spyre {
namespace {

constexpr int64_t kGroup = 128;
constexpr at::ScalarType kCode = at::kFloat8_e4m3fn;

int64_t groups(int64_t cols) { return (cols + kGroup - 1) / kGroup; }

bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

bool aligned16(const at::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

void check_device(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on ", t.device(),
              ", expected ", like.device());
}

// A tensor as rows of its last dimension: element (r, c) at r * ld + c.
struct Rows {
  at::Tensor t;
  int64_t rows, cols, ld;
};

Rows as_rows(const at::Tensor& in, const char* op) {
  TORCH_CHECK(in.dim() >= 1, op, ": needs at least one dimension");
  const int64_t cols = in.size(-1);
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < in.dim(); ++d) rows *= in.size(d);
  // Leading dimensions that one row stride walks (any 2-D view, a
  // contiguous tensor) need no copy.
  bool ok = cols <= 1 || in.stride(-1) == 1;
  int64_t ld = cols, next = -1;
  for (int64_t d = in.dim() - 2; ok && d >= 0; --d) {
    if (in.size(d) == 1) continue;
    if (next < 0)
      ld = in.stride(d);
    else
      ok = in.stride(d) == next;
    next = in.stride(d) * in.size(d);
  }
  ok = ok && (rows <= 1 || ld >= cols);
  at::Tensor t = ok ? in : contiguous_on_device(in);
  Rows r{t, rows, cols, ok ? ld : cols};
  if (in.numel() > 0) {
    const int64_t s[2] = {rows, cols}, st[2] = {r.ld, 1};
    check_extent(t, t.data_ptr(), 2, s, st, t.element_size(), op);
  }
  return r;
}

// Codes of `sizes`: rows of a length off 16 bytes are padded to the next 16, so
// that a product can read them in whole chunks.
at::Tensor empty_codes(at::IntArrayRef sizes, c10::Device device) {
  const int64_t cols = sizes.back();
  if (cols % 16 == 0) return empty_spyre(sizes, kCode, device);
  std::vector<int64_t> padded(sizes.begin(), sizes.end());
  padded.back() = (cols + 15) / 16 * 16;
  return empty_spyre(padded, kCode, device).narrow(-1, 0, cols);
}

// One scale per row and group, a group's scales of all rows side by side.
at::Tensor empty_scales(at::IntArrayRef sizes, int64_t rows, c10::Device device) {
  c10::SmallVector<int64_t, 5> shape(sizes.begin(), sizes.end()), strides(sizes.size());
  shape.back() = groups(sizes.back());
  strides.back() = rows;
  int64_t s = 1;
  for (size_t d = sizes.size() - 1; d-- > 0; s *= sizes[d]) strides[d] = s;
  return at::empty_strided(shape, strides, at::TensorOptions().dtype(at::kFloat).device(device));
}

int64_t row_stride(const at::Tensor& q) { return (q.size(-1) + 15) / 16 * 16; }

std::tuple<at::Tensor, at::Tensor> quantize_fp8(const at::Tensor& x, int64_t block_rows) {
  TORCH_CHECK(x.scalar_type() == at::kFloat || half_type(x.scalar_type()),
              "quantize_fp8: x must be fp16, bf16 or fp32, got ", x.scalar_type());
  TORCH_CHECK(block_rows == 1 || block_rows == kGroup,
              "quantize_fp8: block_rows must be 1 or 128, got ", block_rows);
  TORCH_CHECK(block_rows == 1 || x.dim() == 2,
              "quantize_fp8: blocks of 128 rows need a 2-dimensional x");
  c10::DeviceGuard guard(x.device());
  const Rows r = as_rows(x, "quantize_fp8");
  at::Tensor q = empty_codes(x.sizes(), x.device()), s;
  int64_t sr = 1, sg = r.rows;
  if (block_rows == 1) {
    s = empty_scales(x.sizes(), r.rows, x.device());
  } else {
    s = empty_spyre({(r.rows + kGroup - 1) / kGroup, groups(r.cols)}, at::kFloat, x.device());
    sr = s.size(1);
    sg = 1;
  }
  SPYRE_SPH_CHECK(sph_quantize_fp8(to_sph(x.scalar_type()), r.t.data_ptr(), r.ld, r.rows, r.cols,
                                   block_rows, q.data_ptr(), row_stride(q),
                                   static_cast<float*>(s.data_ptr()), sr, sg,
                                   stream(x.get_device())));
  return {q, s};
}

// rms_norm_fp8 and, with a residual, add_rms_norm_fp8.
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm(const char* op, const at::Tensor& x,
                                                    const at::Tensor* residual,
                                                    const std::optional<at::Tensor>& weight,
                                                    double eps) {
  TORCH_CHECK(half_type(x.scalar_type()), op, ": x must be fp16 or bf16, got ", x.scalar_type());
  c10::DeviceGuard guard(x.device());
  const Rows r = as_rows(x, op);
  Rows res{};
  at::Tensor h;
  if (residual) {
    check_device(*residual, x, op, "residual");
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), op,
                ": residual must have x's shape and type");
    res = as_rows(*residual, op);
    h = empty_spyre(x.sizes(), x.scalar_type(), x.device());
  }
  at::Tensor w;
  if (weight.has_value() && weight->defined()) {
    check_device(*weight, x, op, "weight");
    TORCH_CHECK(weight->dim() == 1 && weight->size(0) == r.cols, op, ": weight must be [", r.cols,
                "], got ", weight->sizes());
    TORCH_CHECK(weight->scalar_type() == x.scalar_type() || weight->scalar_type() == at::kFloat,
                op, ": weight must have x's type or fp32");
    w = contiguous_on_device(*weight);
  }
  at::Tensor q = empty_codes(x.sizes(), x.device());
  at::Tensor s = empty_scales(x.sizes(), r.rows, x.device());
  SPYRE_SPH_CHECK(sph_rmsnorm_fp8(
      to_sph(x.scalar_type()), to_sph(w.defined() ? w.scalar_type() : x.scalar_type()),
      r.t.data_ptr(), r.ld, residual ? res.t.data_ptr() : nullptr, res.ld,
      w.defined() ? w.data_ptr() : nullptr, h.defined() ? h.data_ptr() : nullptr, r.cols, r.rows,
      r.cols, static_cast<float>(eps), q.data_ptr(), row_stride(q),
      static_cast<float*>(s.data_ptr()), 1, r.rows, stream(x.get_device())));
  return {q, s, h};
}

std::tuple<at::Tensor, at::Tensor> rms_norm_fp8(const at::Tensor& x,
                                                const std::optional<at::Tensor>& weight,
                                                double eps) {
  auto [q, s, h] = norm("rms_norm_fp8", x, nullptr, weight, eps);
  return {q, s};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_fp8(
    const at::Tensor& x, const at::Tensor& residual, const std::optional<at::Tensor>& weight,
    double eps) {
  return norm("add_rms_norm_fp8", x, &residual, weight, eps);
}

std::tuple<at::Tensor, at::Tensor> silu_mul_fp8(const at::Tensor& gu) {
  TORCH_CHECK(half_type(gu.scalar_type()), "silu_mul_fp8: gate_up must be fp16 or bf16, got ",
              gu.scalar_type());
  c10::DeviceGuard guard(gu.device());
  const Rows r = as_rows(gu, "silu_mul_fp8");
  TORCH_CHECK(r.cols % 2 == 0, "silu_mul_fp8: the last dimension must be even, got ", r.cols);
  std::vector<int64_t> shape(gu.sizes().begin(), gu.sizes().end());
  shape.back() = r.cols / 2;
  at::Tensor q = empty_codes(shape, gu.device());
  at::Tensor s = empty_scales(shape, r.rows, gu.device());
  SPYRE_SPH_CHECK(sph_silu_mul_fp8(to_sph(gu.scalar_type()), r.t.data_ptr(), r.ld, r.rows,
                                   r.cols / 2, q.data_ptr(), row_stride(q),
                                   static_cast<float*>(s.data_ptr()), 1, r.rows,
                                   stream(gu.get_device())));
  return {q, s};
}

// Codes whose rows the product can read in whole chunks: as they lie where the
// rows begin on 16 bytes and are at most kMaxLd apart (the entry point's limit),
// else copied into padded rows.
constexpr int64_t kMaxLd = 4194303;
Rows code_rows(const at::Tensor& in, const char* op) {
  Rows r = as_rows(in, op);
  if (r.rows <= 1) r.ld = r.cols;
  if (r.t.numel() == 0 || (aligned16(r.t) && (r.rows <= 1 || (r.ld % 16 == 0 && r.ld <= kMaxLd))))
    return r;
  const int64_t ld = (r.cols + 15) / 16 * 16;
  at::Tensor padded = empty_spyre({r.rows, ld}, kCode, in.device());
  at::Tensor view = padded.narrow(1, 0, r.cols);
  device_copy(view, r.t.as_strided({r.rows, r.cols}, {r.ld, 1}));
  return Rows{view, r.rows, r.cols, ld};
}

at::Tensor mm_fp8(const at::Tensor& x_in, const at::Tensor& x_scale, const at::Tensor& w_in,
                  const at::Tensor& w_scale, at::ScalarType dtype,
                  const std::optional<at::Tensor>& bias_in) {
  const char* op = "mm_fp8";
  check_device(x_scale, x_in, op, "x_scale");
  check_device(w_in, x_in, op, "w");
  check_device(w_scale, x_in, op, "w_scale");
  TORCH_CHECK(x_in.scalar_type() == kCode && w_in.scalar_type() == kCode,
              "mm_fp8: x and w must be float8_e4m3fn, got ", x_in.scalar_type(), " and ",
              w_in.scalar_type());
  TORCH_CHECK(x_scale.scalar_type() == at::kFloat && w_scale.scalar_type() == at::kFloat,
              "mm_fp8: the scales must be fp32");
  TORCH_CHECK(half_type(dtype), "mm_fp8: the result must be fp16 or bf16, got ", dtype);
  TORCH_CHECK(x_in.dim() >= 1 && w_in.dim() == 2 && x_in.size(-1) == w_in.size(1),
              "mm_fp8: x must be [..., K] and w [N, K], got ", x_in.sizes(), " and ",
              w_in.sizes());
  const int64_t k = w_in.size(1), n = w_in.size(0), kb = groups(k);
  std::vector<int64_t> sshape(x_in.sizes().begin(), x_in.sizes().end());
  sshape.back() = kb;
  TORCH_CHECK(x_scale.sizes() == at::IntArrayRef(sshape), "mm_fp8: x_scale must be ",
              at::IntArrayRef(sshape), ", got ", x_scale.sizes());
  TORCH_CHECK(w_scale.dim() == 2 && w_scale.size(0) == groups(n) && w_scale.size(1) == kb,
              "mm_fp8: w_scale must be [", groups(n), ", ", kb, "], got ", w_scale.sizes());
  c10::DeviceGuard guard(x_in.device());
  at::Tensor bias;
  if (bias_in.has_value() && bias_in->defined()) {
    check_device(*bias_in, x_in, op, "bias");
    TORCH_CHECK(bias_in->dim() == 1 && bias_in->size(0) == n && bias_in->scalar_type() == dtype,
                "mm_fp8: bias must be [", n, "] of the result's type");
    bias = contiguous_on_device(*bias_in);
  }
  const Rows x = code_rows(x_in, op), w = code_rows(w_in, op);
  // x_scale as [rows, kb] by two strides
  at::Tensor xs = x_scale.dim() == 2 ? x_scale : x_scale.reshape({x.rows, kb});
  if (xs.stride(0) > (1 << 21)) xs = contiguous_on_device(xs);  // the entry point's limit
  std::vector<int64_t> shape(x_in.sizes().begin(), x_in.sizes().end());
  shape.back() = n;
  at::Tensor out = empty_spyre(shape, dtype, x_in.device());
  if (out.numel() == 0) return out;
  if (k > 0) {
    const int64_t ss[2] = {x.rows, kb}, sst[2] = {xs.stride(0), xs.stride(1)};
    check_extent(xs, xs.data_ptr(), 2, ss, sst, 4, "mm_fp8 x_scale");
    const int64_t ws[2] = {groups(n), kb}, wst[2] = {w_scale.stride(0), w_scale.stride(1)};
    check_extent(w_scale, w_scale.data_ptr(), 2, ws, wst, 4, "mm_fp8 w_scale");
  }
  const at::Tensor wsp =
      optional_workspace(sph_gemm_fp8_workspace_bytes(x.rows, n, k), x_in.device());
  SPYRE_SPH_CHECK(sph_gemm_fp8(
      to_sph(dtype), x.rows, n, k, x.t.data_ptr(), x.ld, static_cast<const float*>(xs.data_ptr()),
      xs.stride(0), xs.stride(1), w.t.data_ptr(), w.ld,
      static_cast<const float*>(w_scale.data_ptr()), w_scale.stride(0), w_scale.stride(1),
      bias.defined() ? bias.data_ptr() : nullptr, out.data_ptr(), n,
      wsp.defined() ? wsp.data_ptr() : nullptr, wsp.defined() ? wsp.numel() : 0,
      stream(x_in.get_device())));
  return out;
}

// Rounding to codes has no gradient: a call that would have to record one, or to
// carry a tangent on, is refused instead of returning tensors that silently cut
// the graph.
void refuse_gradients(const c10::OperatorHandle& op, c10::DispatchKeySet ks,
                      torch::jit::Stack* stack) {
  const bool grad = at::GradMode::is_enabled();
  for (const auto& v : torch::jit::last(*stack, op.schema().arguments().size())) {
    if (!v.isTensor() || !v.toTensor().defined()) continue;
    TORCH_CHECK(!(grad && v.toTensor().requires_grad()), op.schema().name(),
                " has no gradient: call it under torch.no_grad()");
    TORCH_CHECK(!v.toTensor()._fw_grad(/*level=*/0).defined(), op.schema().name(),
                " has no gradient: call it without tangents");
  }
  at::AutoDispatchBelowADInplaceOrView below;
  op.redispatchBoxed(ks & c10::after_autograd_keyset, stack);
}

}  // namespace

TORCH_LIBRARY_IMPL(spyre, PrivateUse1, m) {
  m.impl("quantize_fp8", TORCH_FN(quantize_fp8));
  m.impl("rms_norm_fp8", TORCH_FN(rms_norm_fp8));
  m.impl("add_rms_norm_fp8", TORCH_FN(add_rms_norm_fp8));
  m.impl("silu_mul_fp8", TORCH_FN(silu_mul_fp8));
  m.impl("mm_fp8", TORCH_FN(mm_fp8));
}

TORCH_LIBRARY_IMPL(spyre, AutogradPrivateUse1, m) {
  for (const char* name :
       {"quantize_fp8", "rms_norm_fp8", "add_rms_norm_fp8", "silu_mul_fp8", "mm_fp8"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_gradients>());
}

}  // namespace spyre
