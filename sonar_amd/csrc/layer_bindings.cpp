// Torch op registration of the operators of sonar_layer.h, in the library's own namespace `sonar_amd`.  No kernels live
// here: argument checks, the tensors of the results, and the call of the C ABI on the current stream of the inputs' device.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <hip/hip_runtime_api.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "sonar_layer.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void raise_if_failed(int rc) {
  if (rc != SONAR_OK) TORCH_CHECK(false, sonar_layer_last_error());
}

void* current_stream(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

int dtype_code(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kHalf) return SONAR_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return SONAR_DTYPE_BF16;
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be float16, bfloat16 or float32; got ", t.scalar_type());
  return SONAR_DTYPE_F32;
}

// A new contiguous tensor on t's device, straight from the allocator: at::empty finds the same function through the
// dispatcher, which a call of a few microseconds would feel.
Tensor new_tensor(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, at::kStrided, t.device(), std::nullopt, std::nullopt);
}

// The rows of `t` (its last dimension, `cols` long) behind each other, `stride` apart: `t` itself where its strides say
// so, else a copy.  Rows that share memory (an expanded tensor) are copied too.
Tensor rows_of(const Tensor& t, int64_t cols, int64_t& stride) {
  Tensor rows = t.dim() == 2 ? t : t.reshape({-1, cols});
  if (rows.numel() > 0 && ((cols > 1 && rows.stride(1) != 1) || (rows.size(0) > 1 && rows.stride(0) < cols))) rows = rows.contiguous();
  stride = rows.size(0) > 1 ? rows.stride(0) : cols;
  return rows;
}

// ---------------------------------------------------------------- norm
// {codes, scales}, then z where there is a residual, then the norm where it is asked for
std::vector<Tensor> rms_norm_per_token_quant(const Tensor& x, const Tensor& weight, const OptTensor& residual, double epsilon,
                                             at::ScalarType quant_dtype, bool with_norm) {
  TORCH_CHECK(x.is_cuda(), "x is not on GPU");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "x must have a non-empty last dimension");
  const int dtype = dtype_code(x, "x");
  TORCH_CHECK(quant_dtype == at::kChar || quant_dtype == at::kFloat8_e4m3fn, "quant_dtype must be int8 or float8_e4m3fn; got ",
              quant_dtype);
  const int64_t cols = x.size(-1);
  TORCH_CHECK(weight.device() == x.device() && weight.scalar_type() == x.scalar_type() && weight.dim() == 1 &&
                  weight.size(0) == cols, "weight must hold ", cols, " numbers of x's type on x's device");
  if (residual.has_value())
    TORCH_CHECK(residual->device() == x.device() && residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes(),
                "residual must have the shape, type and device of x");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  int64_t x_stride = 0, residual_stride = 0;
  const Tensor in = rows_of(x, cols, x_stride), scale_of_column = weight.contiguous();
  const Tensor old = residual.has_value() ? rows_of(*residual, cols, residual_stride) : Tensor();
  const bool fp8 = quant_dtype == at::kFloat8_e4m3fn;
  Tensor q = new_tensor(x, x.sizes(), quant_dtype);
  auto scale_shape = x.sizes().vec();
  scale_shape.back() = 1;
  Tensor scales = new_tensor(x, scale_shape, at::kFloat);
  Tensor sum = residual.has_value() ? new_tensor(x, x.sizes(), x.scalar_type()) : Tensor();
  Tensor norm = with_norm ? new_tensor(x, x.sizes(), x.scalar_type()) : Tensor();
  raise_if_failed(sonar_rms_norm_per_token_quant(
      in.const_data_ptr(), x_stride, residual.has_value() ? old.const_data_ptr() : nullptr, residual_stride,
      scale_of_column.const_data_ptr(), residual.has_value() ? sum.mutable_data_ptr() : nullptr,
      with_norm ? norm.mutable_data_ptr() : nullptr, q.mutable_data_ptr(), fp8 ? SONAR_ADTYPE_FP8 : SONAR_ADTYPE_INT8,
      static_cast<float*>(scales.mutable_data_ptr()), dtype, in.size(0), cols, epsilon, current_stream(x)));
  std::vector<Tensor> results{std::move(q), std::move(scales)};
  if (residual.has_value()) results.push_back(std::move(sum));
  if (with_norm) results.push_back(std::move(norm));
  return results;
}

// ---------------------------------------------------------------- int8 product
Tensor scaled_mm_int8(const Tensor& a, const Tensor& b, const Tensor& a_scales, const Tensor& b_scales, at::ScalarType out_dtype,
                      const OptTensor& bias) {
  TORCH_CHECK(a.is_cuda(), "a is not on GPU");
  TORCH_CHECK(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar, "a and b must be int8; got ", a.scalar_type(), " and ",
              b.scalar_type());
  TORCH_CHECK(a.dim() >= 1 && b.dim() == 2, "a must have rows (.., K) and b the shape (K, N)");
  const int64_t k = a.size(-1), n = b.size(1);
  TORCH_CHECK(b.device() == a.device() && b.size(0) == k, "Shape mismatch: b must be (", k, ", N) on a's device; got ", b.sizes());
  TORCH_CHECK((b.stride(0) == 1 || k <= 1) && (b.stride(1) >= k || n <= 1 || k == 0),
              "b must lie column by column (the transpose of an (N, K) weight): its strides are ", b.strides());
  TORCH_CHECK(out_dtype == at::kHalf || out_dtype == at::kBFloat16, "out_dtype must be float16 or bfloat16; got ", out_dtype);
  auto shape = a.sizes().vec();
  shape.back() = n;
  int64_t m = 1;
  for (int64_t i = 0; i + 1 < a.dim(); ++i) m *= a.size(i);
  for (const auto& [s, count, name] : {std::make_tuple(&a_scales, m, "a_scales"), std::make_tuple(&b_scales, n, "b_scales")})
    TORCH_CHECK(s->device() == a.device() && s->scalar_type() == at::kFloat && (s->numel() == 1 || s->numel() == count), name,
                " must hold 1 or ", count, " float32 numbers on a's device");
  if (bias.has_value())
    TORCH_CHECK(bias->device() == a.device() && bias->scalar_type() == out_dtype && bias->numel() == n, "bias must hold ", n,
                " numbers of out_dtype on a's device");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  Tensor c = new_tensor(a, shape, out_dtype);
  int64_t lda = k;
  const Tensor rows = k > 0 ? rows_of(a, k, lda) : a;
  const Tensor sa = a_scales.contiguous(), sb = b_scales.contiguous(), bc = bias.has_value() ? bias->contiguous() : Tensor();
  const int64_t ldb = n > 1 && k > 0 ? b.stride(1) : k;
  const auto bits = reinterpret_cast<uintptr_t>(rows.const_data_ptr()) | reinterpret_cast<uintptr_t>(b.const_data_ptr()) |
                    (uintptr_t)lda | (uintptr_t)ldb;
  const size_t scratch_bytes =
      sonar_scaled_mm_int8_scratch_bytes(m, n, k, bits % 16 == 0 && lda < (1 << 23) && ldb < (1 << 23) ? 1 : 0);
  Tensor scratch;
  if (scratch_bytes > 0) scratch = new_tensor(a, {(int64_t)scratch_bytes}, at::kByte);
  raise_if_failed(sonar_scaled_mm_int8(
      static_cast<const int8_t*>(rows.const_data_ptr()), lda, static_cast<const int8_t*>(b.const_data_ptr()),
      ldb, c.mutable_data_ptr(), static_cast<const float*>(sa.const_data_ptr()), sa.numel(),
      static_cast<const float*>(sb.const_data_ptr()), sb.numel(), bias.has_value() ? bc.const_data_ptr() : nullptr,
      scratch_bytes > 0 ? scratch.mutable_data_ptr() : nullptr, scratch_bytes,
      out_dtype == at::kHalf ? SONAR_DTYPE_F16 : SONAR_DTYPE_BF16, m, n, k, current_stream(a)));
  return c;
}

// ---------------------------------------------------------------- router
std::tuple<Tensor, Tensor> topk_routing(const Tensor& logits, int64_t topk, c10::string_view scoring_func, bool renormalize,
                                        const OptTensor& bias, int64_t num_expert_group, int64_t topk_group,
                                        double routed_scaling_factor) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "the router's logits must be a GPU tensor (tokens, experts)");
  const int dtype = dtype_code(logits, "the router's logits");
  TORCH_CHECK(scoring_func == "softmax" || scoring_func == "sigmoid", "scoring_func must be softmax or sigmoid; got ", scoring_func);
  const int64_t experts = logits.size(1);
  if (bias.has_value())
    TORCH_CHECK(bias->device() == logits.device() && bias->scalar_type() == at::kFloat && bias->numel() == experts,
                "bias must hold ", experts, " float32 numbers on the logits' device");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  int64_t stride = experts;
  const Tensor rows = experts > 0 ? rows_of(logits, experts, stride) : logits;
  const Tensor bc = bias.has_value() ? bias->contiguous() : Tensor();
  const int64_t columns = std::max<int64_t>(std::min(topk, experts), 0);   // (of a call that is refused below, none too many)
  Tensor weights = new_tensor(logits, {logits.size(0), columns}, at::kFloat);
  Tensor ids = new_tensor(logits, {logits.size(0), columns}, at::kInt);
  raise_if_failed(sonar_topk_routing(
      rows.const_data_ptr(), dtype, stride, bias.has_value() ? static_cast<const float*>(bc.const_data_ptr()) : nullptr,
      static_cast<float*>(weights.mutable_data_ptr()), static_cast<int32_t*>(ids.mutable_data_ptr()), logits.size(0), experts, topk,
      scoring_func == "sigmoid" ? SONAR_SCORING_SIGMOID : SONAR_SCORING_SOFTMAX, renormalize ? 1 : 0, num_expert_group, topk_group,
      routed_scaling_factor, current_stream(logits)));
  return {weights, ids};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sonar_amd, m) {
  m.def(
      "rms_norm_per_token_quant(Tensor x, Tensor weight, Tensor? residual, float epsilon, ScalarType quant_dtype, bool with_norm) "
      "-> Tensor[]");
  m.def(
      "scaled_mm_int8(Tensor a, Tensor b, Tensor a_scales, Tensor b_scales, ScalarType out_dtype, Tensor? bias) -> Tensor");
  m.def(
      "topk_routing(Tensor logits, int topk, str scoring_func, bool renormalize, Tensor? bias, int num_expert_group, "
      "int topk_group, float routed_scaling_factor) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(sonar_amd, CUDA, m) {
  m.impl("rms_norm_per_token_quant", &rms_norm_per_token_quant);
  m.impl("scaled_mm_int8", &scaled_mm_int8);
  m.impl("topk_routing", &topk_routing);
}
